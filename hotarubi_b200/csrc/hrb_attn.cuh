// What the attention kernels (attn_decode.cu, attn_prompt.cu) share: the
// exponential, FP16 operand arithmetic, the outputs.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#include "hrb_quant.cuh"
#include "hrb_serve.cuh"

namespace hrb {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 6.0f;    // log2 of the most a score may pass m before m moves
// Weights are 2^(s - m + kLift), up to 2^14 (kLift may round to 8 where m is
// large): FP16 keeps what lies down to 2^-31 of the largest (2^-24 without it),
// and the factor cancels in O / l.
constexpr float kLift = 7.0f;
// From here on the rounding of a maximum (the score's product with its factor,
// half a unit of 2^-23) is no longer small beside kLazy, and a fused s factor - m
// would be off by it: the products are rounded first, as the maximum was.
constexpr float kFar = 0x1p20f;
__device__ __forceinline__ bool attn_far(float m) { return fabsf(m) >= kFar && fabsf(m) < INFINITY; }

constexpr uint32_t kAttnTileKeys = 128;  // keys a tile of the prompt kernel

// First tile in scratch of request n (a whole warp; the same in all lanes):
// n times the most tiles of a request where the scratch has room for that
// (tile_stride), else the requests' tiles one after another, which every
// block adds up from their lengths.
__device__ __forceinline__ uint32_t attn_first_tile(const AttnJob& j, uint32_t n) {
  if (j.tile_stride != 0u) return n * j.tile_stride;
  uint32_t sum = 0;
  for (uint32_t i = threadIdx.x & 31u; i < n; i += 32u) {
    int32_t q0, q_len, kv;
    if (attn_request(j, i, &q0, &q_len, &kv) && q_len > 0) {
      // Held to what no scratch has (2^26 tiles), so that no sum wraps.
      sum = min(sum + (static_cast<uint32_t>(kv) + kAttnTileKeys - 1u) / kAttnTileKeys, 1u << 26);
    }
  }
  return __reduce_add_sync(0xFFFFFFFFu, sum);
}
// Whether a request's tiles are in the scratch: total_kv may have said less.
__device__ __forceinline__ bool attn_tiles_fit(const AttnJob& j, uint32_t first, int32_t kv) {
  return first + (static_cast<uint32_t>(kv) + kAttnTileKeys - 1u) / kAttnTileKeys <= j.tiles_cap;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A score x to softcap log2(e) tanh(x / softcap), by 1 - 2 / (1 + e^2x).  Its
// error is about 2^-23 of the cap, whatever the score: up to a cap of 256
// under 2^-14 in the exponent, an eighth of the weights' FP16 rounding.  For
// WIDE caps, arguments under 1/4 take tanh's series (to x^7; the next term is
// under 9e-8 there), whose error goes with the score.
constexpr float kWideCap = 256.0f;

template <bool WIDE>
__device__ __forceinline__ float cap_score(const AttnJob& j, float x) {
  const float y = j.cap_out * (1.0f - __fdividef(2.0f, 1.0f + ex2(x * j.cap_in)));
  if constexpr (!WIDE) return y;
  const float a = x * j.cap_inv, u = a * a;
  const float r = fmaf(u, fmaf(u, fmaf(u, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
  const float series = j.cap_out * (a * r);
  return u < 0.0625f ? series : y;
}

// Pairs of FP32 in a 64-bit register: one instruction for both.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t mul_2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add_2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma_2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) {
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  return half2_bits(__hmul2(*reinterpret_cast<const __half2*>(&a),
                            *reinterpret_cast<const __half2*>(&b)));
}

// Two scale bytes as FP16 powers of two, `lo` in the low half.  Bytes
// outside the cache's range (stale keys) become its ends after the
// conversion, which takes two fewer instructions than before it.
__device__ __forceinline__ uint32_t scale2(uint32_t lo, uint32_t hi) {
  const __half2 h = __floats2half2_rn(__uint_as_float(lo << 23), __uint_as_float(hi << 23));
  const __half2 most = __half2half2(__ushort_as_half(0x7000));   // 2^13
  const __half2 least = __half2half2(__ushort_as_half(0x0002));  // 2^-23
  return half2_bits(__hmax2(__hmin2(h, most), least));
}

// FP32 value of dim 32 b + lane of one output row and head, to BF16 and to
// the MXINT8 copy.
__device__ __forceinline__ void write_block(const AttnJob& j, uint64_t row, uint32_t head,
                                            uint32_t b, uint32_t lane, float x,
                                            uint32_t* error_flag) {
  const uint32_t col = head * j.cache.hd + 32u * b + lane;
  if (j.out != nullptr) j.out[row * j.ldo + col] = attn_bf16(x);
  if (j.oq == nullptr) return;
  const uint32_t bits = __float_as_uint(x), mag = bits & 0x7FFFFFFFu;
  const uint32_t key = __reduce_max_sync(0xFFFFFFFFu, j.vec_rule ? mag >> 23 : mag);
  uint32_t scale;
  const int32_t code = mxint8_code(bits, key, j.vec_rule != 0, scale);
  j.oq[row * j.ldoq + col] = static_cast<int8_t>(code);
  if (lane == 0u) j.oscale[row * (j.ldoq / 32u) + col / 32u] = static_cast<uint8_t>(scale);
  if (mag >= 0x7F800000u && !j.vec_rule) atomicOr(error_flag, 1u);
}

// The same for 32 dims (block b) in one thread.
__device__ __forceinline__ void write_row_block(const AttnJob& j, uint64_t row, uint32_t head,
                                                uint32_t b, const float (&x)[32],
                                                uint32_t* error_flag) {
  const uint64_t col = static_cast<uint64_t>(head) * j.cache.hd + 32u * b;
  if (j.out != nullptr) {
    uint4* to = reinterpret_cast<uint4*>(j.out + row * j.ldo + col);
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
      uint32_t w[4];
#pragma unroll
      for (uint32_t d = 0; d < 4u; ++d) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;"
            : "=r"(w[d])
            : "f"(x[8u * i + 2u * d + 1u]), "f"(x[8u * i + 2u * d]));
      }
      to[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (j.oq == nullptr) return;
  uint32_t top = 0;
#pragma unroll
  for (uint32_t i = 0; i < 32u; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  const uint32_t key = j.vec_rule ? top >> 23 : top;
  uint32_t scale = 0, w[8];
#pragma unroll
  for (uint32_t i = 0; i < 8u; ++i) {
    w[i] = 0;
#pragma unroll
    for (uint32_t d = 0; d < 4u; ++d) {
      const int32_t code = mxint8_code(__float_as_uint(x[4u * i + d]), key, j.vec_rule != 0, scale);
      w[i] |= (static_cast<uint32_t>(code) & 0xFFu) << (8u * d);
    }
  }
  uint4* to = reinterpret_cast<uint4*>(j.oq + row * j.ldoq + col);
  to[0] = make_uint4(w[0], w[1], w[2], w[3]);
  to[1] = make_uint4(w[4], w[5], w[6], w[7]);
  j.oscale[row * (j.ldoq / 32u) + col / 32u] = static_cast<uint8_t>(scale);
  if (top >= 0x7F800000u && !j.vec_rule) atomicOr(error_flag, 1u);
}

}  // namespace hrb
