// hrb_qkv_append: the rows of the QKV Linear to the query operand and the
// 4-bit cache, and hrb_kv_read, the way back.
//
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w          q and k heads
//   (y_a, y_b) = (y_a c - y_b s, y_b c + y_a s)      pairs of the first rot dims
//   q -> BF16;  k, v -> 32-dim blocks, e = floor(log2 max) - 2, E2M1(y / 2^e)
//
// k_qkv: a lane holds four consecutive dims of a head, so a head is hd / 4
// lanes (a warp holds 1, 2 or 4 heads at a time) and a 32-dim block 8 lanes:
// the mean takes log2(hd / 4) shuffles, the block maximum three.  A half-split pair's
// other dim is at the same place of the lane rot / 8 away, one shuffle each.
// A warp takes one token and up to kSteps times its heads: the token's
// position, slot and cos/sin pairs are read once for them, and all their
// rows are loaded before the first is used.
//
// Memory bound: each input is read once (FP32: 4 bytes a value, BF16: 2),
// and per token heads * hd BF16 values and kv_heads * (hd + hd / 16) bytes
// are written.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "hrb_serve.cuh"

namespace hrb {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kSteps = 4;  // heads a lane holds at once

__device__ __forceinline__ float bf16_bits(uint32_t bits) { return __uint_as_float(bits << 16); }

// Four consecutive values of a row.
template <bool BF16, bool VEC>
__device__ __forceinline__ float4 load4(const void* base, uint64_t at) {
  if constexpr (BF16) {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    if constexpr (VEC) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
      return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u),
                         __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u));
    } else {
      return make_float4(bf16_bits(__ldg(p)), bf16_bits(__ldg(p + 1)), bf16_bits(__ldg(p + 2)),
                         bf16_bits(__ldg(p + 3)));
    }
  } else {
    const float* p = static_cast<const float*>(base) + at;
    if constexpr (VEC) {
      return __ldg(reinterpret_cast<const float4*>(p));
    } else {
      return make_float4(__ldg(p), __ldg(p + 1), __ldg(p + 2), __ldg(p + 3));
    }
  }
}

template <uint32_t HD, bool BF16, bool VEC>
__global__ void __launch_bounds__(kWarps * 32)
    k_qkv(const QkvJob j, uint32_t chunks, uint32_t steps, uint32_t* __restrict__ error_flag) {
  constexpr uint32_t kLanes = HD / 4u;                        // lanes a head (24 at hd 96)
  constexpr uint32_t kSpan = HD == 96u ? 32u : kLanes;        // lanes set apart for a head
  constexpr uint32_t kHeads = 32u / kSpan;                    // heads a warp holds
  const uint32_t lane = threadIdx.x & 31u, sub = lane / kSpan, l = lane % kSpan;
  const bool on = l < kLanes;
  const uint64_t unit = static_cast<uint64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (unit >= static_cast<uint64_t>(j.tokens) * chunks) return;
  const uint32_t t = static_cast<uint32_t>(unit / chunks);
  const uint32_t h0 = static_cast<uint32_t>(unit % chunks) * steps * kHeads + sub;
  const uint32_t qk = j.heads + j.cache.kv_heads, all = qk + j.cache.kv_heads;
  // All rows of this warp, in flight together.
  float4 x[kSteps];
#pragma unroll
  for (uint32_t u = 0; u < kSteps; ++u) {
    const uint32_t h = h0 + u * kHeads;
    x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (u < steps && h < all && on) {
      const uint32_t which = h < j.heads ? 0u : h < qk ? 1u : 2u;
      const uint32_t hh = which == 0u ? h : which == 1u ? h - j.heads : h - qk;
      x[u] = load4<BF16, VEC>(j.x[which], t * j.ld[which] + hh * HD + 4u * l);
    }
  }
  // The lane's four (cos, sin): half-split dims d use pair d mod half,
  // interleaved dims 2p and 2p + 1 pair p.
  bool bad_slot = false, non_finite = false;
  float2 cs[4];
  const bool turns = j.rope != nullptr && 4u * l < 2u * j.half && on;
#pragma unroll
  for (uint32_t i = 0; i < 4u; ++i) cs[i] = make_float2(1.f, 0.f);
  if (turns) {
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
      const uint32_t d = 4u * l + i;
      if (j.interleaved && (i & 1u)) {
        cs[i] = cs[i - 1u];
        continue;
      }
      const uint32_t p = j.interleaved ? d / 2u : d < j.half ? d : d - j.half;
      const uint32_t axis = (p >= j.cut[0] ? 1u : 0u) + (p >= j.cut[1] ? 1u : 0u);
      const int32_t pos = __ldg(j.pos + static_cast<uint64_t>(axis) * j.tokens + t);
      if (pos >= 0 && static_cast<uint32_t>(pos) < j.max_pos) {
        cs[i] = __ldg(j.rope + static_cast<uint64_t>(pos) * j.half + p);
      } else {
        bad_slot = true;
      }
    }
  }
  const int32_t slot = __ldg(j.slots + t);
  const bool cached = slot >= 0 &&
                      (static_cast<uint32_t>(slot) >> j.cache.page_log2) < j.cache.pages;
  bad_slot |= slot >= 0 && !cached;
#pragma unroll
  for (uint32_t u = 0; u < kSteps; ++u) {
    const uint32_t h = h0 + u * kHeads;
    if (u >= steps || h0 - sub + u * kHeads >= all) break;  // the same for the whole warp
    const bool mine = h < all && on;
    const uint32_t which = h < j.heads ? 0u : h < qk ? 1u : 2u;
    float y[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
    const float* w = which < 2u ? j.norm[which] : nullptr;
    float ss = y[0] * y[0] + y[1] * y[1] + y[2] * y[2] + y[3] * y[3];
#pragma unroll
    for (uint32_t d = kSpan / 2u; d > 0; d /= 2u) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
    if (w != nullptr && mine) {
      const float r = 1.0f / sqrtf(__fdiv_rn(ss, static_cast<float>(HD)) + j.eps);
      const float* wl = w + 4u * l;
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) y[i] = __fmul_rn(__fmul_rn(y[i], r), __ldg(wl + i));
    }
    if (j.rope != nullptr) {
      float z[4];
      if (j.interleaved) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; i += 2u) {
          z[i] = __fsub_rn(__fmul_rn(y[i], cs[i].x), __fmul_rn(y[i + 1u], cs[i].y));
          z[i + 1u] = __fadd_rn(__fmul_rn(y[i + 1u], cs[i].x), __fmul_rn(y[i], cs[i].y));
        }
      } else {
        const bool first = 4u * l < j.half;
        const uint32_t other = first ? l + j.half / 4u : l - j.half / 4u;
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
          const float o = __shfl_sync(0xFFFFFFFFu, y[i], sub * kSpan + (other & (kSpan - 1u)));
          const float a = __fmul_rn(y[i], cs[i].x), b = __fmul_rn(o, cs[i].y);
          z[i] = first ? __fsub_rn(a, b) : __fadd_rn(a, b);
        }
      }
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) y[i] = turns && which < 2u ? z[i] : y[i];
    }
    if (which == 0u) {
      if (mine) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(y[0], y[1]);
        const __nv_bfloat162 b = __floats2bfloat162_rn(y[2], y[3]);
        uint2 v;
        v.x = *reinterpret_cast<const uint32_t*>(&a);
        v.y = *reinterpret_cast<const uint32_t*>(&b);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(j.q_out) + t * j.ldqo +
                                  static_cast<uint64_t>(h) * HD + 4u * l) = v;
      }
    }
    if (__all_sync(0xFFFFFFFFu, which == 0u)) continue;
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
      const uint32_t mag = __float_as_uint(y[i]) & 0x7FFFFFFFu;
      if (which != 0u && mag >= 0x7F800000u) {
        non_finite = true;
        if (mag > 0x7F800000u) y[i] = 0.f;
      }
      top = max(top, __float_as_uint(y[i]) & 0x7FFFFFFFu);
    }
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
    if (which == 0u || !mine || !cached) continue;
    const int32_t e = kv_block_exp(top);
    const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    const uint32_t codes = e2m1_pair(y[0] * inv, y[1] * inv) |
                           (e2m1_pair(y[2] * inv, y[3] * inv) << 8);
    const uint32_t in_page = static_cast<uint32_t>(slot) & (j.cache.page - 1u);
    uint8_t* rec = kv_record(j.cache, static_cast<uint32_t>(slot) >> j.cache.page_log2,
                             which == 1u ? h - j.heads : h - qk) +
                   (which == 1u ? 0u : kv_vcodes(j.cache));
    *reinterpret_cast<uint16_t*>(rec + in_page * (HD / 2u) + 2u * l) =
        static_cast<uint16_t>(codes);
    if ((l & 7u) == 0u) {
      rec[kv_kscales(j.cache) + in_page * (HD / 32u) + l / 8u] = static_cast<uint8_t>(e + 127);
    }
  }
  const uint32_t err = (bad_slot ? kErrKvSlot : 0u) | (non_finite ? kErrKvNonFinite : 0u);
  if (err != 0u) atomicOr(error_flag, err);
}

// A thread reads eight dims (one word of codes) of K and of V.
__global__ void __launch_bounds__(256)
    k_kv_read(const KvCache c, const int32_t* __restrict__ slots, uint32_t tokens, uint32_t dtype,
              void* k, void* v, uint32_t* __restrict__ error_flag) {
  const uint32_t words = c.hd / 8u, row = c.kv_heads * words;
  const uint64_t n = static_cast<uint64_t>(tokens) * row;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * blockDim.x;
  bool bad = false;
  for (uint64_t at = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; at < n;
       at += step) {
    const uint32_t t = static_cast<uint32_t>(at / row), i = static_cast<uint32_t>(at % row);
    const uint32_t head = i / words, w = i % words;
    const int32_t slot = __ldg(slots + t);
    const uint32_t page = static_cast<uint32_t>(slot) >> c.page_log2;
    const bool there = slot >= 0 && page < c.pages;
    bad |= slot >= 0 && !there;
#pragma unroll
    for (uint32_t part = 0; part < 2u; ++part) {
      void* out = part == 0u ? k : v;
      if (out == nullptr) continue;
      uint32_t h[4] = {0, 0, 0, 0};
      float scale = 0.f;
      if (there) {
        const uint32_t in_page = static_cast<uint32_t>(slot) & (c.page - 1u);
        const uint8_t* rec = kv_record(c, page, head) + (part == 0u ? 0u : kv_vcodes(c));
        const uint32_t codes =
            *reinterpret_cast<const uint32_t*>(rec + in_page * (c.hd / 2u) + 4u * w);
        scale = kv_scale(rec[kv_kscales(c) + in_page * (c.hd / 32u) + w / 4u]);
        e2m1x8_to_f16x2(codes, h);
      }
      float f[8];
#pragma unroll
      for (uint32_t b = 0; b < 4u; ++b) {
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&h[b]));
        f[2u * b] = p.x * scale;
        f[2u * b + 1u] = p.y * scale;
      }
      const uint64_t o = at * 8u;
      if (dtype == HRB_DT_F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + o);
        p[0] = make_float4(f[0], f[1], f[2], f[3]);
        p[1] = make_float4(f[4], f[5], f[6], f[7]);
      } else if (dtype == HRB_DT_BF16) {
        uint32_t r[4];
#pragma unroll
        for (uint32_t b = 0; b < 4u; ++b) {
          const __nv_bfloat162 p = __floats2bfloat162_rn(f[2u * b], f[2u * b + 1u]);
          r[b] = *reinterpret_cast<const uint32_t*>(&p);
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + o) =
            make_uint4(r[0], r[1], r[2], r[3]);
      } else {
        uint32_t r[4];
#pragma unroll
        for (uint32_t b = 0; b < 4u; ++b) {
          uint16_t two;
          asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;"
              : "=h"(two)
              : "f"(f[2u * b + 1u]), "f"(f[2u * b]));
          r[b] = two;
        }
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(out) + o) =
            make_uint2(r[0] | (r[1] << 16), r[2] | (r[3] << 16));
      }
    }
  }
  if (bad) atomicOr(error_flag, kErrKvSlot);
}

template <uint32_t HD>
void launch_hd(const QkvJob& job, bool bf16, bool vec, uint32_t* err, int sm_count,
               cudaStream_t stream) {
  constexpr uint32_t kHeads = HD == 32u ? 4u : HD == 64u ? 2u : 1u;
  const uint32_t rows = (job.heads + 2u * job.cache.kv_heads + kHeads - 1u) / kHeads;
  // One head step a warp while that does not fill the GPU.
  const uint64_t fill = static_cast<uint64_t>(sm_count) * 32u;
  const uint32_t steps = static_cast<uint64_t>(job.tokens) * rows > fill ? kSteps : 1u;
  const uint32_t chunks = (rows + steps - 1u) / steps;
  const uint64_t units = static_cast<uint64_t>(job.tokens) * chunks;
  const unsigned grid = static_cast<unsigned>((units + kWarps - 1u) / kWarps);
  if (bf16) {
    if (vec) k_qkv<HD, true, true><<<grid, kWarps * 32, 0, stream>>>(job, chunks, steps, err);
    else k_qkv<HD, true, false><<<grid, kWarps * 32, 0, stream>>>(job, chunks, steps, err);
  } else {
    if (vec) k_qkv<HD, false, true><<<grid, kWarps * 32, 0, stream>>>(job, chunks, steps, err);
    else k_qkv<HD, false, false><<<grid, kWarps * 32, 0, stream>>>(job, chunks, steps, err);
  }
}

}  // namespace

void launch_qkv_append(const QkvJob& job, bool bf16, bool vec, uint32_t* error_flag, int sm_count,
                       cudaStream_t stream) {
  switch (job.cache.hd) {
    case 32: launch_hd<32>(job, bf16, vec, error_flag, sm_count, stream); break;
    case 64: launch_hd<64>(job, bf16, vec, error_flag, sm_count, stream); break;
    case 96: launch_hd<96>(job, bf16, vec, error_flag, sm_count, stream); break;
    default: launch_hd<128>(job, bf16, vec, error_flag, sm_count, stream); break;
  }
}

void launch_kv_read(const KvCache& cache, const int32_t* slots, uint32_t tokens, uint32_t dtype,
                    void* k, void* v, uint32_t* error_flag, int sm_count, cudaStream_t stream) {
  const uint64_t n = static_cast<uint64_t>(tokens) * cache.kv_heads * (cache.hd / 8u);
  const uint64_t blocks = (n + 255u) / 256u, most = static_cast<uint64_t>(sm_count) * 16u;
  k_kv_read<<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, stream>>>(
      cache, slots, tokens, dtype, k, v, error_flag);
}

}  // namespace hrb
