// hrb_qkv_append: the rows of the QKV Linear to the query operand and the
// 4-bit cache, and hrb_kv_read, the way back.
//
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w          q and k heads
//   (y_a, y_b) = (y_a c - y_b s, y_b c + y_a s)      pairs of the first rot dims
//   q -> BF16;  k, v -> 32-dim blocks, e = floor(log2 max) - 2, E2M1(y / 2^e)
//
// k_qkv: a head is hd / 8 lanes (12 of 16 at hd = 96), a warp holds 8, 4 or
// 2 heads at a time; a lane has the four dims 4l .. 4l + 3 and the four hd / 2
// further, so that the pairs of a whole half-split rotation meet in a lane
// and need no shuffle (those of a partial one take two a dim).  A warp takes
// a token and a run of its heads, in steps that are all of q, of k or of v:
// the token's position, slot and cos/sin pairs are read once for them, and
// four steps' rows are in flight together.  With eight dims a lane the sums
// and maxima over a head cost half the shuffles of four.
//
// Memory bound: each input is read once (FP32: 4 bytes a value, BF16: 2),
// and per token heads * hd BF16 values and kv_heads * (hd + hd / 16) bytes
// are written.  Measured: 16387 tokens of 32/8 heads of 128 (BF16, three
// axes) 81 to 83 us with the read-back, 4.8 to 4.9 TB/s, 73 to 75 % of a copy's
// rate; k_qkv alone uses DRAM to 53 % and the issue slots to 57 %.  With rsqrtf where the norm divides by a square root
// (two units in the last place), packed FP32 pairs, and rows in phases of q,
// k and v it takes 43 M warp instructions, against 199 M for a lane of four
// dims with one code path for all three.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "hrb_attn.cuh"
#include "hrb_kernels.cuh"
#include "sm100.cuh"

namespace hrb {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kAhead = 4;  // steps whose rows are in flight

__device__ __forceinline__ float bf16_bits(uint32_t bits) { return __uint_as_float(bits << 16); }

// Four consecutive values of a row, as they are (BF16: two words).
template <bool BF16, bool VEC>
__device__ __forceinline__ uint4 load4(const void* base, uint64_t at) {
  if constexpr (BF16) {
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    if constexpr (VEC) {
      const uint2 v = ld(reinterpret_cast<const uint2*>(p));
      return make_uint4(v.x, v.y, 0, 0);
    } else {
      return make_uint4(ld(p) | (static_cast<uint32_t>(ld(p + 1)) << 16),
                        ld(p + 2) | (static_cast<uint32_t>(ld(p + 3)) << 16), 0, 0);
    }
  } else {
    const uint32_t* p = static_cast<const uint32_t*>(base) + at;
    if constexpr (VEC) {
      return ld(reinterpret_cast<const uint4*>(p));
    } else {
      return make_uint4(ld(p), ld(p + 1), ld(p + 2), ld(p + 3));
    }
  }
}
template <bool BF16>
__device__ __forceinline__ void values4(const uint4& v, float* y) {
  if constexpr (BF16) {
    y[0] = bf16_bits(v.x);
    y[1] = __uint_as_float(v.x & 0xFFFF0000u);
    y[2] = bf16_bits(v.y);
    y[3] = __uint_as_float(v.y & 0xFFFF0000u);
  } else {
    y[0] = __uint_as_float(v.x);
    y[1] = __uint_as_float(v.y);
    y[2] = __uint_as_float(v.z);
    y[3] = __uint_as_float(v.w);
  }
}

template <uint32_t W>
struct Which {
  static constexpr uint32_t value = W;
};

// Where a warp's run of steps lies: q, k and v steps of a token in order.
struct Steps {
  uint32_t q, k, all;  // steps of q, of q and k, of all three
  uint32_t run;        // a warp's
  uint32_t runs;       // a token's
};

template <uint32_t HD, bool BF16, bool VEC>
__global__ void __launch_bounds__(kWarps * 32, BF16 ? 7 : 6)
    k_qkv(const QkvJob j, const Steps st, uint32_t* __restrict__ error_flag) {
  constexpr uint32_t kLanes = HD / 8u;                  // lanes a head
  constexpr uint32_t kSpan = HD == 96u ? 16u : kLanes;  // lanes set apart for one
  constexpr uint32_t kHeads = 32u / kSpan;              // heads a step
  const uint32_t lane = threadIdx.x & 31u, sub = lane / kSpan, l = lane % kSpan;
  const bool on = l < kLanes;
  // Runs of a token only split small calls: their number fits 32 bits.
  const uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit >= j.tokens * st.runs) return;
  const uint32_t t = unit / st.runs;
  const uint32_t begin = (unit - t * st.runs) * st.run;
  const uint32_t end = min(begin + st.run, st.all);
  bool non_finite = false;
  sm100::griddep_wait();

  // The lane's cos and sin, of its dims 4l + i (c = 0) and hd / 2 further
  // (c = 1): half-split dims d use pair d mod half, interleaved dims 2p and
  // 2p + 1 pair p.  Sines are negated where they multiply a pair's second.
  const bool paired = !j.interleaved && 2u * j.half == HD;  // pairs meet in the lane
  float co[2][4], si[2][4];
#pragma unroll
  for (uint32_t i = 0; i < 4u; ++i) {
    co[0][i] = co[1][i] = 1.f;
    si[0][i] = si[1][i] = 0.f;
  }
  // A token with a position outside the table, on an axis that has pairs, is
  // neither rotated nor cached.
  bool bad_pos = false;
  if (j.rope != nullptr) {
    const int32_t p0 = j.cut[0] > 0u ? ld(j.pos + t) : 0;
    const int32_t p1 = j.cut[0] < j.cut[1] ? ld(j.pos + j.tokens + t) : 0;
    const int32_t p2 = j.cut[1] < j.half ? ld(j.pos + 2ull * j.tokens + t) : 0;
    bad_pos = max(max(static_cast<uint32_t>(p0), static_cast<uint32_t>(p1)),
                  static_cast<uint32_t>(p2)) >= j.max_pos;
#pragma unroll
    for (uint32_t c = 0; c < 2u; ++c) {
      if (bad_pos || begin >= st.k) break;
      if (c == 1u && paired) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
          co[1][i] = co[0][i];
          si[1][i] = si[0][i];
        }
        continue;
      }
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) {
        const uint32_t d = 4u * l + c * (HD / 2u) + i;
        if (d >= 2u * j.half || !on) continue;
        if (j.interleaved && (i & 1u)) {
          co[c][i] = co[c][i - 1u];
          si[c][i] = si[c][i - 1u];
          continue;
        }
        const uint32_t p = j.interleaved ? d / 2u : d < j.half ? d : d - j.half;
        const int32_t pos = p < j.cut[0] ? p0 : p < j.cut[1] ? p1 : p2;
        const float2 v = ld(j.rope + static_cast<uint64_t>(static_cast<uint32_t>(pos)) * j.half + p);
        co[c][i] = v.x;
        si[c][i] = v.y;
      }
    }
  }
  const int32_t slot = ld(j.slots + t);
  const bool in_cache = slot >= 0 &&
                        (static_cast<uint32_t>(slot) >> j.cache.page_log2) < j.cache.pages;
  const bool cached = in_cache && !bad_pos;
  const bool bad_slot = bad_pos || (slot >= 0 && !in_cache);

  // Steps [begin, end) of q (W = 0), k (1) or v (2): numbers a .. b of its own.
  auto phase = [&](auto which, uint32_t a, uint32_t b) {
    constexpr uint32_t W = decltype(which)::value;
    if (a >= b) return;
    const uint32_t count = W == 0u ? j.heads : j.cache.kv_heads;
    uint32_t h = a * kHeads + sub;
    uint64_t at = t * j.ld[W] + h * HD + 4u * l;
    float w[2][4];
    const bool norm = W < 2u && j.norm[W < 2u ? W : 0u] != nullptr;
#pragma unroll
    for (uint32_t c = 0; c < 2u; ++c)
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) {
        w[c][i] = norm && on ? ld(j.norm[W < 2u ? W : 0u] + 4u * l + c * (HD / 2u) + i) : 0.f;
      }
    uint16_t* to = W == 0u ? static_cast<uint16_t*>(j.q_out) + t * j.ldqo + h * HD + 4u * l : nullptr;
    uint8_t* rec = nullptr;
    if (W != 0u && cached) {
      rec = kv_record(j.cache, static_cast<uint32_t>(slot) >> j.cache.page_log2, h) +
            (W == 1u ? 0u : kv_vcodes(j.cache)) +
            (static_cast<uint32_t>(slot) & (j.cache.page - 1u)) * (HD / 2u) + 2u * l;
    }
    // From a lane's codes to its block's scale byte.
    const uint32_t scales = W == 0u ? 0u
        : kv_kscales(j.cache) - (static_cast<uint32_t>(slot) & (j.cache.page - 1u)) * (HD / 2u - HD / 32u) - 2u * l;
    for (uint32_t s = a; s < b; s += kAhead) {
      uint4 raw[kAhead][2];
#pragma unroll
      for (uint32_t u = 0; u < kAhead; ++u) {
        raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);
        if (s + u < b && on && h + u * kHeads < count) {
          raw[u][0] = load4<BF16, VEC>(j.x[W], at + u * (kHeads * HD));
          raw[u][1] = load4<BF16, VEC>(j.x[W], at + u * (kHeads * HD) + HD / 2u);
        }
      }
#pragma unroll
      for (uint32_t u = 0; u < kAhead; ++u) {
        if (s + u >= b) break;  // the same for the whole warp
        const bool mine = on && h + u * kHeads < count;
        float y[2][4];
        values4<BF16>(raw[u][0], y[0]);
        values4<BF16>(raw[u][1], y[1]);
        if constexpr (W < 2u) {
          if (norm) {
            uint64_t sq = 0;
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c)
#pragma unroll
              for (uint32_t i = 0; i < 4u; i += 2u) {
                const uint64_t v = pack2(y[c][i], y[c][i + 1u]);
                sq = fma_2(v, v, sq);
              }
            float ss = unpack2(sq).x + unpack2(sq).y;
#pragma unroll
            for (uint32_t d = kSpan / 2u; d > 0; d /= 2u) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
            const float r = rsqrtf(ss * (1.0f / HD) + j.eps);
            const uint64_t rr = pack2(r, r);
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c)
#pragma unroll
              for (uint32_t i = 0; i < 4u; i += 2u) {
                const float2 v = unpack2(mul_2(mul_2(pack2(y[c][i], y[c][i + 1u]), rr),
                                               pack2(w[c][i], w[c][i + 1u])));
                y[c][i] = v.x;
                y[c][i + 1u] = v.y;
              }
          }
          if (paired) {
#pragma unroll
            for (uint32_t i = 0; i < 4u; i += 2u) {
              const uint64_t va = pack2(y[0][i], y[0][i + 1u]), vb = pack2(y[1][i], y[1][i + 1u]);
              const uint64_t c2 = pack2(co[0][i], co[0][i + 1u]);
              const uint64_t s2 = pack2(si[0][i], si[0][i + 1u]);
              const uint64_t n2 = pack2(-si[0][i], -si[0][i + 1u]);
              const float2 x = unpack2(add_2(mul_2(va, c2), mul_2(vb, n2)));
              const float2 z = unpack2(add_2(mul_2(vb, c2), mul_2(va, s2)));
              y[0][i] = x.x;
              y[0][i + 1u] = x.y;
              y[1][i] = z.x;
              y[1][i + 1u] = z.y;
            }
          } else if (j.interleaved) {
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c)
#pragma unroll
              for (uint32_t i = 0; i < 4u; i += 2u) {
                const float p = y[c][i], q = y[c][i + 1u];
                y[c][i] = __fsub_rn(__fmul_rn(p, co[c][i]), __fmul_rn(q, si[c][i]));
                y[c][i + 1u] = __fadd_rn(__fmul_rn(q, co[c][i]), __fmul_rn(p, si[c][i]));
              }
          } else if (j.half != 0u) {
            // Fours of dims: number f is slot f / kLanes of lane f % kLanes.
            float z[2][4];
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c) {
              const uint32_t f = l + c * kLanes, hf = j.half / 4u;
              const bool low = f < hf;
              const uint32_t from = low ? f + hf : f - hf;
              const uint32_t lane_of = (sub * kSpan + from % kLanes) & 31u;
#pragma unroll
              for (uint32_t i = 0; i < 4u; ++i) {
                const float o0 = __shfl_sync(0xFFFFFFFFu, y[0][i], lane_of);
                const float o1 = __shfl_sync(0xFFFFFFFFu, y[1][i], lane_of);
                const float p = __fmul_rn(y[c][i], co[c][i]);
                const float q = __fmul_rn(from < kLanes ? o0 : o1, si[c][i]);
                z[c][i] = f >= 2u * hf ? y[c][i] : low ? __fsub_rn(p, q) : __fadd_rn(p, q);
              }
            }
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c)
#pragma unroll
              for (uint32_t i = 0; i < 4u; ++i) y[c][i] = z[c][i];
          }
        }
        if constexpr (W == 0u) {
          if (mine) {
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c) {
              const __nv_bfloat162 p = __floats2bfloat162_rn(y[c][0], y[c][1]);
              const __nv_bfloat162 q = __floats2bfloat162_rn(y[c][2], y[c][3]);
              *reinterpret_cast<uint2*>(to + u * (kHeads * HD) + c * (HD / 2u)) = make_uint2(
                  *reinterpret_cast<const uint32_t*>(&p), *reinterpret_cast<const uint32_t*>(&q));
            }
          }
        } else {
          uint32_t top[2];
#pragma unroll
          for (uint32_t c = 0; c < 2u; ++c) {
            top[c] = __float_as_uint(fmaxf(fmaxf(fabsf(y[c][0]), fabsf(y[c][1])),
                                           fmaxf(fabsf(y[c][2]), fabsf(y[c][3]))));
          }
          // fmaxf passes NaNs over: a sum of the values' products with zero does not.
          float odd = 0.f;
#pragma unroll
          for (uint32_t c = 0; c < 2u; ++c)
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) odd = fmaf(y[c][i], 0.f, odd);
          if (odd != odd) {  // rare: NaN counts as zero, Inf saturates
            non_finite |= mine && cached;  // rows that pad a step may hold anything
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c)
#pragma unroll
              for (uint32_t i = 0; i < 4u; ++i) {
                if (y[c][i] != y[c][i]) y[c][i] = 0.f;
              }
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c) {
              top[c] = __float_as_uint(fmaxf(fmaxf(fabsf(y[c][0]), fabsf(y[c][1])),
                                             fmaxf(fabsf(y[c][2]), fabsf(y[c][3]))));
            }
          }
          uint32_t block[2];  // the blocks that the lane's fours lie in
          if constexpr (HD == 96u) {
            uint32_t all[3];
#pragma unroll
            for (uint32_t k = 0; k < 3u; ++k) {
              all[k] = max(l / 8u == k ? top[0] : 0u, (l + kLanes) / 8u == k ? top[1] : 0u);
#pragma unroll
              for (uint32_t d = 8; d > 0; d /= 2u) {
                all[k] = max(all[k], __shfl_xor_sync(0xFFFFFFFFu, all[k], d));
              }
            }
            block[0] = l / 8u;
            block[1] = min((l + kLanes) / 8u, 2u);
            top[0] = block[0] == 0u ? all[0] : all[1];
            top[1] = block[1] == 1u ? all[1] : all[2];
          } else if constexpr (HD == 32u) {
            block[0] = block[1] = 0u;
            top[0] = max(top[0], top[1]);
            top[0] = max(top[0], __shfl_xor_sync(0xFFFFFFFFu, top[0], 1));
            top[0] = max(top[0], __shfl_xor_sync(0xFFFFFFFFu, top[0], 2));
            top[1] = top[0];
          } else {
            block[0] = l / 8u;
            block[1] = HD / 64u + l / 8u;
#pragma unroll
            for (uint32_t d = 1; d < 8u; d *= 2u) {
              top[0] = max(top[0], __shfl_xor_sync(0xFFFFFFFFu, top[0], d));
              top[1] = max(top[1], __shfl_xor_sync(0xFFFFFFFFu, top[1], d));
            }
          }
          if (mine && cached) {
            uint8_t* r8 = rec + static_cast<uint64_t>(u * kHeads) * j.cache.record;
#pragma unroll
            for (uint32_t c = 0; c < 2u; ++c) {
              const int32_t e = kv_block_exp(top[c]);
              const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
              const uint32_t codes = e2m1_pair(y[c][0] * inv, y[c][1] * inv) |
                                     (e2m1_pair(y[c][2] * inv, y[c][3] * inv) << 8);
              *reinterpret_cast<uint16_t*>(r8 + c * (HD / 4u)) = static_cast<uint16_t>(codes);
              if ((l + c * kLanes) % 8u == 0u) {
                r8[static_cast<int64_t>(static_cast<int32_t>(scales)) + block[c]] = static_cast<uint8_t>(e + 127);
              }
            }
          }
        }
      }
      h += kAhead * kHeads;
      at += kAhead * kHeads * HD;
      if (W == 0u) to += kAhead * kHeads * HD;
      if (W != 0u && cached) rec += static_cast<uint64_t>(kAhead * kHeads) * j.cache.record;
    }
  };
  phase(Which<0>{}, min(begin, st.q), min(end, st.q));
  phase(Which<1>{}, max(begin, st.q) - st.q, min(max(end, st.q), st.k) - st.q);
  phase(Which<2>{}, max(begin, st.k) - st.k, max(end, st.k) - st.k);
  const uint32_t err = (bad_slot ? kErrKvSlot : 0u) | (non_finite ? kErrKvNonFinite : 0u);
  if (err != 0u) atomicOr(error_flag, err);
}

// Sixteen dims (two words of codes) of K and of V a step; a block takes
// kTokens tokens.  Values are exact in FP16, and from there in each type.
constexpr uint32_t kTokens = 8;

template <uint32_t DT>
__device__ __forceinline__ void put16(void* out, uint64_t at, const uint32_t (&h)[8]) {
  if constexpr (DT == HRB_DT_E5M2) {
    uint32_t r[4];
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
      uint16_t a, b;
      asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(a) : "r"(h[2u * i]));
      asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(b) : "r"(h[2u * i + 1u]));
      r[i] = a | (static_cast<uint32_t>(b) << 16);
    }
    *reinterpret_cast<uint4*>(static_cast<uint8_t*>(out) + at) = make_uint4(r[0], r[1], r[2], r[3]);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i) {
      float2 f[4];
#pragma unroll
      for (uint32_t d = 0; d < 4u; ++d) f[d] = __half22float2(*reinterpret_cast<const __half2*>(&h[4u * i + d]));
      if constexpr (DT == HRB_DT_F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(out) + at + 8u * i);
        p[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
        p[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
      } else {
        uint32_t r[4];
#pragma unroll
        for (uint32_t d = 0; d < 4u; ++d) {
          const __nv_bfloat162 p = __floats2bfloat162_rn(f[d].x, f[d].y);
          r[d] = *reinterpret_cast<const uint32_t*>(&p);
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at + 8u * i) =
            make_uint4(r[0], r[1], r[2], r[3]);
      }
    }
  }
}

template <uint32_t DT>
__global__ void __launch_bounds__(256)
    k_kv_read(const KvCache c, const int32_t* slots, uint32_t tokens, FastDiv row_div,
              FastDiv head_div, void* k, void* v, uint32_t* __restrict__ error_flag) {
  const uint32_t t0 = blockIdx.x * kTokens, n = min(kTokens, tokens - t0) * row_div.d;
  bool bad = false;
  sm100::griddep_wait();
  for (uint32_t i = threadIdx.x; i < n; i += 256u) {
    const uint32_t t = fast_div(i, row_div), x = i - t * row_div.d;
    const uint32_t head = fast_div(x, head_div), w = x - head * head_div.d;
    const int32_t slot = ld(slots + t0 + t);
    const uint32_t page = static_cast<uint32_t>(slot) >> c.page_log2;
    const bool there = slot >= 0 && page < c.pages;
    bad |= slot >= 0 && !there;
    uint2 codes[2] = {make_uint2(0, 0), make_uint2(0, 0)};
    uint32_t scale[2] = {127u, 127u};
    if (there) {
      const uint32_t in_page = static_cast<uint32_t>(slot) & (c.page - 1u);
      const uint8_t* rec = kv_record(c, page, head);
#pragma unroll
      for (uint32_t p = 0; p < 2u; ++p) {
        const uint8_t* part = rec + (p == 0u ? 0u : kv_vcodes(c));
        codes[p] = *reinterpret_cast<const uint2*>(part + in_page * (c.hd / 2u) + 8u * w);
        scale[p] = part[kv_kscales(c) + in_page * (c.hd / 32u) + w / 2u];
      }
    }
    const uint64_t at = (static_cast<uint64_t>(t0 + t) * row_div.d + x) * 16u;
#pragma unroll
    for (uint32_t p = 0; p < 2u; ++p) {
      void* out = p == 0u ? k : v;
      if (out == nullptr) continue;
      uint32_t a[4], b[4], h[8];
      e2m1x8_to_f16x2(codes[p].x, a);
      e2m1x8_to_f16x2(codes[p].y, b);
      const uint32_t sc = scale2(scale[p], scale[p]);
#pragma unroll
      for (uint32_t d = 0; d < 4u; ++d) {
        h[d] = mul2(a[d], sc);
        h[4u + d] = mul2(b[d], sc);
      }
      put16<DT>(out, at, h);
    }
  }
  if (bad) atomicOr(error_flag, kErrKvSlot);
}

template <uint32_t HD>
void launch_hd(const QkvJob& job, bool bf16, bool vec, uint32_t* err, int sm_count,
               cudaStream_t stream) {
  constexpr uint32_t kHeads = 32u / (HD == 96u ? 16u : HD / 8u);
  Steps st;
  st.q = (job.heads + kHeads - 1u) / kHeads;
  const uint32_t kv = (job.cache.kv_heads + kHeads - 1u) / kHeads;
  st.k = st.q + kv;
  st.all = st.k + kv;
  // A warp takes as many steps as leave two warps a scheduler, in whole
  // loads of kAhead where that is more.
  const uint64_t warps = static_cast<uint64_t>(sm_count) * 8u;
  const uint64_t run = static_cast<uint64_t>(job.tokens) * st.all / warps;
  st.run = run < 1u ? 1u : run < st.all ? static_cast<uint32_t>(run) : st.all;
  if (st.run > kAhead) st.run = (st.run + kAhead - 1u) / kAhead * kAhead;
  st.runs = (st.all + st.run - 1u) / st.run;
  const uint64_t units = static_cast<uint64_t>(job.tokens) * st.runs;
  const unsigned grid = static_cast<unsigned>((units + kWarps - 1u) / kWarps);
  if (bf16) {
    if (vec) launch_early(k_qkv<HD, true, true>, dim3(grid), kWarps * 32, 0, stream, job, st, err);
    else launch_early(k_qkv<HD, true, false>, dim3(grid), kWarps * 32, 0, stream, job, st, err);
  } else {
    if (vec) launch_early(k_qkv<HD, false, true>, dim3(grid), kWarps * 32, 0, stream, job, st, err);
    else launch_early(k_qkv<HD, false, false>, dim3(grid), kWarps * 32, 0, stream, job, st, err);
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
                    void* k, void* v, uint32_t* error_flag, cudaStream_t stream) {
  const FastDiv row = make_fast_div(cache.kv_heads * (cache.hd / 16u));
  const FastDiv head = make_fast_div(cache.hd / 16u);
  const unsigned grid = (tokens + kTokens - 1u) / kTokens;
  if (dtype == HRB_DT_F32) {
    launch_early(k_kv_read<HRB_DT_F32>, dim3(grid), 256, 0, stream, cache, slots, tokens, row, head, k, v,
                 error_flag);
  } else if (dtype == HRB_DT_BF16) {
    launch_early(k_kv_read<HRB_DT_BF16>, dim3(grid), 256, 0, stream, cache, slots, tokens, row, head, k, v,
                 error_flag);
  } else {
    launch_early(k_kv_read<HRB_DT_E5M2>, dim3(grid), 256, 0, stream, cache, slots, tokens, row, head, k, v,
                 error_flag);
  }
}

}  // namespace hrb
