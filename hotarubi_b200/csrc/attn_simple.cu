// hrb_attention on the CUDA cores: one block per (row of q, query head), the
// keys in tiles of 128, the softmax with a running maximum and sum.
//
//   m' = max(m, max_j s_j);  l = l e^(m - m') + sum_j e^(s_j - m');
//   o = o e^(m - m') + sum_j e^(s_j - m') v_j;  out = o / l  (0 where l = 0)
//
// A thread scores one key of a tile, then sums one dim over the tile's keys.
#include <cuda_fp16.h>

#include <cstdint>

#include "hrb_quant.cuh"
#include "hrb_serve.cuh"

namespace hrb {
namespace {

constexpr uint32_t kThreads = 128;

__global__ void __launch_bounds__(kThreads)
    k_attn_simple(const AttnJob j, uint32_t* __restrict__ error_flag) {
  __shared__ float q[128], p[kThreads], part[kThreads / 32u];
  __shared__ uint32_t pages[kThreads];
  const uint32_t row = blockIdx.x, h = blockIdx.y, t = threadIdx.x, hd = j.cache.hd;
  uint32_t lo = 0, hi = j.seqs;  // the request of this row
  while (hi - lo > 1u) {
    const uint32_t mid = (lo + hi) / 2u;
    if (static_cast<uint32_t>(j.q_start[mid]) <= row) lo = mid; else hi = mid;
  }
  while (lo + 1u < j.seqs && static_cast<uint32_t>(j.q_start[lo + 1u]) <= row) ++lo;
  int32_t q0, q_len, kv;
  if (!attn_request(j, lo, &q0, &q_len, &kv)) {
    if (h == 0u && t == 0u) atomicOr(error_flag, kErrKvSlot);
    return;
  }
  if (static_cast<int32_t>(row) < q0 || static_cast<int32_t>(row) >= q0 + q_len) return;
  const int32_t i = kv - q_len + (static_cast<int32_t>(row) - q0);
  const Seen seen = attn_seen(j, i, kv, j.prefix != nullptr ? j.prefix[lo] : 0);
  const float slope = j.slopes != nullptr ? j.slopes[h] : 0.f;
  if (t < hd) {
    q[t] = __uint_as_float(static_cast<uint32_t>(j.q[row * j.ldq + h * hd + t]) << 16);
  }
  float m = -INFINITY, l = 0.f, o = 0.f;
  bool bad = false;
  const int32_t end = max(seen.hi, seen.pre);
  for (int32_t c = 0; c < end; c += kThreads) {
    __syncthreads();
    const int32_t k = c + static_cast<int32_t>(t);
    float s = -INFINITY;
    pages[t] = j.cache.pages;
    if (k < end && attn_sees(seen, k)) {
      const uint32_t page = static_cast<uint32_t>(
          j.table[static_cast<uint64_t>(lo) * j.table_ld + (k >> j.cache.page_log2)]);
      pages[t] = page;
      float dot = 0.f;
      if (page < j.cache.pages) {
        const uint8_t* rec = kv_record(j.cache, page, h / j.group);
        const uint32_t in = static_cast<uint32_t>(k) & (j.cache.page - 1u);
        for (uint32_t b = 0; b < hd / 32u; ++b) {
          float sum = 0.f;
          for (uint32_t d = 0; d < 16u; ++d) {
            const uint32_t two = e2m1_to_f16x2(rec[in * (hd / 2u) + 16u * b + d]);
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&two));
            sum += q[32u * b + 2u * d] * v.x + q[32u * b + 2u * d + 1u] * v.y;
          }
          dot += sum * kv_scale(rec[kv_kscales(j.cache) + in * (hd / 32u) + b]);
        }
      } else {
        bad = true;
      }
      s = j.scale * dot;
      if (j.softcap != 0.f) s = j.softcap * tanhf(s / j.softcap);
      s -= slope * fabsf(static_cast<float>(i - k));
    }
    float top = s;
    for (uint32_t d = 16; d > 0; d /= 2u) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    if ((t & 31u) == 0u) part[t >> 5] = top;
    __syncthreads();
    const float m2 = fmaxf(m, fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
    p[t] = s == -INFINITY ? 0.f : expf(s - m2);
    __syncthreads();
    const float keep = m == -INFINITY ? 0.f : expf(m - m2);
    m = m2;
    l *= keep;
    o *= keep;
    for (uint32_t k2 = 0; k2 < kThreads; ++k2) {
      l += p[k2];
      if (t < hd && p[k2] != 0.f && pages[k2] < j.cache.pages) {
        const uint8_t* rec = kv_record(j.cache, pages[k2], h / j.group) + kv_vcodes(j.cache);
        const uint32_t in = static_cast<uint32_t>(c + k2) & (j.cache.page - 1u);
        const uint32_t two = e2m1_to_f16x2(rec[in * (hd / 2u) + t / 2u]);
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&two));
        o += p[k2] * ((t & 1u) ? v.y : v.x) *
             kv_scale(rec[kv_kscales(j.cache) + in * (hd / 32u) + t / 32u]);
      }
    }
  }
  if (bad) atomicOr(error_flag, kErrKvSlot);
  if (t >= hd) return;
  const float r = l != 0.f ? o / l : 0.f;  // NaN passes
  if (j.out != nullptr) {
    j.out[row * j.ldo + h * hd + t] = attn_bf16(r);
  }
  if (j.oq != nullptr) {
    const uint32_t mag = __float_as_uint(r) & 0x7FFFFFFFu;
    const uint32_t key = __reduce_max_sync(0xFFFFFFFFu, j.vec_rule ? mag >> 23 : mag);
    uint32_t scale;
    const int32_t code = mxint8_code(__float_as_uint(r), key, j.vec_rule != 0, scale);
    j.oq[row * j.ldoq + h * hd + t] = static_cast<int8_t>(code);
    if ((t & 31u) == 0u) j.oscale[row * (j.ldoq / 32u) + (h * hd + t) / 32u] = static_cast<uint8_t>(scale);
    if (mag >= 0x7F800000u && !j.vec_rule) atomicOr(error_flag, 1u);
  }
}

}  // namespace

void launch_attn_simple(const AttnJob& job, uint32_t* error_flag, cudaStream_t stream) {
  k_attn_simple<<<dim3(job.total_q, job.heads), kThreads, 0, stream>>>(job, error_flag);
}

}  // namespace hrb
