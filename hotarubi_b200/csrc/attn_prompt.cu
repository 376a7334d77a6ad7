// hrb_attention for many rows a request (prompts and chunks of them), on the
// tensor cores with TMEM accumulators.
//
// k_kv_expand decodes the requests' keys once into FP16 operand tiles of 128
// keys in scratch memory: K [128 keys][hd] and V^T [hd][128 keys], rows of
// 128 bytes in the 128-byte swizzle, exactly as the tensor cores read them
// from shared memory, so that one bulk copy brings a tile.  (Every block of
// rows would otherwise decode the same keys again: a prompt of 8191 tokens
// with four query heads a key/value head reads each key 128 times.)
//
// k_attn_prompt: a block takes 256 rows (query token x query head of one
// key/value head), two halves of 128 that alternate on the tensor cores:
//   warps 0-3, 4-7  softmax of half A, B: a thread a row.  S = Q K^T from
//                   TMEM, running maximum and sum, P = 2^(s - m + 7) as FP16
//                   back to TMEM over S, O scaled there when m moves
//   warp 8          issues S_A, S_B and O_A += P_A V, O_B += P_B V
//                   (tcgen05.mma kind::f16, P from TMEM)
//   warp 9          bulk copies of K and V^T tiles, two stages each
// (with one half a block, 0-3, 4 and 5, and one stage at hd 96 and 128).  While
// one half's softmax runs, the other half's products do; with one half, another
// block's.  m moves only when a row's scores pass it by 2^6,
// so O is rarely scaled.
//
// Few blocks (a short chunk over a long cache) split the keys; k_attn_join
// (attn_decode.cu) joins the rows' (m, l, O).
//
// Its floor is the tensor cores: 4 hd FLOP a pair of query and key that see
// each other.  Measured: a prompt of 8191 tokens, 32/8 heads of 128, 508 to
// 520 us, 1057 to 1083 TFLOP/s, 64 to 65 % of a large BF16 product's rate.  A tile
// takes about 3600 clocks for both halves, the tensor cores work 2048 of them: a
// half's softmax (2200) and its products (1200 with the waits) follow each
// other.  Two S of 64 keys a half, which would let a softmax run ahead, measured
// 660 us where this stood at 555.
#include <cuda_fp16.h>

#include <atomic>
#include <cstdint>

#include "hrb_attn.cuh"
#include "sm100.cuh"

namespace hrb {
namespace {

using namespace sm100;

constexpr uint32_t kKeys = kAttnTileKeys;
constexpr uint32_t kHalf = 128;      // rows a half
constexpr uint32_t kRowB = 128;      // bytes of a swizzled row

// Bytes of a tile's parts: K in chunks of 64 dims, V^T in chunks of 64 keys.
__host__ __device__ constexpr uint32_t k_bytes(uint32_t hd) { return (hd + 63u) / 64u * kKeys * kRowB; }
__host__ __device__ constexpr uint32_t v_bytes(uint32_t hd) { return 2u * hd * kRowB; }
__host__ __device__ constexpr uint32_t tile_bytes(uint32_t hd) { return k_bytes(hd) + v_bytes(hd); }

// Eight dims of a key (a word of codes) as FP16.
__device__ __forceinline__ uint4 key_dims(uint32_t word, uint32_t scale) {
  uint32_t h[4];
  e2m1x8_to_f16x2(word, h);
  return make_uint4(mul2(h[0], scale), mul2(h[1], scale), mul2(h[2], scale), mul2(h[3], scale));
}

// Eight dims of eight keys (a word of codes each, a scale byte each) turned:
// row d holds dim d of the keys.
__device__ __forceinline__ void turn_values(const uint32_t (&w)[8], const uint32_t (&sb)[8],
                                            uint32_t (&h)[8][4]) {
#pragma unroll
  for (uint32_t r = 0; r < 4u; ++r) {
    const uint32_t a = w[2u * r], b = w[2u * r + 1u], sc = scale2(sb[2u * r], sb[2u * r + 1u]);
    uint32_t lo[4], hi[4];
    e2m1x8_to_f16x2((a & 0x0F0F0F0Fu) | ((b << 4) & 0xF0F0F0F0u), lo);
    e2m1x8_to_f16x2(((a >> 4) & 0x0F0F0F0Fu) | (b & 0xF0F0F0F0u), hi);
#pragma unroll
    for (uint32_t d = 0; d < 4u; ++d) {
      h[2u * d][r] = mul2(lo[d], sc);
      h[2u * d + 1u][r] = mul2(hi[d], sc);
    }
  }
}

// Where eight dims (number u) of a key lie in a K tile, and eight keys
// (number kg) of a dim in a V^T tile.
__device__ __forceinline__ uint32_t k_place(uint32_t key, uint32_t u) {
  return (u / 8u) * (kKeys * kRowB) + key * kRowB + (((u & 7u) ^ (key & 7u)) * 16u);
}
template <uint32_t HD>
__device__ __forceinline__ uint32_t v_place(uint32_t dim, uint32_t kg) {
  return (kg / 8u) * (HD * kRowB) + dim * kRowB + (((kg & 7u) ^ (dim & 7u)) * 16u);
}

// A block: one tile of one request and key/value head.
template <uint32_t HD>
__global__ void __launch_bounds__(256)
    k_kv_expand(const AttnJob j, uint32_t* __restrict__ error_flag) {
  constexpr uint32_t kLd = HD / 2u + 4u;  // padded row of codes in shared memory
  __shared__ __align__(16) uint8_t codes[2][kKeys * kLd];
  __shared__ uint8_t scales[2][kKeys * (HD / 32u)];
  // First what comes before in the stream is done; then k_attn_prompt may set
  // up, and load Q, while this runs.
  griddep_wait();
  griddep_launch_dependents();
  const uint32_t n = blockIdx.z, head = blockIdx.y, k0 = blockIdx.x * kKeys;
  int32_t q0, q_len, kv;
  if (!attn_request(j, n, &q0, &q_len, &kv)) {
    if (head == 0u && blockIdx.x == 0u && threadIdx.x == 0u) atomicOr(error_flag, kErrKvSlot);
    return;
  }
  if (q_len == 0 || k0 >= static_cast<uint32_t>(kv)) return;
  const uint32_t tile = attn_first_tile(j, n) + blockIdx.x;
  if (tile >= j.tiles_cap) {  // more keys than total_kv said
    if (threadIdx.x == 0u) atomicOr(error_flag, kErrKvSlot);
    return;
  }
  const uint32_t keys = min(kKeys, static_cast<uint32_t>(kv) - k0);
  // The second 64 keys of a request's last tile are not read where it has
  // none there (the products stop before them): not written either.
  const uint32_t span = keys <= 64u ? 64u : kKeys;
  // A block of 32 dims of a key's K and V, and its scales, a thread at a time;
  // keys past the end and pages outside the cache are zeros.
  bool bad = false;
  const int32_t* table = j.table + static_cast<uint64_t>(n) * j.table_ld;
#pragma unroll
  for (uint32_t i = threadIdx.x; i < kKeys * (HD / 32u); i += 256u) {
    const uint32_t key = i / (HD / 32u), b = i % (HD / 32u);
    uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    uint32_t sb[2] = {127u, 127u};
    if (key < keys) {
      const uint32_t page = static_cast<uint32_t>(ld(table + ((k0 + key) >> j.cache.page_log2)));
      if (page < j.cache.pages) {
        const uint32_t in = (k0 + key) & (j.cache.page - 1u);
        const uint8_t* rec = kv_record(j.cache, page, head);
#pragma unroll
        for (uint32_t p = 0; p < 2u; ++p) {
          const uint8_t* part = rec + (p == 0u ? 0u : kv_vcodes(j.cache));
          x[p] = ld(reinterpret_cast<const uint4*>(part + in * (HD / 2u) + 16u * b));
          sb[p] = part[kv_kscales(j.cache) + in * (HD / 32u) + b];
        }
      } else {
        bad = true;
      }
    }
#pragma unroll
    for (uint32_t p = 0; p < 2u; ++p) {
      uint32_t* to = reinterpret_cast<uint32_t*>(&codes[p][key * kLd + 16u * b]);
      to[0] = x[p].x;
      to[1] = x[p].y;
      to[2] = x[p].z;
      to[3] = x[p].w;
      scales[p][i] = static_cast<uint8_t>(sb[p]);
    }
  }
  if (bad) atomicOr(error_flag, kErrKvSlot);
  __syncthreads();
  uint8_t* out = j.tiles + (static_cast<uint64_t>(head) * j.tiles_cap + tile) * tile_bytes(HD);
  // K: 16 bytes (8 dims of a key) a step, neighbours in a row.
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < span * (HD / 8u); i += 256u) {
    const uint32_t key = i / (HD / 8u), u = i % (HD / 8u);
    const uint32_t b = scales[0][key * (HD / 32u) + u / 4u];
    *reinterpret_cast<uint4*>(out + k_place(key, u)) =
        key_dims(*reinterpret_cast<const uint32_t*>(&codes[0][key * kLd + 4u * u]), scale2(b, b));
  }
  // V^T: a thread turns 8 keys x 8 dims; 8 neighbours fill a row.
  out += k_bytes(HD);
  for (uint32_t i = threadIdx.x; i < (kKeys / 8u) * (HD / 8u); i += 256u) {
    const uint32_t kg = i % (kKeys / 8u), dg = i / (kKeys / 8u);
    if (8u * kg >= span) continue;
    uint32_t w[8], sb[8], h[8][4];
#pragma unroll
    for (uint32_t r = 0; r < 8u; ++r) {
      w[r] = *reinterpret_cast<const uint32_t*>(&codes[1][(8u * kg + r) * kLd + 4u * dg]);
      sb[r] = scales[1][(8u * kg + r) * (HD / 32u) + dg / 4u];
    }
    turn_values(w, sb, h);
#pragma unroll
    for (uint32_t d = 0; d < 8u; ++d) {
      *reinterpret_cast<uint4*>(out + v_place<HD>(8u * dg + d, kg)) =
          make_uint4(h[d][0], h[d][1], h[d][2], h[d][3]);
    }
  }
}

// HV halves of 128 rows.  Two share their tiles and fill an SM: 384 threads
// (three warpgroups, warps 10 and 11 only give up registers), all of TMEM.
// One is half of that, two blocks an SM: for short histories, where a block
// is mostly set-up, Q and output.
template <uint32_t HD, uint32_t HV>
struct Cfg {
  static constexpr uint32_t kThreads = HV * 128u + 128u;
  static constexpr uint32_t kStages = HV == 2u || HD <= 64u ? 2u : 1u;  // of K and of V^T
  static constexpr uint32_t kO = HV * 128u;                    // TMEM column of O (S at 0)
  static constexpr uint32_t kTmem = HV * 256u;
  static constexpr uint32_t kQ = HV * k_bytes(HD);
  static constexpr uint32_t kK = kQ;
  static constexpr uint32_t kV = kK + kStages * k_bytes(HD);
  static constexpr uint32_t kBars = kV + kStages * v_bytes(HD);
  static constexpr uint32_t kUsed = kBars + 160u;
  // No more blocks an SM than its 512 columns of TMEM hold.
  static constexpr uint32_t kLeast = (HV == 2u ? 120u : 78u) * 1024u;
  static constexpr uint32_t kBytes = (kUsed > kLeast ? kUsed : kLeast) + 1024u;
};

// Instruction descriptor of kind::f16 with FP16 A and B, FP32 D, K-major
// operands (the fields of idesc_bf16 with formats 0).
constexpr uint32_t idesc_f16(uint32_t m, uint32_t n) {
  return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// The low word of a desc_sw128 descriptor (its start address, in 16-byte
// units, and fields that do not change); the high word is the same for all.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t smem_byte_addr) {
  return static_cast<uint32_t>(desc_sw128(smem_byte_addr));
}
// The lowest n bits (none for n below 0, all from 32).
__device__ __forceinline__ uint32_t low_bits(int32_t n) {
  return n >= 32 ? 0xFFFFFFFFu : (1u << max(n, 0)) - 1u;
}
// Keeps a value where it is: what is added to it is not computed ahead for a
// whole loop, in registers the issuing thread does not have.
__device__ __forceinline__ uint32_t here(uint32_t x) {
  asm volatile("" : "+r"(x));
  return x;
}

// kind::f16 with FP16 operands: A and B in shared memory, and A in TMEM.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
      ::"r"(d), "r"(a_tmem), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
      : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A row's raw scores to softcap log2(e) tanh(factor s / softcap).  Where a
// warp's arguments are all small, tanh is its power series on the FMA pipe: up
// to x^7 under 1/4 and x^11 under 1/2 (the next terms are under 9e-8 and 4.4e-7
// there); else cap_score, a score at a time.  A chunk of 512 tokens over 8703
// keys, 32/8 heads of 128, a pass alone with cold L2: 128 us with small scores,
// 196 with scores near a cap of 30 (two MUFU operations a score more).
template <uint32_t TERMS>
__device__ __forceinline__ void tanh_series(uint32_t (&s)[4][32], float f, float b) {
  constexpr float kSeries[6] = {1.f, -1.f / 3.f, 2.f / 15.f, -17.f / 315.f, 62.f / 2835.f, -1382.f / 155925.f};
  uint64_t a[TERMS];
#pragma unroll
  for (uint32_t t = 0; t < TERMS; ++t) a[t] = pack2(b * kSeries[t], b * kSeries[t]);
  const uint64_t f2 = pack2(f, f);
#pragma unroll
  for (uint32_t c = 0; c < 4u; ++c)
#pragma unroll
    for (uint32_t i = 0; i < 32u; i += 2u) {
      const uint64_t x = mul_2(pack2(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1u])), f2);
      const uint64_t u = mul_2(x, x);
      uint64_t r = a[TERMS - 1u];
#pragma unroll
      for (uint32_t t = TERMS - 1u; t > 0u; --t) r = fma_2(r, u, a[t - 1u]);
      const float2 y = unpack2(mul_2(r, x));
      s[c][i] = __float_as_uint(y.x);
      s[c][i + 1u] = __float_as_uint(y.y);
    }
}

__device__ __forceinline__ void cap_scores(const AttnJob& j, float factor, uint32_t (&s)[4][32]) {
  // For a cap near the type's end the factor would lose its bits under 2^-126;
  // under 2^-100 no product of S passes 2^-60, where tanh x is x.
  const bool linear = factor * j.cap_inv < 0x1p-100f;
  const float f = linear ? 0x1p-100f : factor * j.cap_inv;
  const float b = linear ? factor * kLog2e * 0x1p100f : j.cap_out;
  float top[8];
#pragma unroll
  for (uint32_t c = 0; c < 8u; ++c) top[c] = 0.f;
#pragma unroll
  for (uint32_t i = 0; i < 16u; i += 2u)
#pragma unroll
    for (uint32_t c = 0; c < 8u; ++c) {
      const uint32_t at = 16u * (c & 1u) + i;
      top[c] = max3(top[c], fabsf(__uint_as_float(s[c >> 1][at])), fabsf(__uint_as_float(s[c >> 1][at + 1u])));
    }
  const float high = max3(max3(top[0], top[1], top[2]), max3(top[3], top[4], top[5]),
                          fmaxf(top[6], top[7])) * f;
  if (__all_sync(0xFFFFFFFFu, high < 0.25f)) {
    tanh_series<4>(s, f, b);
  } else if (__all_sync(0xFFFFFFFFu, high < 0.5f)) {
    tanh_series<6>(s, f, b);
  } else if (j.softcap > kWideCap) {
#pragma unroll
    for (uint32_t c = 0; c < 4u; ++c)
#pragma unroll
      for (uint32_t i = 0; i < 32u; ++i) {
        s[c][i] = __float_as_uint(cap_score<true>(j, __uint_as_float(s[c][i]) * factor));
      }
  } else {
#pragma unroll
    for (uint32_t c = 0; c < 4u; ++c)
#pragma unroll
      for (uint32_t i = 0; i < 32u; ++i) {
        s[c][i] = __float_as_uint(cap_score<false>(j, __uint_as_float(s[c][i]) * factor));
      }
  }
}

// SHAPED: a cap or a distance bias on the scores; apart, because their code
// would cost the plain kernel registers.
template <uint32_t HD, uint32_t HV, bool SHAPED>
__global__ void __launch_bounds__(Cfg<HD, HV>::kThreads, HV == 2u ? 1 : 2)
    k_attn_prompt(const AttnJob j, uint32_t* __restrict__ error_flag) {
  using S = Cfg<HD, HV>;
  constexpr uint32_t kNs = S::kStages;
  constexpr int32_t kBlockRows = static_cast<int32_t>(HV * kHalf);
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 3, *v_full = bars + 5,
           *v_empty = bars + 7, *s_full = bars + 9, *o_full = bars + 11,
           *p_full = bars + 13,  // [half][first or second 64 keys]
           *done = bars + 17;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;

  const uint32_t head = blockIdx.x % j.cache.kv_heads, n = blockIdx.z;
  const uint32_t chunk = blockIdx.x / j.cache.kv_heads;
  int32_t q0, q_len, kv;
  if (!attn_request(j, n, &q0, &q_len, &kv)) return;  // k_kv_expand reports it
  const int32_t rows = q_len * static_cast<int32_t>(j.group);
  // The last rows see the most keys: they start first.
  const int32_t q_tiles = (rows + kBlockRows - 1) / kBlockRows;
  if (static_cast<int32_t>(blockIdx.y) >= q_tiles) return;
  const int32_t r0 = (q_tiles - 1 - static_cast<int32_t>(blockIdx.y)) * kBlockRows;
  const int32_t r1 = min(rows, r0 + kBlockRows);
  const int32_t c0 = static_cast<int32_t>(chunk * j.chunk);
  const bool whole = kv <= static_cast<int32_t>(j.chunk);
  if (c0 >= kv && c0 > 0) return;
  const int32_t c1 = c0 + min(kv - c0, static_cast<int32_t>(j.chunk));
  const uint32_t base = attn_first_tile(j, n);
  if (!attn_tiles_fit(j, base, kv)) {  // reported too
    griddep_wait();  // what follows in the stream must find k_kv_expand done
    return;
  }
  const uint32_t halves = HV == 2u && r1 - r0 > static_cast<int32_t>(kHalf) ? 2u : 1u;

  // The tiles that some row of the block sees: numbers 0 .. gap - 1 and
  // resume .. of the chunk's, `count` in all.
  const int32_t pre = j.prefix != nullptr ? __ldcg(j.prefix + n) : 0;
  const int32_t group = static_cast<int32_t>(j.group);
  const Seen first = attn_seen(j, kv - q_len + r0 / group, kv, pre);
  const Seen last = attn_seen(j, kv - q_len + (r1 - 1) / group, kv, pre);
  auto tiles_to = [&](int32_t k) {
    return (min(max(k, c0), c1) - c0 + static_cast<int32_t>(kKeys) - 1) / static_cast<int32_t>(kKeys);
  };
  const int32_t gap = tiles_to(first.pre), end = max(gap, tiles_to(last.hi));
  const int32_t resume = max(gap, min(end, tiles_to(first.lo + 1 - static_cast<int32_t>(kKeys))));
  const int32_t count = gap + end - resume;
  auto tile_at = [&](int32_t it) { return it < gap ? it : it - gap + resume; };
  // Of the last tile only the first 64 keys, where no row sees another.
  const int32_t half_end = c0 + tile_at(count - 1) * static_cast<int32_t>(kKeys) + 64;
  const bool last_half = min(max(last.hi, first.pre), c1) <= half_end;

  // A softmax thread's row (its half's thread number) and its part of Q, on
  // their way while the block sets up.
  const uint32_t in_half = threadIdx.x & (kHalf - 1u);
  const int32_t r = r0 + static_cast<int32_t>(threadIdx.x);
  const bool mine = warp < 4u * HV && r < r1;
  const uint64_t row = static_cast<uint64_t>(q0 + (mine ? r : r0) / group);
  const uint32_t qh = head * j.group + static_cast<uint32_t>((mine ? r : r0) % group);
  uint4 q_row[HD / 8u];
#pragma unroll
  for (uint32_t i = 0; i < HD / 8u; ++i) {
    q_row[i] = mine ? __ldcg(reinterpret_cast<const uint4*>(j.q + row * j.ldq + static_cast<uint64_t>(qh) * HD) + i)
                    : make_uint4(0, 0, 0, 0);
  }

  if (threadIdx.x == 0u) {
    mbar_init(q_full, HV * 128u);
    mbar_init(done, 1);
    for (uint32_t i = 0; i < 2u; ++i) {
      mbar_init(k_full + i, 1);
      mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, 1);
      mbar_init(v_empty + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(p_full + 2u * i, kHalf);
      mbar_init(p_full + 2u * i + 1u, kHalf);
      mbar_init(o_full + i, 1);
    }
    fence_barrier_init();
  }
  if (warp == 4u * HV) {
    tmem_alloc(tmem_slot, S::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // A softmax thread holds a row's 128 scores (measured on one box, split 224/56:
  // 475 us for the 8191 prompt but 124.5 for 512 tokens over 8703 keys, 216/72
  // 481 and 119.5, 208/88 478 and 119.6).  Registers at launch: 384 x 168 =
  // 256 x 208 + 128 x 88 (HV 2), 256 x 128 = 128 x 200 + 128 x 56.
  if (warp >= 4u * HV) {
    if constexpr (HV == 2u) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    }
    if (warp == 4u * HV + 1u) {
      if (lane == 0u) {
        griddep_wait();  // k_kv_expand's tiles
        const uint8_t* src = j.tiles + (static_cast<uint64_t>(head) * j.tiles_cap + base +
                                        static_cast<uint32_t>(c0) / kKeys) * tile_bytes(HD);
        int32_t it = 0;
        for (; it < count; ++it) {
          const uint32_t st = static_cast<uint32_t>(it) % kNs, ph = (static_cast<uint32_t>(it) / kNs) & 1u;
          const bool wait = it >= static_cast<int32_t>(kNs);
          const uint8_t* tile = src + static_cast<uint64_t>(tile_at(it)) * tile_bytes(HD);
          if (wait && !mbar_wait(k_empty + st, ph ^ 1u, error_flag)) break;
          mbar_arrive_expect_tx(k_full + st, k_bytes(HD));
          bulk_g2s(smem + S::kK + st * k_bytes(HD), tile, k_bytes(HD), k_full + st);
          if (wait && !mbar_wait(v_empty + st, ph ^ 1u, error_flag)) break;
          mbar_arrive_expect_tx(v_full + st, v_bytes(HD));
          bulk_g2s(smem + S::kV + st * v_bytes(HD), tile + k_bytes(HD), v_bytes(HD), v_full + st);
        }
        // Nothing of this block's may still be arriving when it ends.
        for (int32_t w = max(it - static_cast<int32_t>(kNs), 0); w < min(it + 1, count); ++w) {
          const uint32_t st = static_cast<uint32_t>(w) % kNs, ph = (static_cast<uint32_t>(w) / kNs) & 1u;
          if (w < it && !mbar_wait(v_full + st, ph, error_flag)) break;
          if (w == it && !mbar_wait(k_full + st, ph, error_flag, 1000u)) break;
        }
      }
    } else if (warp == 4u * HV) {
      if (lane == 0u && count > 0) {
        const uint32_t q_at = desc_low(smem_addr(smem)), k_at = desc_low(smem_addr(smem + S::kK));
        const uint32_t v_at = desc_low(smem_addr(smem + S::kV));
        auto scores = [&](uint32_t h, uint32_t st) {
          const uint32_t a = here(q_at + h * (k_bytes(HD) / 16u));
          const uint32_t b = here(k_at + st * (k_bytes(HD) / 16u));
#pragma unroll
          for (uint32_t k = 0; k < HD / 16u; ++k) {
            const uint32_t off = ((k >> 2) * (kKeys * kRowB) + 32u * (k & 3u)) / 16u;
            mma_ss(tmem + 128u * h, a + off, b + off, idesc_f16(128, 128), k != 0u);
          }
          mma_commit(s_full + h);
        };
        bool ok = mbar_wait(q_full, 0, error_flag) && mbar_wait(k_full, 0, error_flag);
        if (ok) {
          tc_fence_after();
          for (uint32_t h = 0; h < halves; ++h) scores(h, 0);
          mma_commit(k_empty);
        }
        for (int32_t it = 0; it < count && ok; ++it) {
          const uint32_t st = static_cast<uint32_t>(it) % kNs, ph = (static_cast<uint32_t>(it) / kNs) & 1u;
          const uint32_t nst = static_cast<uint32_t>(it + 1) % kNs;
          const bool more = it + 1 < count;
          // Both tiles' arrivals first: the softmax's are then the only waits
          // between the products.
          ok = mbar_wait(v_full + st, ph, error_flag) &&
               (!more || mbar_wait(k_full + nst, (static_cast<uint32_t>(it + 1) / kNs) & 1u, error_flag));
          for (uint32_t h = 0; h < halves && ok; ++h) {
            const uint32_t a = here(tmem + 128u * h), b = here(v_at + st * (v_bytes(HD) / 16u));
            const uint32_t d = tmem + S::kO + 128u * h;
#pragma unroll
            for (uint32_t k = 0; k < kKeys / 16u; ++k) {
              if (k == 4u && last_half && !more) break;
              if ((k & 3u) == 0u) {  // 64 keys' weights
                ok = mbar_wait(p_full + 2u * h + (k >> 2), static_cast<uint32_t>(it) & 1u, error_flag);
                if (!ok) break;
                tc_fence_after();
              }
              mma_ts(d, a + 8u * k, b + ((k >> 2) * (HD * kRowB) + 32u * (k & 3u)) / 16u, idesc_f16(128, HD),
                     it != 0 || k != 0u);
            }
            if (!ok) break;
            if (more) {
              scores(h, nst);
            } else {
              mma_commit(o_full + h);
            }
          }
          mma_commit(v_empty + st);
          if (more) mma_commit(k_empty + nst);
        }
        // The block keeps its barriers and TMEM until all products, and their
        // arrivals that nothing else waits for, are in (also after a timeout).
        mma_commit(done);
        mbar_wait(done, 0, error_flag);
      }
    }
  } else {
    if constexpr (HV == 2u) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    }
    const uint32_t h = warp >> 2;
    float factor;
    bool odd;  // Inf or NaN in the row of Q: its outputs are NaN
    {
      // The row of Q as FP16, scaled so that its largest value is in
      // [2^13, 2^14) and signed so that the scores' factor is not negative.
      uint32_t top = 0;
#pragma unroll
      for (uint32_t i = 0; i < HD / 8u; ++i) {
        const uint32_t w[4] = {q_row[i].x, q_row[i].y, q_row[i].z, q_row[i].w};
#pragma unroll
        for (uint32_t d = 0; d < 4u; ++d) top = max(top, max(w[d] & 0x7FFFu, (w[d] >> 16) & 0x7FFFu));
      }
      odd = top >= 0x7F80u;
      const int32_t e = min(max(static_cast<int32_t>(top >> 7), 27), 254) - 127;
      float up = __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
      if (j.scale < 0.f) up = -up;
      factor = fabsf(j.scale) * __uint_as_float(static_cast<uint32_t>(127 - 13 + e) << 23) *
               (SHAPED && j.softcap != 0.f ? 1.0f : kLog2e);
      factor = fmaxf(factor, 1.2e-38f);  // times a masked score's -inf is no NaN
      uint8_t* dst = smem + h * k_bytes(HD) + in_half * kRowB;
#pragma unroll
      for (uint32_t i = 0; i < HD / 8u; ++i) {
        const uint32_t w[4] = {q_row[i].x, q_row[i].y, q_row[i].z, q_row[i].w};
        uint32_t o[4];
#pragma unroll
        for (uint32_t d = 0; d < 4u; ++d) {
          o[d] = half2_bits(__floats2half2_rn(__uint_as_float(w[d] << 16) * up,
                                              __uint_as_float(w[d] & 0xFFFF0000u) * up));
        }
        *reinterpret_cast<uint4*>(dst + (i >> 3) * (kKeys * kRowB) + (((i & 7u) ^ (in_half & 7u)) * 16u)) =
            make_uint4(o[0], o[1], o[2], o[3]);
      }
      fence_proxy_async_smem();
      mbar_arrive(q_full);
    }
    const int32_t pos = kv - q_len + (mine ? r : r0) / group;
    Seen seen = attn_seen(j, pos, kv, pre);
    const bool idle = !__any_sync(0xFFFFFFFFu, mine);  // a warp without rows
    const float slope = SHAPED && j.slopes != nullptr ? ld(j.slopes + qh) * kLog2e : 0.f;
    const uint32_t lanes = ((warp & 3u) * 32u) << 16;
    const uint32_t t_s = tmem + lanes + 128u * h, t_o = tmem + lanes + S::kO + 128u * h;
    float m = -INFINITY, l = 0.f;
    bool ok = true, far = false;  // far: some row's m of the warp has been (kFar)
    if (h < halves) {
      for (int32_t it = 0; it < count; ++it) {
        ok = mbar_wait(s_full + h, static_cast<uint32_t>(it) & 1u, error_flag);
        if (!__all_sync(0xFFFFFFFFu, ok)) break;
        const bool both = !(last_half && it == count - 1);  // 64s of keys
        if (idle) {  // what its rows of P and O hold does not matter
          mbar_arrive(p_full + 2u * h);
          if (both) mbar_arrive(p_full + 2u * h + 1u);
          continue;
        }
        tc_fence_after();
        uint32_t s[4][32];
        tmem_ld32(t_s, s[0]);
        tmem_ld32(t_s + 32u, s[1]);
        if (both) {
          tmem_ld32(t_s + 64u, s[2]);
          tmem_ld32(t_s + 96u, s[3]);
        }
        tmem_wait_ld();
        if (!both) {  // masked below, no row sees them; zeros leave a cap's series open
#pragma unroll
          for (uint32_t i = 0; i < 32u; ++i) s[2][i] = s[3][i] = 0;
        }
        const int32_t k0 = c0 + tile_at(it) * static_cast<int32_t>(kKeys);
        const int32_t k1 = k0 + static_cast<int32_t>(kKeys);
        auto at = [&](uint32_t c, uint32_t i) -> float { return __uint_as_float(s[c][i]); };
        auto pair = [&](uint32_t c, uint32_t i) { return pack2(at(c, i), at(c, i + 1u)); };
        float scale = factor;
        if (SHAPED && j.softcap != 0.f) {
          scale = 1.0f;
          cap_scores(j, factor, s);
        }
        if (SHAPED && j.slopes != nullptr) {
          const float far = static_cast<float>(pos - k0);
#pragma unroll
          for (uint32_t c = 0; c < 4u; ++c)
#pragma unroll
            for (uint32_t i = 0; i < 32u; ++i) {
              s[c][i] = __float_as_uint(fmaf(-slope, fabsf(far - static_cast<float>(32u * c + i)),
                                             at(c, i) * scale));
            }
          scale = 1.0f;
        }
        const bool clear = !mine || (k0 >= seen.lo && k1 <= seen.hi) || k1 <= seen.pre;
        if (!__all_sync(0xFFFFFFFFu, clear)) {
          // Keys [lo, hi) and [0, pre) of the tile, a bit each.
#pragma unroll
          for (uint32_t c = 0; c < 4u; ++c) {
            const int32_t k = k0 + static_cast<int32_t>(32u * c);
            const uint32_t see = (low_bits(seen.hi - k) & ~low_bits(seen.lo - k)) | low_bits(seen.pre - k);
#pragma unroll
            for (uint32_t i = 0; i < 32u; ++i) {
              if (((see >> i) & 1u) == 0u) s[c][i] = 0xFF800000u;
            }
          }
        }
        float top[8];
#pragma unroll
        for (uint32_t c = 0; c < 8u; ++c) {
          const uint32_t at0 = 16u * (c & 1u);
          top[c] = max3(at(c >> 1, at0), at(c >> 1, at0 + 1u), at(c >> 1, at0 + 2u));
        }
#pragma unroll
        for (uint32_t i = 3; i < 15u; i += 2u)
#pragma unroll
          for (uint32_t c = 0; c < 8u; ++c) {
            const uint32_t at0 = 16u * (c & 1u) + i;
            top[c] = max3(top[c], at(c >> 1, at0), at(c >> 1, at0 + 1u));
          }
#pragma unroll
        for (uint32_t c = 0; c < 8u; ++c) top[c] = fmaxf(top[c], at(c >> 1, 16u * (c & 1u) + 15u));
        const float high = max3(max3(top[0], top[1], top[2]), max3(top[3], top[4], top[5]),
                                fmaxf(top[6], top[7])) * scale;
        const bool moves = high - m > kLazy;
        if (__any_sync(0xFFFFFFFFu, moves || far)) {
          const float keep = moves ? ex2(m - high) : 1.0f;
          if (moves) m = high;
          if constexpr (!SHAPED) {
            far = far || __any_sync(0xFFFFFFFFu, attn_far(m));
            if (far) {
#pragma unroll
              for (uint32_t c = 0; c < 4u; ++c)
#pragma unroll
                for (uint32_t i = 0; i < 32u; ++i) s[c][i] = __float_as_uint(__fmul_rn(at(c, i), scale));
              scale = 1.0f;
            }
          }
          l *= keep;
          if (it != 0) {
#pragma unroll 1
            for (uint32_t c = 0; c < HD / 16u; ++c) {
              uint32_t o[16];
              tmem_ld16(t_o + 16u * c, o);
              tmem_wait_ld();
#pragma unroll
              for (uint32_t i = 0; i < 16u; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
              tmem_st16(t_o + 16u * c, o);
            }
          }
        }
        const float shift = m == -INFINITY ? 0.f : kLift - m;
        const uint64_t scale2x = pack2(scale, scale), shift2x = pack2(shift, shift);
        uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t c = 0; c < 2u; ++c) {
          if (c == 1u && !both) break;
          uint32_t p[32];
#pragma unroll
          for (uint32_t i = 0; i < 32u; ++i) {
            const uint64_t x = fma_2(pair(2u * c + i / 16u, 2u * (i % 16u)), scale2x, shift2x);
            const float2 v = unpack2(x), e = make_float2(ex2(v.x), ex2(v.y));
            sum[i & 3u] = add_2(sum[i & 3u], pack2(e.x, e.y));
            p[i] = half2_bits(__floats2half2_rn(e.x, e.y));
          }
          tmem_st32(t_s + 32u * c, p);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(p_full + 2u * h + c);  // the product of these 64 keys may start
        }
        const float2 all = unpack2(add_2(add_2(sum[0], sum[1]), add_2(sum[2], sum[3])));
        l += all.x + all.y;
      }
      if (count > 0 && ok && !idle) ok = mbar_wait(o_full + h, 0, error_flag);
      if (__all_sync(0xFFFFFFFFu, ok && !idle)) {
        tc_fence_after();
        if (odd && (seen.lo < seen.hi || seen.pre > 0)) l = NAN;
        const float inv = l != 0.f ? 1.0f / l : 0.f;
        const uint64_t cell = (static_cast<uint64_t>(chunk) * j.total_q + row) * j.heads + qh;
#pragma unroll 1
        for (uint32_t c = 0; c < HD / 32u; ++c) {
          uint32_t o[32];
          __syncwarp();
          if (count > 0) {
            tmem_ld32(t_o + 32u * c, o);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (uint32_t i = 0; i < 32u; ++i) o[i] = 0;
          }
          if (mine) {
            float x[32];
#pragma unroll
            for (uint32_t i = 0; i < 32u; ++i) x[i] = __uint_as_float(o[i]) * (whole ? inv : 1.0f);
            if (whole) {
              write_row_block(j, row, qh, c, x, error_flag);
            } else {
              float4* to = reinterpret_cast<float4*>(j.part_o + cell * HD + 32u * c);
#pragma unroll
              for (uint32_t i = 0; i < 8u; ++i) {
                to[i] = make_float4(x[4u * i], x[4u * i + 1u], x[4u * i + 2u], x[4u * i + 3u]);
              }
              if (c == 0u) j.part_ml[cell] = make_float2(m, l);
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 4u * HV) tmem_dealloc(tmem, S::kTmem);
}

template <uint32_t HD, uint32_t HV, bool SHAPED>
int launch(const AttnJob& job, uint32_t chunks, uint32_t* err, cudaStream_t stream) {
  using S = Cfg<HD, HV>;
  static std::atomic<uint64_t> set{0};  // devices whose limit is raised
  if (((set.load(std::memory_order_relaxed) >> (job.device & 63u)) & 1u) == 0u || job.device > 63u) {
    if (cudaFuncSetAttribute(k_attn_prompt<HD, HV, SHAPED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             S::kBytes) != cudaSuccess) {
      return -1;
    }
    set.fetch_or(uint64_t{1} << (job.device & 63u), std::memory_order_relaxed);
  }
  const uint32_t key_tiles = (job.max_kv + kKeys - 1u) / kKeys;
  const uint32_t q_tiles = (job.max_q * job.group + HV * kHalf - 1u) / (HV * kHalf);
  const bool expand = key_tiles != 0u;
  if (expand) {
    if (launch_early(k_kv_expand<HD>, dim3(key_tiles, job.cache.kv_heads, job.seqs), 256, 0, stream, job,
                     err) != cudaSuccess) {
      return -1;
    }
  }
  // Its blocks may start, load Q and set up while k_kv_expand still runs: that
  // lets them when all before it is done, so Q and the lists are there.
  const dim3 grid(chunks * job.cache.kv_heads, q_tiles, job.seqs);
  if (expand) {
    if (launch_early(k_attn_prompt<HD, HV, SHAPED>, grid, S::kThreads, S::kBytes, stream, job, err) !=
        cudaSuccess) {
      return -1;
    }
  } else {
    k_attn_prompt<HD, HV, SHAPED><<<grid, S::kThreads, S::kBytes, stream>>>(job, err);
  }
  return expand ? 2 : 1;
}

template <uint32_t HD>
int launch_hd(const AttnJob& job, uint32_t chunks, uint32_t* err, cudaStream_t stream) {
  // One half a block for short histories, two for long ones: 32 prompts of 141
  // tokens 23.7 and 28.9 us (15/5 heads of 64), 70.9 and 72.6 us (32/8 of 128);
  // one of 512 12.1 and 15.1 us (64); 80 rows over 500 keys, 32 requests, 36.7
  // and 43.9 us (128); but 600 rows over 3000 keys 58.2 and 54.7 us (64).
  const bool shaped = job.softcap != 0.f || job.slopes != nullptr;
  if (job.max_kv <= 1024u) {
    return shaped ? launch<HD, 1, true>(job, chunks, err, stream)
                  : launch<HD, 1, false>(job, chunks, err, stream);
  }
  return shaped ? launch<HD, 2, true>(job, chunks, err, stream)
                : launch<HD, 2, false>(job, chunks, err, stream);
}

}  // namespace

uint64_t attn_prompt_tiles(const AttnJob& job, uint64_t total_kv, uint32_t* stride) {
  // Tiles at a fixed stride a request cost no sum over the requests before
  // it (64 requests: 1.5 us a block); requests of very different lengths
  // would waste scratch, so only up to twice what they need.
  const uint64_t tight = total_kv / kKeys + job.seqs;
  const uint64_t most = (job.max_kv + kKeys - 1u) / kKeys;
  const uint64_t even = most * job.seqs;
  const bool use = even <= 2u * tight && even <= 0xFFFFFFFFull;
  *stride = use ? static_cast<uint32_t>(most) : 0u;
  return use ? even : tight;
}
uint64_t attn_prompt_tile_bytes(const AttnJob& job) { return tile_bytes(job.cache.hd); }

uint32_t attn_prompt_chunk(const AttnJob& job, int sm_count) {
  // Blocks for every SM where the rows alone do not give them: chunks of 512
  // keys at least.
  const uint64_t rows = static_cast<uint64_t>(job.total_q) * job.group;
  const uint64_t blocks = (rows + 2u * kHalf - 1u) / (2u * kHalf) * job.cache.kv_heads;
  const uint64_t split = static_cast<uint64_t>(sm_count) / blocks;
  uint64_t chunk = job.max_kv;
  if (split > 1u) chunk = (job.max_kv + split - 1u) / split;
  if (chunk < 512u) chunk = 512u;
  chunk = (chunk + kKeys - 1u) / kKeys * kKeys;
  return static_cast<uint32_t>(chunk < 0x40000000u ? chunk : 0x40000000u);  // 31 bits
}

int launch_attn_prompt(const AttnJob& job, uint32_t* error_flag, cudaStream_t stream) {
  const uint32_t chunks = job.max_kv == 0u ? 1u : (job.max_kv + job.chunk - 1u) / job.chunk;
  int n;
  switch (job.cache.hd) {
    case 32: n = launch_hd<32>(job, chunks, error_flag, stream); break;
    case 64: n = launch_hd<64>(job, chunks, error_flag, stream); break;
    case 96: n = launch_hd<96>(job, chunks, error_flag, stream); break;
    default: n = launch_hd<128>(job, chunks, error_flag, stream); break;
  }
  if (n < 0 || chunks == 1u) return n;
  return launch_attn_join(job, stream, error_flag) < 0 ? -1 : n + 1;
}

}  // namespace hrb
