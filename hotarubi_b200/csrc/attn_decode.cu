// hrb_attention for few rows a request (single tokens, a few speculated
// ones): the cache is streamed once.
//
// A block serves one request, one key/value head and a chunk of its keys;
// the rows that read that head (rows of q times query heads a key/value head)
// are one operand, in blocks of 8 NT.  Each of its warps takes tiles of 32 keys
// on its own: bulk copies bring a tile's codes and scales into the warp's
// ring in shared memory, the lanes turn them into FP16 in registers
// (cvt.e2m1x2, times the block scale: both exact) straight in the layout of
// an mma.sync operand, and with the running maximum m and sum l of a row
//   S^T = K Q^T           (keys x rows; m16n8k16, the keys as the 16)
//   p = 2^(s - m + 7)     (FP16 for the product, FP32 for l)
//   O^T += V^T P^T        (dims x rows; the dims as the 16)
// Keys and dims, not rows, fill the 16 of the instruction, so 8 rows or
// fewer waste nothing; tcgen05 would need the decoded keys written to shared
// memory first (2 bytes a code against half a byte read).  The order of the
// reduced index is free, so a lane reads consecutive dims of a key: its 32
// nibbles are one 16-byte load at hd = 128.
// m only moves when a score passes it by 2^6 (a vote, no shuffles): weights
// reach 2^14, which FP16 allows.
//
// Chunks of one request are joined by k_attn_join from the rows' (m, l, O)
// in FP32.
//
// Its floor is HBM: hd + hd / 16 bytes a key and head.  Measured (32/8 heads of
// 128; ranges over several boxes): 64 requests of up to 16384 keys 181 to
// 187 us, 3.9 to 4.0 TB/s, 59 to 61 % of a copy's rate; one request of 131071 keys
// 44 us; one of 241 keys (15/5 heads of 64) 4.6 to 4.8 us.  Bound by the lanes'
// work: with all pages in L2 it takes as long, 63 % of the issue slots and 54 %
// of the ALU pipe (the conversions) are used.
#include <cuda_fp16.h>

#include <atomic>
#include <cstdint>

#include "hrb_attn.cuh"
#include "sm100.cuh"

namespace hrb {
namespace {

using namespace sm100;

constexpr uint32_t kTile = 32;   // keys a stage
constexpr uint32_t kWarps = 4;
constexpr uint32_t kStages = 3;

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                    uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Where a tile's parts lie in a stage: pages of 16 tokens (P16) bring two
// records, larger pages 32 tokens of one.  Fixed when the kernel is built, so
// that a load's offset is in its instruction.
template <uint32_t HD, bool P16>
struct Geom {
  static constexpr uint32_t kN = P16 ? 16u : 32u;
  static constexpr uint32_t kKs = kN * (HD / 2u);                 // K scales (K codes at 0)
  static constexpr uint32_t kV = kN * (HD / 2u + HD / 32u);       // V codes
  static constexpr uint32_t kVs = kV + kN * (HD / 2u);            // V scales
  // From tokens 0..15 to 16..31.
  static constexpr uint32_t kCodeHalf = P16 ? 16u * (HD + HD / 16u) : 16u * (HD / 2u);
  static constexpr uint32_t kScaleHalf = P16 ? 16u * (HD + HD / 16u) : 16u * (HD / 32u);
};

template <uint32_t HD, uint32_t NT>
struct Smem {
  static constexpr uint32_t kStageBytes = kTile * (HD + HD / 16u);
  static constexpr uint32_t kRing = kWarps * kStages * kStageBytes;
  static constexpr uint32_t kJoin = kWarps * 8u * NT * (HD + 4u) * 4u;
  static constexpr uint32_t kBuf = kRing > kJoin ? kRing : kJoin;
  static constexpr uint32_t kQ = NT > 2u ? 8u * NT * HD * 2u : 0u;  // Q fragments, see below
  static constexpr uint32_t kScales = kBuf + kQ;               // [256] words
  static constexpr uint32_t kBars = kScales + 1024u;
  static constexpr uint32_t kBytes = kBars + kWarps * kStages * 8u;
};

template <uint32_t HD, uint32_t NT, bool P16>
__global__ void __launch_bounds__(kWarps * 32, NT == 1u ? 4 : 2)
    k_attn_decode(const AttnJob j, uint32_t* __restrict__ error_flag) {
  using S = Smem<HD, NT>;
  using Geo = Geom<HD, P16>;
  constexpr uint32_t kSteps = HD / 16u;           // MMAs along dims; m16 tiles of dims
  constexpr uint32_t kRows = 8u * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  const uint32_t g = lane >> 2, t = lane & 3u;
  uint8_t* ring = smem + warp * kStages * S::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars) + warp * kStages;
  // Every scale byte as a pair of FP16: a load instead of a shift, a
  // conversion and two clamps, which the pipe of the codes' conversions takes.
  uint32_t* scales = reinterpret_cast<uint32_t*>(smem + S::kScales);

  for (uint32_t b = threadIdx.x; b < 256u; b += kWarps * 32u) scales[b] = scale2(b, b);
  if (lane < kStages) mbar_init(full + lane, 1);
  fence_barrier_init();
  __syncwarp();
  griddep_wait();

  const uint32_t n = blockIdx.z, head = blockIdx.y;
  int32_t q0, q_len, kv;
  if (!attn_request(j, n, &q0, &q_len, &kv)) {
    if (blockIdx.x == 0u && threadIdx.x == 0u) atomicOr(error_flag, kErrKvSlot);
    return;
  }
  // Rows r0 .. r0 + rows - 1 of the request's, a block of kRows.
  const int32_t group = static_cast<int32_t>(j.group);
  const uint32_t chunk = blockIdx.x / j.row_blocks;
  const int32_t r0 = static_cast<int32_t>((blockIdx.x - chunk * j.row_blocks) * kRows);
  const int32_t rows = min(q_len * group - r0, static_cast<int32_t>(kRows));
  const int32_t c0 = static_cast<int32_t>(chunk * j.chunk);
  if (rows <= 0 || (c0 >= kv && c0 > 0)) return;
  const int32_t c1 = c0 + min(kv - c0, static_cast<int32_t>(j.chunk));
  const bool whole = kv <= static_cast<int32_t>(j.chunk);  // no other chunk of this request

  // The keys that the rows see, and the tiles of this warp among them.
  const int32_t pre = j.prefix != nullptr ? ld(j.prefix + n) : 0;
  const Seen first = attn_seen(j, kv - q_len + r0 / group, kv, pre);
  const Seen last = attn_seen(j, kv - q_len + (r0 + rows - 1) / group, kv, pre);

  const int32_t* table = j.table + static_cast<uint64_t>(n) * j.table_ld;
  const uint32_t copies = P16 ? 2u : j.cache.page == 32u ? 1u : 4u;
  // Lane l holds the pages of the warp's tile number base + l: -2 past the
  // request's keys, -1 for any negative entry of the table.
  int32_t page_a = -1, page_b = -1, base = 0;
  auto load_pages = [&](int32_t at) {  // tiles number at .. at + 31 of this warp
    base = at;
    // Unsigned: the last tiles' numbers run up to 2^12 keys past kv.
    const uint32_t i = warp + (static_cast<uint32_t>(at) + lane) * kWarps, end = static_cast<uint32_t>(kv);
    const uint32_t k = static_cast<uint32_t>(c0) + i * kTile;
    page_a = k < end ? max(ld(table + (k >> j.cache.page_log2)), -1) : -2;
    page_b = page_a;
    if (P16) page_b = k + 16u < end ? max(ld(table + ((k + 16u) >> 4)), -1) : -2;
  };
  const uint8_t* const head_data = j.cache.data + static_cast<uint64_t>(head) * j.cache.record;
  // Pages outside the cache read as zeros.
  auto issue = [&](int32_t number, uint32_t stage) {
    const int32_t i = static_cast<int32_t>(warp) + number * static_cast<int32_t>(kWarps);
    const uint32_t k = static_cast<uint32_t>(c0 + i * static_cast<int32_t>(kTile));
    const int32_t pa = __shfl_sync(0xFFFFFFFFu, page_a, number - base);
    const int32_t pb = __shfl_sync(0xFFFFFFFFu, page_b, number - base);
    const int32_t page = lane == 1u && P16 ? pb : pa;
    const bool there = static_cast<uint32_t>(page) < j.cache.pages;
    uint8_t* dst = ring + stage * S::kStageBytes;
    uint32_t bytes, from;
    if (j.cache.page <= 32u) {
      bytes = j.cache.record;
      from = 0;
      dst += lane * j.cache.record;
    } else {
      const uint32_t in = k & (j.cache.page - 1u);
      const bool of_scales = (lane & 1u) != 0u;
      bytes = of_scales ? kTile * (HD / 32u) : kTile * (HD / 2u);
      from = (lane >= 2u ? kv_vcodes(j.cache) : 0u) +
             (of_scales ? kv_kscales(j.cache) + in * (HD / 32u) : in * (HD / 2u));
      dst += (lane >= 2u ? Geo::kV : 0u) + (of_scales ? Geo::kKs : 0u);
    }
    const uint32_t in_a = static_cast<uint32_t>(pa) < j.cache.pages ? 1u : 0u;
    const uint32_t in_b = static_cast<uint32_t>(pb) < j.cache.pages ? 1u : 0u;
    // Two records, one, or a tile's part of a larger one.
    const uint32_t total = P16 ? (in_a + in_b) * j.cache.record
                                               : in_a * S::kStageBytes;
    if (lane == 0u) mbar_arrive_expect_tx(full + stage, total);
    __syncwarp();
    if (lane < copies && there) {
      bulk_g2s(dst, head_data + static_cast<uint64_t>(static_cast<uint32_t>(page)) * j.cache.page_stride + from,
               bytes, full + stage);
    }
  };

  // Q: row r of the operand is row r / group of q, head r % group of this
  // key/value head's.  Lane (g, t) holds dims [t HD / 4, (t + 1) HD / 4) of
  // row 8 nt + g as FP16 pairs, its row scaled so that its largest value is
  // in [2^13, 2^14): bf16's 8 bits fit in 11, and what falls under FP16's
  // range is 2^-37 of the row's largest.
  uint32_t qf[NT <= 2u ? NT : 1u][kSteps][2];
  uint32_t* q_smem = reinterpret_cast<uint32_t*>(smem + S::kBuf);
  float row_scale[NT];  // of row 8 nt + g
#pragma unroll
  for (uint32_t nt = 0; nt < NT; ++nt) {
    const int32_t r = static_cast<int32_t>(8u * nt + g);
    uint32_t w[HD / 8u];
#pragma unroll
    for (uint32_t i = 0; i < HD / 8u; ++i) w[i] = 0;
    if (r < rows) {
      const uint64_t row = static_cast<uint64_t>(q0 + (r0 + r) / group);
      const uint32_t h = head * j.group + static_cast<uint32_t>((r0 + r) % group);
      const uint4* src = reinterpret_cast<const uint4*>(j.q + row * j.ldq + h * HD + t * (HD / 4u));
#pragma unroll
      for (uint32_t i = 0; i < HD / 32u; ++i) {
        const uint4 v = ld(src + i);
        w[4u * i] = v.x;
        w[4u * i + 1u] = v.y;
        w[4u * i + 2u] = v.z;
        w[4u * i + 3u] = v.w;
      }
    }
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < HD / 8u; ++i) {
      top = max(top, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
    }
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    const int32_t e = min(max(static_cast<int32_t>(top >> 7), 27), 254) - 127;
    float up = __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
    if (j.scale < 0.f) up = -up;  // the scores' factor is not negative
    row_scale[nt] = __uint_as_float(static_cast<uint32_t>(127 - 13 + e) << 23);
    if (top >= 0x7F80u) row_scale[nt] = NAN;  // Inf or NaN in the row
#pragma unroll
    for (uint32_t i = 0; i < HD / 8u; ++i) {
      const uint32_t h2 = half2_bits(__floats2half2_rn(__uint_as_float(w[i] << 16) * up,
                                                       __uint_as_float(w[i] & 0xFFFF0000u) * up));
      if constexpr (NT <= 2u) {
        qf[nt][i / 2u][i & 1u] = h2;
      } else if (warp == 0u) {
        q_smem[((nt * kSteps + i / 2u) * 32u + lane) * 2u + (i & 1u)] = h2;
      }
    }
  }
  __syncthreads();  // the scales, and Q
  // The lane's two rows of each n tile in S^T and O^T: 8 nt + 2 t + {0, 1}.
  float factor[NT][2], m[NT][2], l[NT][2], slope[NT][2];
  Seen seen[NT][2];
  int32_t pos[NT][2];
  const bool capped = j.softcap != 0.f, wide = j.softcap > kWideCap;
#pragma unroll
  for (uint32_t nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (uint32_t c = 0; c < 2u; ++c) {
      const int32_t r = static_cast<int32_t>(8u * nt + 2u * t + c);
      const float sc = __shfl_sync(0xFFFFFFFFu, row_scale[nt], (2u * t + c) * 4u);
      factor[nt][c] = fmaxf(fabsf(j.scale) * sc, 1.2e-38f) * (capped ? 1.0f : kLog2e);
      m[nt][c] = -INFINITY;
      l[nt][c] = 0.f;
      pos[nt][c] = kv - q_len + (r0 + r) / group;
      seen[nt][c] = attn_seen(j, pos[nt][c], kv, pre);
      if (r >= rows) seen[nt][c].lo = seen[nt][c].hi = seen[nt][c].pre = 0;
      // Inf or NaN in the row: its scores and outputs are NaN, unless it sees no key.
      if (sc != sc && (seen[nt][c].lo < seen[nt][c].hi || seen[nt][c].pre > 0)) factor[nt][c] = sc;
      slope[nt][c] = j.slopes != nullptr && r < rows
                         ? ld(j.slopes + head * j.group + static_cast<uint32_t>((r0 + r) % group)) * kLog2e
                         : 0.f;
    }
  }
  float o[NT][kSteps][4];
#pragma unroll
  for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
    for (uint32_t i = 0; i < kSteps; ++i)
#pragma unroll
      for (uint32_t c = 0; c < 4u; ++c) o[nt][i][c] = 0.f;

  // The warp's tiles: number x is tile warp + x kWarps of the chunk, those
  // below `gap` or from `resume` to `mine` hold keys that a row sees (the
  // prefix, and the window or all).
  auto numbers_to = [&](int32_t k) {  // numbers whose tiles start before key k
    const int32_t tiles = (min(max(k, c0), c1) - c0 + static_cast<int32_t>(kTile) - 1) /
                          static_cast<int32_t>(kTile);
    return (tiles - static_cast<int32_t>(warp) + static_cast<int32_t>(kWarps) - 1) /
           static_cast<int32_t>(kWarps);
  };
  const int32_t gap = numbers_to(first.pre), mine = max(gap, numbers_to(last.hi));
  const int32_t resume = max(gap, min(mine, numbers_to(first.lo + 1 - static_cast<int32_t>(kTile))));
  auto next = [&](int32_t x) { return x >= gap && x < resume ? resume : x; };
  int32_t ahead = next(0);  // next to issue
  load_pages(ahead);
  int32_t at = ahead;       // next to use
  uint32_t in_flight = 0;
  // Pages of the tile in use are read again from lane registers: keep the
  // numbers in use and in flight within the 32 that are loaded.
  for (uint32_t s = 0; s < kStages; ++s) {
    if (ahead < mine && ahead < base + 32) {
      issue(ahead, s);
      ++in_flight;
      ahead = next(ahead + 1);
    }
  }
  uint32_t stage = 0, parity = 0;
  bool ok = true, bad_page = false;
  // Scores take their factor before the maximum: a cap, a bias, or an m that
  // has been far (kFar).
  bool shaped = capped || j.slopes != nullptr;
  while (at < mine) {
    if (in_flight == 0u) {  // the loaded pages are used up
      load_pages(at);
      for (uint32_t s = 0, st = stage; s < kStages; ++s) {
        if (ahead < mine && ahead < base + 32) {
          issue(ahead, st);
          ++in_flight;
          ahead = next(ahead + 1);
        }
        st = st + 1u == kStages ? 0u : st + 1u;
      }
    }
    const int32_t pa = __shfl_sync(0xFFFFFFFFu, page_a, at - base);
    const int32_t pb = __shfl_sync(0xFFFFFFFFu, page_b, at - base);
    const bool bad_a = pa != -2 && static_cast<uint32_t>(pa) >= j.cache.pages;
    const bool bad_b = pb != -2 && static_cast<uint32_t>(pb) >= j.cache.pages;
    const int32_t k0 = c0 + (static_cast<int32_t>(warp) + at * static_cast<int32_t>(kWarps)) *
                                static_cast<int32_t>(kTile);
    ok = mbar_wait(full + stage, parity, error_flag);
    if (!__all_sync(0xFFFFFFFFu, ok)) break;
    const uint8_t* tile = ring + stage * S::kStageBytes;

    // S^T: keys k0 + 16 hf + {g, g + 8}, rows {2t, 2t + 1} of each n tile.
    float s[NT][2][4];
#pragma unroll
    for (uint32_t hf = 0; hf < 2u; ++hf) {
      const uint8_t* kc = tile + hf * Geo::kCodeHalf;
      const uint8_t* ks = tile + Geo::kKs + hf * Geo::kScaleHalf;
      uint32_t w[2][HD / 32u];
      uint32_t sc[2][2];  // the lane's block scales (two blocks at hd 96)
#pragma unroll
      for (uint32_t r = 0; r < 2u; ++r) {
        const uint8_t* p = kc + (g + 8u * r) * (HD / 2u) + t * (HD / 8u);
        if constexpr (HD == 128u) {
          const uint4 v = *reinterpret_cast<const uint4*>(p);
          w[r][0] = v.x;
          w[r][1] = v.y;
          w[r][2] = v.z;
          w[r][3] = v.w;
        } else if constexpr (HD == 64u) {
          const uint2 v = *reinterpret_cast<const uint2*>(p);
          w[r][0] = v.x;
          w[r][1] = v.y;
        } else {
#pragma unroll
          for (uint32_t i = 0; i < HD / 32u; ++i) w[r][i] = *reinterpret_cast<const uint32_t*>(p + 4u * i);
        }
        const uint8_t* q = ks + (g + 8u * r) * (HD / 32u);
        const uint32_t b0 = q[t * (HD / 4u) / 32u];
        sc[r][0] = scales[b0];
        if constexpr (HD == 96u) {
          const uint32_t b1 = q[(t * 24u + 23u) / 32u];
          sc[r][1] = scales[b1];
        } else {
          sc[r][1] = sc[r][0];
        }
      }
#pragma unroll
      for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
        for (uint32_t c = 0; c < 4u; ++c) s[nt][hf][c] = 0.f;
#pragma unroll
      for (uint32_t i = 0; i < HD / 32u; ++i) {
        uint32_t a[2][4];
#pragma unroll
        for (uint32_t r = 0; r < 2u; ++r) {
          e2m1x8_to_f16x2(w[r][i], a[r]);
#pragma unroll
          for (uint32_t d = 0; d < 4u; ++d) {
            // Dims 24 t + 8 i + 2 d of hd 96 pass a block's end inside the lane.
            const uint32_t x = HD == 96u && t * 24u + 8u * i + 2u * d >= 32u * (t * 24u / 32u + 1u)
                                   ? sc[r][1] : sc[r][0];
            a[r][d] = mul2(a[r][d], x);
          }
        }
#pragma unroll
        for (uint32_t st = 0; st < 2u; ++st) {
#pragma unroll
          for (uint32_t nt = 0; nt < NT; ++nt) {
            uint32_t b0, b1;
            if constexpr (NT <= 2u) {
              b0 = qf[nt][2u * i + st][0];
              b1 = qf[nt][2u * i + st][1];
            } else {
              const uint2 b = *reinterpret_cast<const uint2*>(
                  q_smem + ((nt * kSteps + 2u * i + st) * 32u + lane) * 2u);
              b0 = b.x;
              b1 = b.y;
            }
            mma(s[nt][hf], a[0][2u * st], a[1][2u * st], a[0][2u * st + 1u], a[1][2u * st + 1u],
                b0, b1);
          }
        }
      }
    }
    if (bad_a || bad_b) {
      bad_page = true;
#pragma unroll
      for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
        for (uint32_t c = 0; c < 8u; ++c)
          if (c < 4u ? bad_a : bad_b) s[nt][c / 4u][c & 3u] = 0.f;
    }
    // Scores to the exponent of two.  Tiles that all rows see whole (all but
    // a request's last for single tokens) skip the masks.
    const bool clear = (k0 >= last.lo && first.hi - k0 >= static_cast<int32_t>(kTile)) ||
                       first.pre - k0 >= static_cast<int32_t>(kTile);
    if (wide) {  // a branch of its own: the others' arithmetic is not doubled
#pragma unroll
      for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
        for (uint32_t c = 0; c < 8u; ++c) {
          float& x = s[nt][c / 4u][c & 3u];
          x = cap_score<true>(j, x * factor[nt][c & 1u]);
        }
    } else if (shaped) {
#pragma unroll
      for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
        for (uint32_t c = 0; c < 8u; ++c) {
          float& x = s[nt][c / 4u][c & 3u];
          x *= factor[nt][c & 1u];
          if (capped) x = cap_score<false>(j, x);
        }
    }
    if (j.slopes != nullptr) {
#pragma unroll
      for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
        for (uint32_t c = 0; c < 8u; ++c) {
          const uint32_t k = static_cast<uint32_t>(k0) + 16u * (c / 4u) + 8u * ((c >> 1) & 1u) + g;
          const int32_t away = static_cast<int32_t>(static_cast<uint32_t>(pos[nt][c & 1u]) - k);
          s[nt][c / 4u][c & 3u] -= slope[nt][c & 1u] * fabsf(static_cast<float>(away));
        }
    }
    if (!clear) {
#pragma unroll
      for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
        for (uint32_t c = 0; c < 8u; ++c) {
          const uint32_t k = static_cast<uint32_t>(k0) + 16u * (c / 4u) + 8u * ((c >> 1) & 1u) + g;
          if (!attn_sees(seen[nt][c & 1u], k)) s[nt][c / 4u][c & 3u] = -INFINITY;
        }
    }
    // m moves where a score passes it by more than kLazy.
    bool moves = false;
    float top[NT][2];
#pragma unroll
    for (uint32_t nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (uint32_t c = 0; c < 2u; ++c) {
        top[nt][c] = fmaxf(fmaxf(s[nt][0][c], s[nt][0][c + 2u]), fmaxf(s[nt][1][c], s[nt][1][c + 2u])) *
                     (shaped ? 1.0f : factor[nt][c]);
        moves |= top[nt][c] - m[nt][c] > kLazy;
      }
    }
    if (__any_sync(0xFFFFFFFFu, moves)) {
      bool large = false;
#pragma unroll
      for (uint32_t nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (uint32_t c = 0; c < 2u; ++c) {
          float x = top[nt][c];
          x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 16));
          const float to = fmaxf(m[nt][c], x);
          const float keep = to == -INFINITY ? 1.0f : ex2(m[nt][c] - to);
          m[nt][c] = to;
          large |= attn_far(to);
          l[nt][c] *= keep;
#pragma unroll
          for (uint32_t i = 0; i < kSteps; ++i) {
            o[nt][i][c] *= keep;
            o[nt][i][c + 2u] *= keep;
          }
        }
      }
      if (!shaped && __any_sync(0xFFFFFFFFu, large)) {
        shaped = true;
#pragma unroll
        for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
          for (uint32_t c = 0; c < 8u; ++c) s[nt][c / 4u][c & 3u] *= factor[nt][c & 1u];
      }
    }
    // P^T as the B operand: pairs of keys in a lane, rows across lanes.
    uint32_t p[NT][2][2];
#pragma unroll
    for (uint32_t nt = 0; nt < NT; ++nt) {
      const float m0 = m[nt][0] == -INFINITY ? 0.f : kLift - m[nt][0];
      const float m1 = m[nt][1] == -INFINITY ? 0.f : kLift - m[nt][1];
      const float f0 = shaped ? 1.0f : factor[nt][0], f1 = shaped ? 1.0f : factor[nt][1];
#pragma unroll
      for (uint32_t hf = 0; hf < 2u; ++hf) {
#pragma unroll
        for (uint32_t r = 0; r < 2u; ++r) {
          const float x = ex2(fmaf(s[nt][hf][2u * r], f0, m0));
          const float y = ex2(fmaf(s[nt][hf][2u * r + 1u], f1, m1));
          l[nt][0] += x;
          l[nt][1] += y;
          p[nt][hf][r] = transpose8x8(half2_bits(__floats2half2_rn(x, y)));
        }
      }
    }
    if (bad_a || bad_b) {
#pragma unroll
      for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
        for (uint32_t hf = 0; hf < 2u; ++hf)
          if (hf == 0u ? bad_a : bad_b) p[nt][hf][0] = p[nt][hf][1] = 0u;
    }
    // O^T: m16 tile i holds dims D(i, g, 0) as its rows g and D(i, g, 1) as
    // its rows g + 8, two dims of one byte.
#pragma unroll
    for (uint32_t hf = 0; hf < 2u; ++hf) {
      const uint8_t* vc = tile + Geo::kV + hf * Geo::kCodeHalf;
      const uint8_t* vs = tile + Geo::kVs + hf * Geo::kScaleHalf;
      // Words of codes a lane and key (the last half used at hd 96 and 32).
      constexpr uint32_t kWords = (HD + 63u) / 64u;
      uint32_t w[4][kWords], sc[2][2];
#pragma unroll
      for (uint32_t r = 0; r < 4u; ++r) {  // keys 2t, 2t + 1, 2t + 8, 2t + 9
        const uint32_t key = 2u * t + (r & 1u) + 8u * (r >> 1);
        const uint8_t* p8 = vc + key * (HD / 2u);
        if constexpr (HD == 128u) {
          const uint2 v = *reinterpret_cast<const uint2*>(p8 + 8u * g);
          w[r][0] = v.x;
          w[r][1] = v.y;
        } else if constexpr (HD == 96u) {
          w[r][0] = *reinterpret_cast<const uint32_t*>(p8 + 4u * g);
          w[r][1] = *reinterpret_cast<const uint16_t*>(p8 + 32u + 2u * g);
        } else if constexpr (HD == 64u) {
          w[r][0] = *reinterpret_cast<const uint32_t*>(p8 + 4u * g);
        } else {
          w[r][0] = *reinterpret_cast<const uint16_t*>(p8 + 2u * g);
        }
      }
#pragma unroll
      for (uint32_t r = 0; r < 2u; ++r) {
        const uint8_t* q = vs + (2u * t + 8u * r) * (HD / 32u);
        const uint32_t b = HD == 128u ? g >> 1 : HD == 32u ? 0u : g >> 2;
        sc[r][0] = __byte_perm(scales[q[b]], scales[q[b + HD / 32u]], 0x5410);
        sc[r][1] = HD == 96u ? __byte_perm(scales[q[2]], scales[q[2u + HD / 32u]], 0x5410) : sc[r][0];
      }
#pragma unroll
      for (uint32_t x = 0; x < kWords; ++x) {
        uint32_t lo[2][4], hi[2][4];  // of the key pairs (2t, 2t + 1) and 8 further
#pragma unroll
        for (uint32_t r = 0; r < 2u; ++r) {
          const uint32_t a = w[2u * r][x], b = w[2u * r + 1u][x];
          e2m1x8_to_f16x2((a & 0x0F0F0F0Fu) | ((b << 4) & 0xF0F0F0F0u), lo[r]);
          e2m1x8_to_f16x2(((a >> 4) & 0x0F0F0F0Fu) | (b & 0xF0F0F0F0u), hi[r]);
        }
#pragma unroll
        for (uint32_t d = 0; d < 4u; ++d) {
          const uint32_t i = 4u * x + d;
          if (i < kSteps) {
            const uint32_t which = HD == 96u && x == 1u ? 1u : 0u;
            const uint32_t a0 = mul2(lo[0][d], sc[0][which]), a1 = mul2(hi[0][d], sc[0][which]);
            const uint32_t a2 = mul2(lo[1][d], sc[1][which]), a3 = mul2(hi[1][d], sc[1][which]);
#pragma unroll
            for (uint32_t nt = 0; nt < NT; ++nt) {
              mma(o[nt][i], a0, a1, a2, a3, p[nt][hf][0], p[nt][hf][1]);
            }
          }
        }
      }
    }
    __syncwarp();  // all lanes have read the stage
    --in_flight;
    at = next(at + 1);
    if (ahead < mine && ahead < base + 32) {
      issue(ahead, stage);
      ++in_flight;
      ahead = next(ahead + 1);
    }
    if (++stage == kStages) {
      stage = 0;
      parity ^= 1u;
    }
  }
  if (!ok) {  // timed out: wait (bounded) for the copies in flight
    while (in_flight-- > 0u) {
      mbar_wait(full + stage, parity, error_flag);
      if (++stage == kStages) {
        stage = 0;
        parity ^= 1u;
      }
    }
  }
  if (bad_page && lane == 0u) atomicOr(error_flag, kErrKvSlot);

  // Join the warps: rows of (m, l, O) in shared memory over the rings.
  __syncthreads();
  constexpr uint32_t kLd = HD + 4u;
  float* mine_o = reinterpret_cast<float*>(smem) + warp * kRows * kLd;
#pragma unroll
  for (uint32_t nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (uint32_t c = 0; c < 2u; ++c) {
      float x = l[nt][c];
      x += __shfl_xor_sync(0xFFFFFFFFu, x, 4);
      x += __shfl_xor_sync(0xFFFFFFFFu, x, 8);
      x += __shfl_xor_sync(0xFFFFFFFFu, x, 16);
      float* to = mine_o + (8u * nt + 2u * t + c) * kLd;
      if (g == 0u) {
        to[HD] = m[nt][c];
        to[HD + 1u] = x;
      }
#pragma unroll
      for (uint32_t i = 0; i < kSteps; ++i) {
        uint32_t d;
        if constexpr (HD == 128u) {
          d = 16u * g + 2u * i;
        } else if constexpr (HD == 32u) {
          d = 4u * g + 2u * i;
        } else {
          d = i < 4u ? 8u * g + 2u * i : 64u + 4u * g + 2u * (i - 4u);
        }
        to[d] = o[nt][i][c];
        to[d + 1u] = o[nt][i][c + 2u];
      }
    }
  }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(smem);
  for (int32_t r = static_cast<int32_t>(warp); r < rows; r += static_cast<int32_t>(kWarps)) {
    float top = -INFINITY;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) top = fmaxf(top, all[(w * kRows + r) * kLd + HD]);
    float part[kWarps], sum = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
      const float mw = all[(w * kRows + r) * kLd + HD];
      part[w] = mw == -INFINITY ? 0.f : ex2(mw - top);
      // A row of NaNs alone has m = -inf and l = NaN.
      const float lw = all[(w * kRows + r) * kLd + HD + 1u];
      sum += mw == -INFINITY ? lw : lw * part[w];
      if (mw == -INFINITY && lw != 0.f) part[w] = 1.f;
    }
    const uint64_t row = static_cast<uint64_t>(q0 + (r0 + r) / group);
    const uint32_t h = head * j.group + static_cast<uint32_t>((r0 + r) % group);
    const uint64_t cell = (static_cast<uint64_t>(chunk) * j.total_q + row) * j.heads + h;
    const float inv = sum != 0.f ? 1.0f / sum : 0.f;
#pragma unroll
    for (uint32_t b = 0; b < HD / 32u; ++b) {
      float x = 0.f;
#pragma unroll
      for (uint32_t w = 0; w < kWarps; ++w) {
        x += part[w] * all[(w * kRows + r) * kLd + 32u * b + lane];
      }
      if (whole) {
        write_block(j, row, h, b, lane, x * inv, error_flag);
      } else {
        j.part_o[cell * HD + 32u * b + lane] = x;
      }
    }
    if (!whole && lane == 0u) j.part_ml[cell] = make_float2(top, sum);
  }
}

// Joins the chunks of a request's rows, W warps a row and head, each summing
// every W-th chunk (many chunks have many loads in flight; their order does
// not depend on anything but their number).
constexpr uint32_t kJoinWarps = 8;

template <uint32_t W>
__global__ void __launch_bounds__(kJoinWarps * 32)
    k_attn_join(const AttnJob j, uint32_t* __restrict__ error_flag) {
  __shared__ float part[kJoinWarps][W > 1u ? 128 : 1], sums[kJoinWarps];
  const uint32_t lane = threadIdx.x & 31u, hd = j.cache.hd;
  const uint32_t warp = W > 1u ? threadIdx.x >> 5 : 0u;
  const uint32_t cell = W > 1u ? blockIdx.x : blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
  const uint32_t r = cell / j.heads, h = cell % j.heads;
  griddep_wait();
  int32_t q0, q_len, kv;
  attn_request(j, blockIdx.y, &q0, &q_len, &kv);
  if (static_cast<int32_t>(r) >= q_len) return;
  const uint64_t row = static_cast<uint64_t>(q0) + r, unit = row * j.heads + h;
  const uint32_t chunks = (static_cast<uint32_t>(kv) + j.chunk - 1u) / j.chunk;
  if (chunks <= 1u) return;
  // k_attn_prompt left the request out: there is nothing to join.
  if (j.tiles != nullptr && !attn_tiles_fit(j, attn_first_tile(j, blockIdx.y), kv)) return;
  const uint64_t stride = static_cast<uint64_t>(j.total_q) * j.heads;
  float top = -INFINITY;
  for (uint32_t c = lane; c < chunks; c += 32u) top = fmaxf(top, j.part_ml[c * stride + unit].x);
#pragma unroll
  for (uint32_t d = 16; d > 0; d /= 2u) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
  float sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (uint32_t c = warp; c < chunks; c += W) {
    const float2 ml = j.part_ml[c * stride + unit];
    const float* o = j.part_o + (c * stride + unit) * hd + lane;
    const float w = ml.x == -INFINITY ? (ml.y != 0.f ? 1.f : 0.f) : ex2(ml.x - top);
    sum += ml.y * w;
#pragma unroll
    for (uint32_t b = 0; b < 4u; ++b) {
      if (b < hd / 32u) x[b] += w * o[32u * b];
    }
  }
  if constexpr (W == 1u) {
    const float inv = sum != 0.f ? 1.0f / sum : 0.f;
#pragma unroll
    for (uint32_t b = 0; b < 4u; ++b) {
      if (b < hd / 32u) write_block(j, row, h, b, lane, x[b] * inv, error_flag);
    }
    return;
  }
#pragma unroll
  for (uint32_t b = 0; b < 4u; ++b) part[warp][W > 1u ? 32u * b + lane : 0u] = x[b];
  if (lane == 0u) sums[warp] = sum;
  __syncthreads();
  if (warp >= hd / 32u) return;
  float y = 0.f, all = 0.f;
#pragma unroll
  for (uint32_t w = 0; w < kJoinWarps; ++w) {
    y += part[w][W > 1u ? 32u * warp + lane : 0u];
    all += sums[w];
  }
  write_block(j, row, h, warp, lane, y * (all != 0.f ? 1.0f / all : 0.f), error_flag);
}

template <uint32_t HD, uint32_t NT, bool P16>
cudaError_t launch(const AttnJob& job, uint32_t chunks, uint32_t* err, cudaStream_t stream) {
  static std::atomic<uint64_t> set{0};  // devices whose limit is raised
  if (((set.load(std::memory_order_relaxed) >> (job.device & 63u)) & 1u) == 0u || job.device > 63u) {
    const cudaError_t st = cudaFuncSetAttribute(
        k_attn_decode<HD, NT, P16>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<HD, NT>::kBytes);
    if (st != cudaSuccess) return st;
    set.fetch_or(uint64_t{1} << (job.device & 63u), std::memory_order_relaxed);
  }
  AttnJob j = job;
  j.row_blocks = (job.max_q * job.group + 8u * NT - 1u) / (8u * NT);
  return launch_early(k_attn_decode<HD, NT, P16>,
                      dim3(chunks * j.row_blocks, job.cache.kv_heads, job.seqs), kWarps * 32,
                      Smem<HD, NT>::kBytes, stream, j, err);
}

template <uint32_t HD, uint32_t NT>
cudaError_t launch_page(const AttnJob& job, uint32_t chunks, uint32_t* err, cudaStream_t stream) {
  return job.cache.page == 16u ? launch<HD, NT, true>(job, chunks, err, stream)
                               : launch<HD, NT, false>(job, chunks, err, stream);
}

template <uint32_t HD>
cudaError_t launch_rows(const AttnJob& job, uint32_t rows, uint32_t chunks, uint32_t* err,
                        cudaStream_t stream) {
  if (rows <= 8u) return launch_page<HD, 1>(job, chunks, err, stream);
  if (rows <= 16u) return launch_page<HD, 2>(job, chunks, err, stream);
  return launch_page<HD, 4>(job, chunks, err, stream);
}

}  // namespace

int launch_attn_join(const AttnJob& job, cudaStream_t stream, uint32_t* error_flag) {
  const uint32_t cells = job.max_q * job.heads;
  const uint32_t chunks = (job.max_kv + job.chunk - 1u) / job.chunk;
  // A block a row and head where there are many chunks (74 of one request:
  // 32 blocks), else a warp.
  const bool many = chunks > 8u;
  const dim3 grid(many ? cells : (cells + kJoinWarps - 1u) / kJoinWarps, job.seqs);
  const cudaError_t st =
      many ? launch_early(k_attn_join<kJoinWarps>, grid, kJoinWarps * 32, 0, stream, job, error_flag)
           : launch_early(k_attn_join<1>, grid, kJoinWarps * 32, 0, stream, job, error_flag);
  return st == cudaSuccess ? 1 : -1;
}

uint32_t attn_decode_chunk(const AttnJob& job, uint64_t total_kv, int sm_count) {
  // Blocks that the GPU holds at once (4 an SM with one n tile, 2 else; their
  // registers).  Requests of one length take one wave of chunks, others four
  // smaller ones that even out (64 requests of 4 K to 16 K keys: 185 us with
  // four, 225 with one; one of 131071 keys 47 and 53).  Chunks have 256 keys at
  // least, and a request 128 chunks at most.
  const uint32_t rows = job.max_q * job.group, nt = rows <= 8u ? 1u : rows <= 16u ? 2u : 4u;
  const uint64_t row_blocks = (rows + 8u * nt - 1u) / (8u * nt);
  const uint64_t wave = static_cast<uint64_t>(sm_count) * (nt == 1u ? 4u : 2u);
  const uint64_t units = job.cache.kv_heads * row_blocks;  // chunks of all of these are blocks
  uint64_t chunk;
  if (total_kv == static_cast<uint64_t>(job.seqs) * job.max_kv) {
    const uint64_t each = wave / (units * job.seqs);
    chunk = each > 1u ? (job.max_kv + each - 1u) / each : job.max_kv;
  } else {
    chunk = total_kv * units / (4u * wave);
  }
  const uint64_t least = (static_cast<uint64_t>(job.max_kv) + 127u) / 128u;
  if (chunk < least) chunk = least;
  if (chunk < 256u) chunk = 256u;
  chunk = (chunk + kWarps * kTile - 1u) / (kWarps * kTile) * (kWarps * kTile);
  return static_cast<uint32_t>(chunk < 0x40000000u ? chunk : 0x40000000u);
}

int launch_attn_decode(const AttnJob& job, uint32_t* error_flag, cudaStream_t stream) {
  const uint32_t rows = job.max_q * job.group;
  const uint32_t chunks = job.max_kv == 0u ? 1u : (job.max_kv + job.chunk - 1u) / job.chunk;
  cudaError_t st;
  switch (job.cache.hd) {
    case 32: st = launch_rows<32>(job, rows, chunks, error_flag, stream); break;
    case 64: st = launch_rows<64>(job, rows, chunks, error_flag, stream); break;
    case 96: st = launch_rows<96>(job, rows, chunks, error_flag, stream); break;
    default: st = launch_rows<128>(job, rows, chunks, error_flag, stream); break;
  }
  if (st != cudaSuccess) return -1;
  if (chunks == 1u) return 1;
  return launch_attn_join(job, stream, error_flag) < 0 ? -1 : 2;
}

}  // namespace hrb
