// hrb_block_tables: pages and slots of a step's tokens from request lengths.
//
// One launch with no communication between its blocks.  Block b owns the
// tokens [256 b, 256 b + 256) of the step and an equal share of the requests.
// Every block scans all requests' lengths (8 bytes each, from L2 after the
// first block), which gives each request its first token (exclusive sum of
// fresh) and its first free-list entry (exclusive sum of need); the requests
// with tokens in the block's range go to a shared list, in order, and each
// token finds its request there by bisection.  A token's page comes from the
// old part of the table or straight from the free list, never from an entry
// another block writes.  The token at a new page's first position writes the
// page's table entry: a new page always starts at one of the step's tokens.
//
// Bound by latency: the lengths' loads, one block scan and two dependent
// loads (free list or table): 3.7 us for 8 requests, 4.9 us for 1024 with
// 67 K tokens.
#include <cstdint>

#include "hrb_kv.cuh"
#include "hrb_serve.cuh"
#include "sm100.cuh"

namespace hrb {
namespace {

constexpr uint32_t kThreads = 256;  // and tokens a block

constexpr uint32_t kMost = 0x80000000u;  // sums are held to this: more than any max_tokens or nfree

__device__ __forceinline__ uint32_t held_add(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;
  return s < a ? kMost : min(s, kMost);
}

// Sums of two values over the threads before each one; `total` receives the
// block's sums.  HELD: for values whose sums may pass kMost.
template <bool HELD>
__device__ __forceinline__ uint2 block_scan(uint2 v, uint2* total, uint2* warp_sums) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  auto add = [](uint2 a, uint2 b) {
    return HELD ? make_uint2(held_add(a.x, b.x), held_add(a.y, b.y)) : make_uint2(a.x + b.x, a.y + b.y);
  };
  const uint2 own = v;
#pragma unroll
  for (uint32_t d = 1; d < 32; d *= 2) {
    const uint2 u = make_uint2(__shfl_up_sync(0xFFFFFFFFu, v.x, d), __shfl_up_sync(0xFFFFFFFFu, v.y, d));
    if (lane >= d) v = add(v, u);
  }
  if (lane == 31u) warp_sums[warp] = v;
  if constexpr (HELD) {
    v = make_uint2(__shfl_up_sync(0xFFFFFFFFu, v.x, 1), __shfl_up_sync(0xFFFFFFFFu, v.y, 1));
    if (lane == 0u) v = make_uint2(0, 0);
  } else {
    v = make_uint2(v.x - own.x, v.y - own.y);
  }
  __syncthreads();
  uint2 before = make_uint2(0, 0), all = make_uint2(0, 0);
#pragma unroll
  for (uint32_t w = 0; w < kThreads / 32u; ++w) {
    const uint2 s = warp_sums[w];
    if (w < warp) before = add(before, s);
    all = add(all, s);
  }
  __syncthreads();
  *total = all;
  return add(v, before);
}

template <bool H>
struct Held {
  static constexpr bool value = H;
};

struct Request {
  uint32_t seq, first, cached, have, base;  // first token, cached tokens, old pages, free entry
};

__global__ void __launch_bounds__(kThreads)
    k_block_tables(const BlocksJob j, uint32_t* __restrict__ error_flag) {
  __shared__ Request list[kThreads];
  __shared__ uint2 warp_sums[kThreads / 32u];
  const uint32_t t0 = blockIdx.x * kThreads, t1 = min(t0 + kThreads, j.max_tokens);
  const uint32_t share = (j.seqs + gridDim.x - 1u) / gridDim.x;
  const uint32_t s0 = blockIdx.x * share, s1 = s0 + share;
  sm100::griddep_wait();
  const uint32_t head = j.head_in != nullptr ? static_cast<uint32_t>(*j.head_in) : 0u;
  const uint32_t mask = (1u << j.page_log2) - 1u;
  bool bad = false, short_of = false;
  uint2 carry = make_uint2(0, 0);
  uint32_t listed = 0;  // requests listed so far
  // Scans the requests.  Held<false> takes lengths and sums as they are, and
  // gives false where some are out of range: Held<true> then does it again.
  auto scan = [&](auto which) -> bool {
    constexpr bool kHeld = decltype(which)::value;
    bool fits = true;
    carry = make_uint2(0, 0);
    listed = 0;
    for (uint32_t c = 0; c < j.seqs; c += kThreads) {
      const uint32_t i = c + threadIdx.x;
      int32_t cached = 0, fresh = 0;
      if (i < j.seqs) {
        cached = ld(j.cached + i);
        fresh = ld(j.fresh + i);
      }
      const bool odd = (cached | fresh | static_cast<int32_t>(
                            static_cast<uint32_t>(cached) + static_cast<uint32_t>(fresh))) < 0;
      if constexpr (kHeld) {
        bad |= odd;
        cached = max(cached, 0);
        fresh = min(max(fresh, 0), 0x7FFFFFFF - cached);
      }
      const uint32_t have = (static_cast<uint32_t>(cached) + mask) >> j.page_log2;
      const uint32_t need =
          ((static_cast<uint32_t>(cached) + static_cast<uint32_t>(fresh) + mask) >> j.page_log2) -
          have;
      // kThreads lengths under 2^18, of pages under 2^15 each, have sums under
      // 2^26 and 2^23; a longer or odd one counts 2^23 pages here, and shows.
      const uint32_t pages = !kHeld && (odd || fresh >= 1 << 18) ? 1u << 23 : need;
      uint2 total;
      const uint2 sum =
          block_scan<kHeld>(make_uint2(static_cast<uint32_t>(fresh), pages), &total, warp_sums);
      const uint32_t first = kHeld ? held_add(carry.x, sum.x) : carry.x + sum.x;
      const uint32_t base = kHeld ? held_add(carry.y, sum.y) : carry.y + sum.y;
      carry.x = kHeld ? held_add(carry.x, total.x) : carry.x + total.x;
      carry.y = kHeld ? held_add(carry.y, total.y) : carry.y + total.y;
      fits = fits && (kHeld || (total.y < 1u << 23 && carry.x < kMost));
      if (i < j.seqs && i >= s0 && i < s1) {
        j.q_start[i] = static_cast<int32_t>(kHeld ? min(first, 0x7FFFFFFFu) : first);
        j.kv_len[i] = cached + fresh;
      }
      // At most one request a token: the range holds kThreads tokens, and a sum
      // that was held starts past all ranges.
      const bool mine = fits && fresh > 0 && first < t1 && first + static_cast<uint32_t>(fresh) > t0;
      uint2 in_chunk;
      const uint2 rank = block_scan<false>(make_uint2(mine ? 1u : 0u, 0u), &in_chunk, warp_sums);
      if (mine) list[listed + rank.x] = Request{i, first, static_cast<uint32_t>(cached), have, base};
      listed += in_chunk.x;
    }
    return fits;
  };
  if (!scan(Held<false>{})) scan(Held<true>{});
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    j.q_start[j.seqs] = static_cast<int32_t>(min(carry.x, 0x7FFFFFFFu));
    if (j.head_out != nullptr) *j.head_out = static_cast<int32_t>(head + carry.y);
    short_of |= carry.x > j.max_tokens;
  }
  const uint32_t t = t0 + threadIdx.x;
  if (t < t1) {
    int32_t slot = -1, pos = 0;
    if (t < carry.x) {
      uint32_t lo = 0, hi = listed;  // the last listed request that starts at or before t
      while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (list[mid].first <= t) {
          lo = mid;
        } else {
          hi = mid;
        }
      }
      const Request r = list[lo];
      const uint32_t p = r.cached + (t - r.first), n = p >> j.page_log2;
      pos = static_cast<int32_t>(p);
      int32_t page = -1;
      if (n < j.table_ld) {
        int32_t* entry = j.table + static_cast<uint64_t>(r.seq) * j.table_ld + n;
        if (n < r.have) {
          page = *entry;
        } else {
          const uint64_t f = uint64_t{head} + r.base + (n - r.have);
          if (f < j.nfree) page = ld(j.free_pages + f);
          if ((p & mask) == 0) *entry = page;
        }
      }
      // A page whose slots pass 31 bits is no page of any cache.
      if (page >= 0 && page <= static_cast<int32_t>(0x7FFFFFFFu >> j.page_log2)) {
        slot = static_cast<int32_t>((static_cast<uint32_t>(page) << j.page_log2) + (p & mask));
      } else {
        short_of = true;
      }
    }
    j.slots[t] = slot;
    if (j.pos != nullptr) j.pos[t] = pos;
  }
  if (bad || short_of) atomicOr(error_flag, kErrKvPages);
}

}  // namespace

void launch_block_tables(const BlocksJob& job, uint32_t* error_flag, cudaStream_t stream) {
  const uint32_t grid = (job.max_tokens + kThreads - 1u) / kThreads;
  launch_early(k_block_tables, dim3(grid != 0 ? grid : 1u), kThreads, 0, stream, job, error_flag);
}

}  // namespace hrb
