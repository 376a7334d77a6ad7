// Job descriptors and launchers of the serving kernels (section 11 of
// hrb_gemm.h), and what their entry points (serve.cu) use of a context.
// Internal to libhrb_gemm.so.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "hrb_gemm.h"
#include "hrb_kv.cuh"

namespace hrb {

// A plain load.  The kernels start before the one that writes their inputs
// has ended (launch_early), so these are not loads of data that is constant
// for the kernel's life (__ldg, which may also be moved ahead of the wait).
template <typename T>
__device__ __forceinline__ T ld(const T* p) {
  return *p;
}

// Launches a kernel that may start while the one before it in the stream
// still runs (programmatic stream serialisation): it calls griddep_wait()
// before it touches global memory.
template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, uint32_t threads, size_t smem,
                         cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

// Context fields for serve.cu (defined in capi.cu).
cudaStream_t ctx_stream(const hrb_ctx* ctx, void* stream);
uint32_t* ctx_error_word(const hrb_ctx* ctx);
int ctx_sm_count(const hrb_ctx* ctx);
void ctx_count_launches(hrb_ctx* ctx, uint32_t n);
// The context's scratch of the serving calls, grown to `bytes`, for a call on
// `stream`.
hrb_status ctx_serve_scratch(hrb_ctx* ctx, size_t bytes, cudaStream_t stream, void** out);

struct BlocksJob {
  const int32_t *cached, *fresh, *free_pages, *head_in;
  int32_t *head_out, *table, *q_start, *kv_len, *slots, *pos;
  uint32_t seqs, page_log2, nfree, table_ld, max_tokens;
};
void launch_block_tables(const BlocksJob& job, uint32_t* error_flag, cudaStream_t stream);

struct QkvJob {
  KvCache cache;
  const void* x[3];       // q, k, v
  uint64_t ld[3];         // elements
  const float* norm[2];   // of q and k, or null
  const float2* rope;     // [max_pos][half], or null
  const int32_t* pos;     // [axes][tokens]
  const int32_t* slots;
  void* q_out;
  uint64_t ldqo;
  float eps;
  uint32_t tokens, heads, max_pos, half, interleaved;
  uint32_t cut[2];        // first pairs of axes 1 and 2 (half where there is none)
};
// vec: every row starts at a multiple of four elements' bytes.
void launch_qkv_append(const QkvJob& job, bool bf16, bool vec, uint32_t* error_flag, int sm_count,
                       cudaStream_t stream);
void launch_kv_read(const KvCache& cache, const int32_t* slots, uint32_t tokens, uint32_t dtype,
                    void* k, void* v, uint32_t* error_flag, cudaStream_t stream);

struct AttnJob {
  KvCache cache;
  const uint16_t* q;      // BF16 bits
  uint64_t ldq;
  const int32_t *q_start, *kv_len, *table, *prefix;
  const float* slopes;
  uint16_t* out;          // BF16 bits, or null
  uint64_t ldo;
  int8_t* oq;             // or null
  uint8_t* oscale;
  uint64_t ldoq;
  uint32_t vec_rule;
  uint32_t seqs, heads, group, total_q, max_q, max_kv, table_ld;
  uint32_t causal, window;
  uint32_t device;
  float scale, softcap;
  float cap_inv, cap_in, cap_out;  // 1 / softcap, 2 log2(e) / softcap, softcap * log2(e)
  // Keys a block of the split kernels takes, and the chunks' results: rows
  // of (m, l) and O, [chunk][total_q][heads] and the same by [hd].
  uint32_t chunk;
  uint32_t row_blocks;    // of a request, in the decoding kernel
  float2* part_ml;
  float* part_o;
  // The prompt kernel's decoded keys: [kv_heads][tiles_cap] tiles.
  uint8_t* tiles;
  uint32_t tiles_cap, tile_stride;
};

// Rows [q0, q0 + q_len) and keys of request n, held to what the descriptor
// says there are; false (and no rows) where the lists contradict it.
__device__ __forceinline__ bool attn_request(const AttnJob& j, uint32_t n, int32_t* q0,
                                             int32_t* q_len, int32_t* kv) {
  // From L2: k_attn_prompt asks before it waits.
  *q0 = __ldcg(j.q_start + n);
  *q_len = __ldcg(j.q_start + n + 1u) - *q0;
  const int32_t len = __ldcg(j.kv_len + n);
  *kv = min(max(len, 0), static_cast<int32_t>(j.max_kv));
  if (*q0 >= 0 && *q_len >= 0 && *q_len <= static_cast<int32_t>(j.max_q) &&
      *q0 <= static_cast<int32_t>(j.total_q) - *q_len && len <= static_cast<int32_t>(j.max_kv)) {
    return true;
  }
  *q_len = 0;
  return false;
}

// The keys row position i of request n may see: [lo, hi) and [0, pre), both
// held to the request's keys.
struct Seen {
  int32_t lo, hi, pre;
};
__device__ __forceinline__ Seen attn_seen(const AttnJob& j, int32_t i, int32_t kv, int32_t pre) {
  Seen s;
  if (!j.causal) {
    s.lo = 0;
    s.hi = kv;
    s.pre = 0;
  } else {
    s.hi = min(max(i + 1, 0), kv);
    s.lo = j.window != 0 && i >= static_cast<int32_t>(j.window)
               ? i + 1 - static_cast<int32_t>(j.window) : 0;
    s.pre = min(max(pre, 0), kv);
  }
  return s;
}
// A tile's last keys may pass 2^31 where the request's do not.
__device__ __forceinline__ bool attn_sees(const Seen& s, uint32_t k) {
  return (k >= static_cast<uint32_t>(s.lo) && k < static_cast<uint32_t>(s.hi)) ||
         k < static_cast<uint32_t>(s.pre);
}

// FP32 to BF16 bits, to nearest even.
__device__ __forceinline__ uint16_t attn_bf16(float x) {
  uint16_t r;
  asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(x));
  return r;
}

// Any number of rows; few (serve.cu).  Returns the launches, or -1.
uint32_t attn_decode_chunk(const AttnJob& job, uint64_t total_kv, int sm_count);
int launch_attn_decode(const AttnJob& job, uint32_t* error_flag, cudaStream_t stream);

// Joins the chunks' results of all rows.
int launch_attn_join(const AttnJob& job, cudaStream_t stream, uint32_t* error_flag);

// Any number of rows.  Scratch for attn_prompt_tiles tiles a key/value head.
uint64_t attn_prompt_tiles(const AttnJob& job, uint64_t total_kv, uint32_t* stride);
uint64_t attn_prompt_tile_bytes(const AttnJob& job);
uint32_t attn_prompt_chunk(const AttnJob& job, int sm_count);
int launch_attn_prompt(const AttnJob& job, uint32_t* error_flag, cudaStream_t stream);

}  // namespace hrb
