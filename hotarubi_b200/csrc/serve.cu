// The entry points of the serving calls (section 11 of hrb_gemm.h): argument
// checks, jobs, dispatch.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "hrb_gemm.h"
#include "hrb_kernels.cuh"
#include "hrb_serve.cuh"

namespace {

hrb_status refuse(hrb_ctx* ctx, hrb_status status, const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return hrb::ctx_fail(ctx, status, buf);
}

hrb_status launched(hrb_ctx* ctx, uint32_t n, const char* what) {
  hrb::ctx_count_launches(ctx, n);
  const cudaError_t err = cudaGetLastError();
  if (err == cudaSuccess) return HRB_OK;
  return refuse(ctx, err == cudaErrorMemoryAllocation ? HRB_ENOMEM : HRB_ECUDA, "%s: %s", what,
                cudaGetErrorString(err));
}

bool on(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

bool page_size(uint32_t page) {
  return page >= 16u && page <= 256u && (page & (page - 1u)) == 0u;
}

hrb_status check_cache(hrb_ctx* ctx, const hrb_kv_cache* c) {
  if (!page_size(c->page)) {
    return refuse(ctx, HRB_EINVAL, "pages of %u tokens (16, 32, 64, 128 or 256)", c->page);
  }
  if (c->hd == 0u || c->hd % 32u != 0u || c->hd > 128u) {
    return refuse(ctx, HRB_EINVAL, "head of %u dims (32, 64, 96 or 128)", c->hd);
  }
  if (c->kv_heads == 0u || c->kv_heads > 65535u || c->pages == 0u ||
      uint64_t{c->pages} * c->page > 0x7FFFFFFFull) {
    return refuse(ctx, HRB_EINVAL, "cache of %u pages of %u tokens, %u heads", c->pages, c->page,
                  c->kv_heads);
  }
  if (c->data == nullptr || !on(c->data, 16)) {
    return refuse(ctx, HRB_EINVAL, "cache data missing or not 16-byte aligned");
  }
  if (c->page_stride != 0u &&
      (c->page_stride % 16u != 0u ||
       c->page_stride < uint64_t{c->kv_heads} * hrb_kv_record_bytes(c->page, c->hd))) {
    return refuse(ctx, HRB_EINVAL, "cache page stride of %llu bytes",
                  static_cast<unsigned long long>(c->page_stride));
  }
  return HRB_OK;
}

hrb_status check_attn(hrb_ctx* ctx, const hrb_attn_desc* d) {
  if (d == nullptr) return refuse(ctx, HRB_EINVAL, "null attention descriptor");
  const hrb_status st = check_cache(ctx, &d->cache);
  if (st != HRB_OK) return st;
  const uint64_t width = uint64_t{d->heads} * d->cache.hd;
  if (d->heads == 0u || d->heads % d->cache.kv_heads != 0u || d->heads > 65535u) {
    return refuse(ctx, HRB_EINVAL, "%u query heads over %u key/value heads", d->heads,
                  d->cache.kv_heads);
  }
  if (d->seqs > 65535u) return refuse(ctx, HRB_EINVAL, "%u requests (at most 65535)", d->seqs);
  if (d->total_q > 0x7FFFFFFFu || d->max_q > d->total_q || d->max_kv > 0x7FFFFFFFu ||
      uint64_t{d->max_q} * (d->heads / d->cache.kv_heads) > 128ull * 65535u) {
    return refuse(ctx, HRB_EINVAL, "%u rows, at most %u a request, %u keys", d->total_q, d->max_q,
                  d->max_kv);
  }
  if (d->total_q != 0u && (d->seqs == 0u || d->max_q == 0u)) {
    return refuse(ctx, HRB_EINVAL, "%u rows of no request", d->total_q);
  }
  if (d->causal == 0u && (d->window != 0u || d->prefix != nullptr)) {
    return refuse(ctx, HRB_EINVAL, "a window or a prefix needs causal attention");
  }
  if (d->window > 0x7FFFFFFFu) return refuse(ctx, HRB_EINVAL, "window of %u keys", d->window);
  // A NaN fails these too.
  if (!(d->scale > -3.0e38f && d->scale < 3.0e38f) || !(d->softcap >= 0.f && d->softcap < 3.0e38f)) {
    return refuse(ctx, HRB_EINVAL, "score scale %g, cap %g", static_cast<double>(d->scale),
                  static_cast<double>(d->softcap));
  }
  if (d->total_q == 0u) return HRB_OK;
  if (d->q == nullptr || d->q_start == nullptr || d->kv_len == nullptr ||
      (d->max_kv != 0u && d->table == nullptr)) {
    return refuse(ctx, HRB_EINVAL, "null buffer");
  }
  if (!on(d->q, 16) || d->ldq % 8u != 0u || d->ldq < width) {
    return refuse(ctx, HRB_EINVAL, "query rows of %llu elements: 16-byte aligned, at least %llu",
                  static_cast<unsigned long long>(d->ldq), static_cast<unsigned long long>(width));
  }
  if (!on(d->q_start, 4) || !on(d->kv_len, 4) || !on(d->table, 4) || !on(d->prefix, 4) ||
      !on(d->slopes, 4)) {
    return refuse(ctx, HRB_EINVAL, "a list is not 4-byte aligned");
  }
  if (d->table_ld < (uint64_t{d->max_kv} + d->cache.page - 1u) / d->cache.page) {
    return refuse(ctx, HRB_EINVAL, "table rows of %u pages for %u keys", d->table_ld, d->max_kv);
  }
  if (d->out == nullptr && d->oq == nullptr) return refuse(ctx, HRB_EINVAL, "missing output");
  if ((d->oq == nullptr) != (d->oscale == nullptr)) {
    return refuse(ctx, HRB_EINVAL, "give both MXINT8 output codes and scales, or neither");
  }
  if (d->out != nullptr && (!on(d->out, 16) || d->ldo % 8u != 0u || d->ldo < width)) {
    return refuse(ctx, HRB_EINVAL, "output rows of %llu elements: 16-byte aligned, at least %llu",
                  static_cast<unsigned long long>(d->ldo), static_cast<unsigned long long>(width));
  }
  if (d->oq != nullptr) {
    if (d->oquant > HRB_QUANT_VEC) return refuse(ctx, HRB_EINVAL, "unknown output quantizer %u", d->oquant);
    if (!on(d->oq, 16) || (d->ldoq != 0u && (d->ldoq % 32u != 0u || d->ldoq < width))) {
      return refuse(ctx, HRB_EINVAL, "MXINT8 output rows of %llu codes: 16-byte aligned, a multiple "
                    "of 32, at least %llu", static_cast<unsigned long long>(d->ldoq),
                    static_cast<unsigned long long>(width));
    }
  }
  if (d->workspace != nullptr && !on(d->workspace, 256)) {
    return refuse(ctx, HRB_EINVAL, "workspace is not 256-byte aligned");
  }
  return HRB_OK;
}

hrb::AttnJob attn_job(const hrb_ctx* ctx, const hrb_attn_desc* d) {
  hrb::AttnJob j{};
  j.device = static_cast<uint32_t>(hrb::ctx_device(ctx));
  j.cache = hrb::make_kv_cache(d->cache);
  j.q = static_cast<const uint16_t*>(d->q);
  j.ldq = d->ldq;
  j.q_start = d->q_start;
  j.kv_len = d->kv_len;
  j.table = d->table;
  j.prefix = d->prefix;
  j.slopes = d->slopes;
  j.out = static_cast<uint16_t*>(d->out);
  j.ldo = d->ldo;
  j.oq = d->oq;
  j.oscale = d->oscale;
  j.ldoq = d->ldoq != 0u ? d->ldoq : uint64_t{d->heads} * d->cache.hd;
  j.vec_rule = d->oquant == HRB_QUANT_VEC;
  j.seqs = d->seqs;
  j.heads = d->heads;
  j.group = d->heads / d->cache.kv_heads;
  j.total_q = d->total_q;
  j.max_q = d->max_q;
  j.max_kv = d->max_kv;
  j.table_ld = d->table_ld;
  j.causal = d->causal != 0u;
  j.window = d->window;
  j.scale = d->scale;
  j.softcap = d->softcap;
  if (d->softcap != 0.f) {
    // Finite for every cap: a score of zero times these is no NaN.  A cap
    // above 2.3e38 is taken as that.
    const double cap = std::min<double>(d->softcap, 2.3e38), most = 3.4e38;
    j.cap_inv = static_cast<float>(std::min(1.0 / cap, most));
    j.cap_in = static_cast<float>(std::min(2.885390081777927 / cap, most));
    j.cap_out = static_cast<float>(cap * 1.4426950408889634);
  }
  return j;
}

uint64_t up256(uint64_t x) { return (x + 255u) / 256u * 256u; }

// Whether a call takes the decoding kernel, in blocks of 32 rows, or the
// prompt kernel.  Measured, 32/8 heads of 128 unless said (decoding, prompt):
//   12 rows, one request of 100, 64 of 100 and 500   7 and 9, 16 and 25, 25 and 66 us
//   28 rows, the same                                12 and 9, 27 and 25, 41 and 67 us
//   27 rows, the same, 15/5 heads of 64              9 and 7, 19 and 16, 27 and 34 us
//   64 rows, one request of 200, 2000, 30000 keys    15 and 12, 20 and 20, 49 and 60 us
//   64 rows, 64 of 500; 16 of 2000; 64 of 4000       82 and 72, 50 and 93, 340 and 439 us
//   96 rows, the same three                          121 and 87, 96 and 92, 505 and 441 us
//   96 rows, the same three, 15/5 heads of 64        55 and 35, 33 and 52, 214 and 224 us
//   126 rows, the same three, 15/5 heads of 64       69 and 35, 61 and 49, 267 and 226 us
bool decoding(const hrb::AttnJob& j) {
  const uint32_t rows = j.max_q * j.group;
  return rows <= 16u || (rows <= 32u && j.max_kv > 128u) ||
         (rows <= (j.cache.hd <= 64u ? 96u : 64u) && j.max_kv > 1024u);
}

// More tiles or partial rows than any GPU's memory holds (2^26 tiles of 24 KB
// at least, 2^36 rows of 136 bytes at least): their bytes fit 64 bits.
constexpr uint64_t kMostTiles = uint64_t{1} << 26, kMostCells = uint64_t{1} << 36;

// Fills in how the call is split and where its scratch lies from `base`
// (null: to learn the size).  False where the scratch passes all memory, else
// its bytes in `bytes`.
bool attn_plan(const hrb_ctx* ctx, const hrb_attn_desc* d, hrb::AttnJob* j, uint8_t* base,
               uint64_t* bytes) {
  // Requests with more than max_kv keys are left out.
  const uint64_t most_kv = uint64_t{d->seqs} * d->max_kv;
  const uint64_t total_kv = d->total_kv != 0u && d->total_kv < most_kv ? d->total_kv : most_kv;
  uint64_t at = 0;
  if (decoding(*j)) {
    j->chunk = hrb::attn_decode_chunk(*j, total_kv, hrb::ctx_sm_count(ctx));
  } else {
    const uint64_t tiles = hrb::attn_prompt_tiles(*j, total_kv, &j->tile_stride);
    if (tiles > kMostTiles) return false;
    j->tiles_cap = static_cast<uint32_t>(tiles);
    j->tiles = base;
    at = up256(tiles * j->cache.kv_heads * hrb::attn_prompt_tile_bytes(*j));
    j->chunk = hrb::attn_prompt_chunk(*j, hrb::ctx_sm_count(ctx));
  }
  if (j->max_kv > j->chunk) {
    const uint64_t cells = (uint64_t{j->max_kv} + j->chunk - 1u) / j->chunk * j->total_q * j->heads;
    if (cells > kMostCells) return false;
    j->part_ml = reinterpret_cast<float2*>(base + at);
    at += up256(cells * 8u);
    j->part_o = reinterpret_cast<float*>(base + at);
    at += cells * j->cache.hd * 4u;
  }
  *bytes = at;
  return true;
}

hrb_status too_large(hrb_ctx* ctx, const hrb_attn_desc* d) {
  return refuse(ctx, HRB_ENOMEM, "hrb_attention: no scratch for %u requests of up to %u keys, %llu together",
                d->seqs, d->max_kv, static_cast<unsigned long long>(d->total_kv));
}

}  // namespace

extern "C" {

uint64_t hrb_kv_record_bytes(uint32_t page, uint32_t hd) {
  return uint64_t{page} * (uint64_t{hd} + hd / 16u);
}

hrb_status hrb_block_tables(hrb_ctx* ctx, const hrb_blocks_desc* d, void* stream) {
  if (ctx == nullptr) return HRB_EINVAL;
  if (d == nullptr) return refuse(ctx, HRB_EINVAL, "null block table descriptor");
  if (!page_size(d->page)) {
    return refuse(ctx, HRB_EINVAL, "pages of %u tokens (16, 32, 64, 128 or 256)", d->page);
  }
  if (d->seqs > 65536u) return refuse(ctx, HRB_EINVAL, "%u requests (at most 65536)", d->seqs);
  if (d->max_tokens > 0x7FFFFFFFu || d->nfree > 0x7FFFFFFFu) {
    return refuse(ctx, HRB_EINVAL, "%u tokens, %u free pages", d->max_tokens, d->nfree);
  }
  if (d->q_start == nullptr ||
      (d->seqs != 0u && (d->cached == nullptr || d->fresh == nullptr || d->kv_len == nullptr ||
                         (d->table == nullptr && d->table_ld != 0u))) ||
      (d->max_tokens != 0u && d->slots == nullptr) || (d->nfree != 0u && d->free_pages == nullptr)) {
    return refuse(ctx, HRB_EINVAL, "null buffer");
  }
  if (!on(d->cached, 4) || !on(d->fresh, 4) || !on(d->free_pages, 4) || !on(d->head_in, 4) ||
      !on(d->head_out, 4) || !on(d->table, 4) || !on(d->q_start, 4) || !on(d->kv_len, 4) ||
      !on(d->slots, 4) || !on(d->pos, 4)) {
    return refuse(ctx, HRB_EINVAL, "a list is not 4-byte aligned");
  }
  const int32_t* const in[] = {d->cached, d->fresh, d->free_pages, d->head_in};
  const int32_t* const out[] = {d->table, d->q_start, d->kv_len, d->slots, d->pos, d->head_out};
  for (const int32_t* a : in) {
    for (const int32_t* b : out) {
      if (a != nullptr && a == b) {
        return refuse(ctx, HRB_EINVAL, "an output list is an input: blocks still read the one while "
                                       "the other is written");
      }
    }
  }
  if (cudaSetDevice(hrb::ctx_device(ctx)) != cudaSuccess) {
    return refuse(ctx, HRB_ECUDA, "cudaSetDevice");
  }
  hrb::BlocksJob j{};
  j.cached = d->cached;
  j.fresh = d->fresh;
  j.free_pages = d->free_pages;
  j.head_in = d->head_in;
  j.head_out = d->head_out;
  j.table = d->table;
  j.q_start = d->q_start;
  j.kv_len = d->kv_len;
  j.slots = d->slots;
  j.pos = d->pos;
  j.seqs = d->seqs;
  while ((1u << j.page_log2) < d->page) ++j.page_log2;
  j.nfree = d->nfree;
  j.table_ld = d->table_ld;
  j.max_tokens = d->max_tokens;
  hrb::launch_block_tables(j, hrb::ctx_error_word(ctx), hrb::ctx_stream(ctx, stream));
  return launched(ctx, 1, "hrb_block_tables");
}

hrb_status hrb_qkv_append(hrb_ctx* ctx, const hrb_qkv_desc* d, void* stream) {
  if (ctx == nullptr) return HRB_EINVAL;
  if (d == nullptr) return refuse(ctx, HRB_EINVAL, "null QKV descriptor");
  const hrb_status st = check_cache(ctx, &d->cache);
  if (st != HRB_OK) return st;
  if (d->dtype > HRB_DT_BF16) return refuse(ctx, HRB_EINVAL, "QKV rows of type %u (FP32 or BF16)", d->dtype);
  if (d->heads == 0u || d->heads > 65535u || d->tokens > 0x7FFFFFFFu) {
    return refuse(ctx, HRB_EINVAL, "%u tokens of %u query heads", d->tokens, d->heads);
  }
  if (!(d->eps >= 0.f)) return refuse(ctx, HRB_EINVAL, "eps %g", static_cast<double>(d->eps));
  if (d->rope != nullptr) {
    if (d->rot == 0u || d->rot % 8u != 0u || d->rot > d->cache.hd) {
      return refuse(ctx, HRB_EINVAL, "rotation of %u of %u dims (a multiple of 8)", d->rot, d->cache.hd);
    }
    if (d->axes == 0u || d->axes > 3u) return refuse(ctx, HRB_EINVAL, "%u position axes (1 to 3)", d->axes);
    uint64_t sum = 0;
    for (uint32_t a = 0; a < d->axes; ++a) sum += d->sections[a];
    if (d->axes > 1u && sum != d->rot / 2u) {
      return refuse(ctx, HRB_EINVAL, "axis sections of %llu pairs, the rotation has %u",
                    static_cast<unsigned long long>(sum), d->rot / 2u);
    }
    if (!on(d->rope, 8)) return refuse(ctx, HRB_EINVAL, "rotation table is not 8-byte aligned");
  }
  if (d->tokens == 0u) return HRB_OK;
  if (d->q == nullptr || d->k == nullptr || d->v == nullptr || d->slots == nullptr ||
      d->q_out == nullptr || (d->rope != nullptr && d->pos == nullptr)) {
    return refuse(ctx, HRB_EINVAL, "null buffer");
  }
  const uint64_t qw = uint64_t{d->heads} * d->cache.hd;
  const uint64_t kw = uint64_t{d->cache.kv_heads} * d->cache.hd;
  if (d->ldq < qw || d->ldk < kw || d->ldv < kw) return refuse(ctx, HRB_EINVAL, "QKV rows overlap");
  const uintptr_t size = d->dtype == HRB_DT_F32 ? 4u : 2u;
  if (!on(d->q, size) || !on(d->k, size) || !on(d->v, size) || !on(d->q_norm, 4) ||
      !on(d->k_norm, 4) || !on(d->pos, 4) || !on(d->slots, 4)) {
    return refuse(ctx, HRB_EINVAL, "a buffer is not aligned to its elements");
  }
  if (!on(d->q_out, 8) || d->ldqo % 4u != 0u || d->ldqo < qw) {
    return refuse(ctx, HRB_EINVAL, "query output rows of %llu elements: 8-byte aligned, at least %llu",
                  static_cast<unsigned long long>(d->ldqo), static_cast<unsigned long long>(qw));
  }
  if (cudaSetDevice(hrb::ctx_device(ctx)) != cudaSuccess) {
    return refuse(ctx, HRB_ECUDA, "cudaSetDevice");
  }
  hrb::QkvJob j{};
  j.cache = hrb::make_kv_cache(d->cache);
  const void* x[3] = {d->q, d->k, d->v};
  const uint64_t ld[3] = {d->ldq, d->ldk, d->ldv};
  bool vec = true;
  for (int i = 0; i < 3; ++i) {
    j.x[i] = x[i];
    j.ld[i] = ld[i];
    vec = vec && on(x[i], 4u * size) && ld[i] % 4u == 0u;
  }
  j.norm[0] = d->q_norm;
  j.norm[1] = d->k_norm;
  j.rope = reinterpret_cast<const float2*>(d->rope);
  j.pos = d->pos;
  j.slots = d->slots;
  j.q_out = d->q_out;
  j.ldqo = d->ldqo;
  j.eps = d->eps;
  j.tokens = d->tokens;
  j.heads = d->heads;
  j.max_pos = d->max_pos;
  j.half = d->rope != nullptr ? d->rot / 2u : 0u;
  j.interleaved = d->interleaved != 0u;
  j.cut[0] = d->axes > 1u ? d->sections[0] : j.half;
  j.cut[1] = d->axes > 2u ? d->sections[0] + d->sections[1] : j.half;
  hrb::launch_qkv_append(j, d->dtype == HRB_DT_BF16, vec, hrb::ctx_error_word(ctx),
                         hrb::ctx_sm_count(ctx), hrb::ctx_stream(ctx, stream));
  return launched(ctx, 1, "hrb_qkv_append");
}

hrb_status hrb_kv_read(hrb_ctx* ctx, const hrb_kv_cache* cache, const int32_t* slots,
                       uint32_t tokens, uint32_t dtype, void* k, void* v, void* stream) {
  if (ctx == nullptr) return HRB_EINVAL;
  if (cache == nullptr) return refuse(ctx, HRB_EINVAL, "null cache");
  const hrb_status st = check_cache(ctx, cache);
  if (st != HRB_OK) return st;
  if (dtype > HRB_DT_E5M2) return refuse(ctx, HRB_EINVAL, "unknown type %u", dtype);
  if (tokens > 0x7FFFFFFFu) return refuse(ctx, HRB_EINVAL, "%u tokens", tokens);
  if (tokens == 0u || (k == nullptr && v == nullptr)) return HRB_OK;
  if (slots == nullptr || !on(slots, 4)) return refuse(ctx, HRB_EINVAL, "slots missing or misaligned");
  if (!on(k, 16) || !on(v, 16)) return refuse(ctx, HRB_EINVAL, "outputs are not 16-byte aligned");
  if (cudaSetDevice(hrb::ctx_device(ctx)) != cudaSuccess) {
    return refuse(ctx, HRB_ECUDA, "cudaSetDevice");
  }
  hrb::launch_kv_read(hrb::make_kv_cache(*cache), slots, tokens, dtype, k, v,
                      hrb::ctx_error_word(ctx), hrb::ctx_stream(ctx, stream));
  return launched(ctx, 1, "hrb_kv_read");
}

hrb_status hrb_attention_workspace(hrb_ctx* ctx, const hrb_attn_desc* d, uint64_t* bytes) {
  if (ctx == nullptr || bytes == nullptr) return HRB_EINVAL;
  *bytes = 0;
  const hrb_status st = check_attn(ctx, d);
  if (st != HRB_OK || d->total_q == 0u) return st;
  hrb::AttnJob j = attn_job(ctx, d);
  return attn_plan(ctx, d, &j, nullptr, bytes) ? HRB_OK : too_large(ctx, d);
}

hrb_status hrb_attention(hrb_ctx* ctx, const hrb_attn_desc* d, void* stream) {
  if (ctx == nullptr) return HRB_EINVAL;
  hrb_status st = check_attn(ctx, d);
  if (st != HRB_OK) return st;
  if (d->total_q == 0u) return HRB_OK;
  if (cudaSetDevice(hrb::ctx_device(ctx)) != cudaSuccess) {
    return refuse(ctx, HRB_ECUDA, "cudaSetDevice");
  }
  cudaStream_t s = hrb::ctx_stream(ctx, stream);
  hrb::AttnJob j = attn_job(ctx, d);
  uint64_t need = 0;
  if (!attn_plan(ctx, d, &j, nullptr, &need)) return too_large(ctx, d);
  if (need != 0u) {
    void* base = d->workspace;
    if (base == nullptr) {
      st = hrb::ctx_serve_scratch(ctx, need, s, &base);
      if (st != HRB_OK) return st;
    } else if (d->workspace_bytes < need) {
      return refuse(ctx, HRB_EINVAL, "workspace of %llu bytes, %llu needed",
                    static_cast<unsigned long long>(d->workspace_bytes),
                    static_cast<unsigned long long>(need));
    }
    attn_plan(ctx, d, &j, static_cast<uint8_t*>(base), &need);
  }
  const int n = decoding(j)
                    ? hrb::launch_attn_decode(j, hrb::ctx_error_word(ctx), s)
                    : hrb::launch_attn_prompt(j, hrb::ctx_error_word(ctx), s);
  if (n < 0) return refuse(ctx, HRB_ECUDA, "hrb_attention: %s", cudaGetErrorString(cudaGetLastError()));
  return launched(ctx, static_cast<uint32_t>(n), "hrb_attention");
}

}  // extern "C"
