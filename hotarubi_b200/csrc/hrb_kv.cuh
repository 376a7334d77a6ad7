// The 4-bit key/value cache of the serving calls on the device: where a
// token's codes and scales lie (hrb_kv_cache in hrb_gemm.h) and the MXFP4
// encoding of 32 values.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "hrb_gemm.h"

namespace hrb {

// Error-flag bits of the serving kernels (hrb_sync reports them).
constexpr uint32_t kErrKvSlot = 32u;       // a slot, position or table entry outside its range
constexpr uint32_t kErrKvNonFinite = 64u;  // Inf or NaN among the keys or values to encode
constexpr uint32_t kErrKvPages = 128u;     // tokens without a page, or past the step's end

// Exponents of the block scales: every E2M1 value (0.5 .. 6) times 2^e in
// this range is an FP16 number (6 * 2^13 = 49152, 0.5 * 2^-23 = 2^-24).
constexpr int32_t kKvExpMin = -23, kKvExpMax = 13;

// A cache with its strides in bytes.
struct KvCache {
  uint8_t* data;
  uint64_t page_stride;
  uint32_t pages, page, page_log2, kv_heads, hd;
  uint32_t record;  // bytes of one (page, head) record
};

inline KvCache make_kv_cache(const hrb_kv_cache& c) {
  KvCache k{};
  k.data = c.data;
  k.pages = c.pages;
  k.page = c.page;
  while ((1u << k.page_log2) < c.page) ++k.page_log2;
  k.kv_heads = c.kv_heads;
  k.hd = c.hd;
  k.record = c.page * (c.hd + c.hd / 16u);
  k.page_stride = c.page_stride != 0 ? c.page_stride : uint64_t{c.kv_heads} * k.record;
  return k;
}

__device__ __forceinline__ uint8_t* kv_record(const KvCache& c, uint32_t page, uint32_t head) {
  return c.data + static_cast<uint64_t>(page) * c.page_stride +
         static_cast<uint64_t>(head) * c.record;
}
// Offsets in a record: K codes at 0, then K scales, V codes; V scales are as far
// from the V codes as K scales from the K codes.
__device__ __forceinline__ uint32_t kv_kscales(const KvCache& c) { return c.page * (c.hd / 2u); }
__device__ __forceinline__ uint32_t kv_vcodes(const KvCache& c) { return c.record / 2u; }

// The exponent of a block whose largest magnitude has these FP32 bits.
__device__ __forceinline__ int32_t kv_block_exp(uint32_t top_bits) {
  const int32_t e = static_cast<int32_t>(top_bits >> 23) - 129;
  return min(max(e, kKvExpMin), kKvExpMax);
}

// Two values, already divided by the block's scale, to a byte of two E2M1
// codes (nearest, ties to even, saturating): `lo` in the low nibble.
__device__ __forceinline__ uint32_t e2m1_pair(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 b;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n\t"
      "cvt.u32.u8 %0, b;\n\t}"
      : "=r"(r)
      : "f"(hi), "f"(lo));
  return r;
}

// The four bytes of a word, two E2M1 codes each, as pairs of FP16 values, a
// byte's low nibble in the low half: one conversion a byte, no shifts (measured:
// 152 values a ns and SM, against 74 for shifts, masks and a multiplication that
// place the code's bits in an FP16).
__device__ __forceinline__ void e2m1x8_to_f16x2(uint32_t word, uint32_t (&r)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(word));
}

}  // namespace hrb
