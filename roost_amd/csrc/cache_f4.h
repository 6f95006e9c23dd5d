// The 4-bit KV cache as its calls share it: the admission of its record, the addresses inside a page and the conversions.
//
// Layout. Codes [pages, kv_heads, page_size, head_dim / 2]: a KV head's part of a page is one piece of memory, so that the
// attention's reads of 16 keys are 16 D / 2 consecutive bytes (512 to 2,048) whatever the number of heads. Scales [pages,
// kv_heads, head_dim / 32, page_size]: the scales that one lane needs for four neighbouring keys (the keys of a matrix
// operand, all of one block of dims) are one aligned word.
#ifndef ROOST_AMD_CACHE_F4_H_
#define ROOST_AMD_CACHE_F4_H_

#include "common.h"

namespace roost {

// Bytes that a span reaches over, for comparing spans: rows of `width` bytes every `stride` bytes (one row: stride 0).
struct Extent {
  uintptr_t first = 0;
  uint64_t rows = 0, stride = 0, width = 0;
  uintptr_t end() const { return first + (rows - 1) * stride + width; }
};

inline Extent ExtentOf(const void* p, uint64_t bytes) { return {reinterpret_cast<uintptr_t>(p), 1, 0, bytes}; }
inline Extent ExtentOf(const void* p, uint64_t rows, uint64_t stride, uint64_t width) {
  return {reinterpret_cast<uintptr_t>(p), rows, stride, width};
}

// Whether two extents share a byte. Column views of one tensor (equal strides) may interleave without sharing any.
inline bool Overlap(const Extent& a, const Extent& b) {
  if (a.first == 0 || b.first == 0 || a.rows == 0 || b.rows == 0 || a.width == 0 || b.width == 0) return false;
  if (!(a.first < b.end() && b.first < a.end())) return false;
  if (a.stride != b.stride || a.stride == 0) return true;
  const uint64_t off = b.first >= a.first ? (b.first - a.first) % a.stride  // b's column in a's rows
                                          : (a.stride - (a.first - b.first) % a.stride) % a.stride;
  return off < a.width || off + b.width > a.stride;
}

// The record's rules; `pages`: the pages that all four spans hold.
inline Gate& AdmitCacheF4(Gate& gate, const RoostAmdCacheF4& c, uint64_t& pages) {
  gate.Expect(c.reserved0 == 0, ROOST_STATUS_INVALID_ARGUMENT, "cache: reserved0 = %u, must be 0", c.reserved0)
      .Expect(c.kv_heads > 0 && c.kv_heads <= 1024, ROOST_STATUS_UNSUPPORTED, "cache: kv_heads = %u, not 1 to 1,024", c.kv_heads)
      .Expect(c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, ROOST_STATUS_UNSUPPORTED,
              "cache: head_dim = %u has no kernel here (built: 64, 128, 256)", c.head_dim)
      .Expect(IsPow2(c.page_size) && c.page_size >= 16 && c.page_size <= 1024, ROOST_STATUS_UNSUPPORTED,
              "cache: page_size = %u is no power of two from 16 to 1,024", c.page_size);
  if (!gate.ok()) return gate;
  const uint64_t values = uint64_t{c.kv_heads} * c.page_size * c.head_dim;  // of a page
  gate.Tensor("cache k", c.k, ROOST_DTYPE_F4E2M1, values)
      .Tensor("cache v", c.v, ROOST_DTYPE_F4E2M1, values)
      .Tensor("cache k_scales", c.k_scales, ROOST_DTYPE_U8, values / 32)
      .Tensor("cache v_scales", c.v_scales, ROOST_DTYPE_U8, values / 32)
      .Aligned("cache k", c.k.address, 16)
      .Aligned("cache v", c.v.address, 16)
      .Aligned("cache k_scales", c.k_scales.address, 16)
      .Aligned("cache v_scales", c.v_scales.address, 16);
  if (!gate.ok()) return gate;
  pages = std::min(std::min(c.k.length, c.v.length) / values, std::min(c.k_scales.length, c.v_scales.length) / (values / 32));
  return gate.Expect(pages <= 0x7FFFFFFF, ROOST_STATUS_UNSUPPORTED, "cache: %llu pages, more than an i32 page id names",
                     static_cast<unsigned long long>(pages));
}

// What the kernels take of the record.
struct CacheF4View {
  uint8_t *k, *k_scales, *v, *v_scales;
  uint32_t kv_heads, page_shift, pages;
};

inline CacheF4View ViewOf(const RoostAmdCacheF4& c, uint64_t pages) {
  return {static_cast<uint8_t*>(c.k.address),
          static_cast<uint8_t*>(c.k_scales.address),
          static_cast<uint8_t*>(c.v.address),
          static_cast<uint8_t*>(c.v_scales.address),
          c.kv_heads,
          static_cast<uint32_t>(__builtin_ctz(c.page_size)),
          static_cast<uint32_t>(pages)};
}

}  // namespace roost

namespace roost_dev {

constexpr uint32_t kF4ByteLow = 7, kF4ByteHigh = 252, kF4ByteNan = 255;

// The scale byte of a block whose largest magnitude has these f32 bits: the smallest power of two s with a <= 7 s, within
// 2^-120 .. 2^125; kF4ByteNan for an infinity or a NaN, which as integers are above every number. a = m 2^e with 1 <= m < 2
// needs s = 2^(e - 2) up to m = 1.75, else 2^(e - 1). 7, not 6: rounding 7 to 6 is off by one scale, as rounding 5 to 4 is.
__device__ __forceinline__ uint32_t F4ScaleByte(uint32_t magnitude) {
  if (magnitude >= 0x7F800000u) return kF4ByteNan;
  const int e = static_cast<int>(magnitude >> 23) + ((magnitude & 0x7FFFFFu) > 0x600000u ? 1 : 0) - 2;
  return static_cast<uint32_t>(min(max(e, static_cast<int>(kF4ByteLow)), static_cast<int>(kF4ByteHigh)));
}

// The byte as the f32 power of two that the conversions below take; byte 255 gives an exponent of all ones, which they read
// as NaN.
__device__ __forceinline__ float F4Scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight values to codes, value i in bits 4 i: v_cvt_scalef32_pk_fp4_f32 divides by the scale and rounds to nearest, ties to
// even, and leaves what is above 6 at 6.
__device__ __forceinline__ uint32_t ToF4(const float (&x)[8], float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
  return w;
}

// Codes 2 kPair and 2 kPair + 1 of a word as packed bf16, exactly: e2m1 times a power of two has two significant bits and,
// from 2^-121 to 6 2^125, a normal bf16's exponent.
template <int kPair>
__device__ __forceinline__ uint32_t FromF4(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, kPair));
}

}  // namespace roost_dev

#endif  // ROOST_AMD_CACHE_F4_H_
