// The paged key-value cache on the device: which page holds a token, and the 8-bit
// and 4-bit numbers of a cache that is quantised as it is written.
#pragma once

#include "as_device.h"
#include "as_internal.h"
#include "elem16.h"

namespace as {

// 8-bit elements: sign, 4 bits of exponent, 3 of fraction, no infinities.
struct E4m3 {
  uint8_t bits;
};
// Two 4-bit elements, the first in the low bits: sign, 2 bits of exponent, 1 of fraction.
struct E2m1Pair {
  uint8_t bits;
};

// One of the two page tensors [pages, heads, page_size, width], rows unit-stride.
struct PageTensor {
  void* data;
  int8_t* exponents;  // e4m3: [pages, heads, page_size]; e2m1: [pages, heads, page_size, ceil(width / 32)], else null
  int64_t stride[3];
  int64_t exponent_stride[3];
  int width;
};

struct PagedCache {
  PageTensor key;
  PageTensor value;
  const int64_t* page_ptr;
  const int64_t* page_idx;
  int64_t page_idx_len;
  int64_t pages;
  int sequences;
  int page_size;
  int heads;
};

namespace {

// The page list of sequence b, inside page_idx whatever page_ptr holds.
struct PageList {
  int64_t begin;
  int64_t count;
};
__device__ __forceinline__ PageList page_list(const PagedCache& c, int b) {
  int64_t begin = c.page_ptr[b];
  int64_t end = c.page_ptr[b + 1];
  begin = begin < 0 ? 0 : (begin > c.page_idx_len ? c.page_idx_len : begin);
  end = end < begin ? begin : (end > c.page_idx_len ? c.page_idx_len : end);
  return PageList{begin, end - begin};
}

// ---- 8-bit numbers ------------------------------------------------------------
// A row x[0 .. width) of one token and head is held as codes and one exponent e:
// 2^e is the smallest power of two (not below 2^-126) with max|x| <= 448 * 2^e,
// 448 being the largest e4m3 number, and x * 2^-e is rounded to e4m3, half to
// even.  A power of two makes the scaling exact: the rounding is that of the
// codes alone (at most 2^-4 of the value), the same in every precision, and the
// held values are numbers of bf16 and of fp32.  Infinities and NaN are held as
// NaN and do not count for the maximum.

// e of a finite maximum, from its bits: 448 = 1.75 * 2^8.
__device__ __forceinline__ int row_exponent(float largest) {
  const uint32_t u = __float_as_uint(largest);
  int e = static_cast<int>(u >> 23) - 127 - 8;
  if ((u & 0x7fffffu) > 0x600000u) ++e;
  return e < -126 ? -126 : e;
}
// 2^e for e in [-126, 127].
__device__ __forceinline__ float power_of_two(int e) {
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// The codes of two scaled numbers in the low 16 bits (magnitudes of at most 448).
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
  const uint32_t pair = __builtin_amdgcn_cvt_pk_fp8_f32(finite(a) ? a : 0.0f, finite(b) ? b : 0.0f, 0, false);
  return (pair & 0xffffu) | (finite(a) ? 0u : 0x7fu) | (finite(b) ? 0u : 0x7f00u);
}
__device__ __forceinline__ float e4m3_value(uint8_t code) { return __builtin_amdgcn_cvt_f32_fp8(code, 0); }

// ---- 4-bit numbers ------------------------------------------------------------
// Every 32 neighbouring numbers of a row (fewer at its end) are held as codes and a
// byte e + 127: 2^e is the smallest power of two (not below 2^-127) with
// max|x| <= 6 * 2^e, 6 being the largest e2m1 number, and x * 2^-e is rounded to
// 0, 1/2, 1, 3/2, 2, 3, 4, 6, half to the even code.  The byte 255 makes all of its
// numbers NaN: that is how a group is held that has a number which is not finite.
constexpr int kGroup = 32;
constexpr int kNanExponent = 255;

// The byte of a finite maximum, from its bits: 6 = 1.5 * 2^2.
__device__ __forceinline__ int group_exponent(float largest) {
  const uint32_t u = __float_as_uint(largest);
  int e = static_cast<int>(u >> 23) - 2;
  if ((u & 0x7fffffu) > 0x400000u) ++e;
  return e < 0 ? 0 : e;
}
template <typename T>
__device__ __forceinline__ T rounded(float v);
template <>
__device__ __forceinline__ float rounded<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ Bf16 rounded<Bf16>(float v) {
  return __builtin_bit_cast(Bf16, static_cast<__bf16>(v));  // half to even, in hardware
}
template <>
__device__ __forceinline__ Fp16 rounded<Fp16>(float v) {
  return __builtin_bit_cast(Fp16, static_cast<_Float16>(v));
}

// Checks the host's description of a cache and lays it out for the kernels.
constexpr int64_t kMaxWidth = 256;

// Whether a cache of this type is quantised as it is written.
inline bool is_coded(int dtype) { return dtype == AS_DTYPE_E4M3 || dtype == AS_DTYPE_E2M1; }

inline int read_paged_cache(const as_paged_cache* c, PagedCache* out) {
  if (c == nullptr) return fail(AS_ERR_INVALID_ARGUMENT, "null cache pointer");
  if ((c->dtype < AS_DTYPE_F32 || c->dtype > AS_DTYPE_E4M3) && c->dtype != AS_DTYPE_E2M1)
    return fail(AS_ERR_INVALID_ARGUMENT, "the cache's dtype must be AS_DTYPE_F32, _BF16, _F16, _E4M3 or _E2M1");
  if (c->sequences < 0 || c->sequences > INT32_MAX || c->page_idx_len < 0)
    return fail(AS_ERR_INVALID_ARGUMENT, "sequences and page lists must have non-negative 32-bit sizes");
  if (c->pages < 1 || c->pages > INT32_MAX || c->page_size < 1 || c->page_size > (1 << 20))
    return fail(AS_ERR_INVALID_ARGUMENT, "a cache has 1 to 2^31 - 1 pages of 1 to 2^20 tokens");
  if (c->heads < 1 || c->heads > 65535) return fail(AS_ERR_INVALID_ARGUMENT, "heads must lie in [1, 65535]");
  if (c->key_width < 1 || c->key_width > kMaxWidth || c->value_width < 1 || c->value_width > kMaxWidth)
    return fail(AS_ERR_UNSUPPORTED, "key and value widths must lie in [1, %d]", static_cast<int>(kMaxWidth));
  if (c->key_pages == nullptr || c->value_pages == nullptr || c->page_ptr == nullptr ||
      (c->page_idx_len > 0 && c->page_idx == nullptr))
    return fail(AS_ERR_INVALID_ARGUMENT, "null pointer argument");
  const bool coded = is_coded(c->dtype);
  if (coded != (c->key_exponents != nullptr) || coded != (c->value_exponents != nullptr))
    return fail(AS_ERR_INVALID_ARGUMENT, "an e4m3 cache has exponents, and so has an e2m1 cache, any other has none");
  if (c->dtype == AS_DTYPE_E2M1 && (c->key_width % 2 != 0 || c->value_width % 2 != 0))
    return fail(AS_ERR_UNSUPPORTED, "an e2m1 cache holds rows of an even width");
  const size_t size = c->dtype == AS_DTYPE_F32 ? 4 : (coded ? 1 : 2);
  if (!aligned(c->key_pages, size) || !aligned(c->value_pages, size))
    return fail(AS_ERR_INVALID_ARGUMENT, "the pages must be aligned to their elements");
  out->key = PageTensor{c->key_pages, c->key_exponents, {}, {}, static_cast<int>(c->key_width)};
  out->value = PageTensor{c->value_pages, c->value_exponents, {}, {}, static_cast<int>(c->value_width)};
  for (int i = 0; i < 3; ++i) {
    out->key.stride[i] = c->key_strides[i];
    out->value.stride[i] = c->value_strides[i];
    out->key.exponent_stride[i] = c->key_exponent_strides[i];
    out->value.exponent_stride[i] = c->value_exponent_strides[i];
  }
  out->page_ptr = c->page_ptr;
  out->page_idx = c->page_idx;
  out->page_idx_len = c->page_idx_len;
  out->pages = c->pages;
  out->sequences = static_cast<int>(c->sequences);
  out->page_size = static_cast<int>(c->page_size);
  out->heads = static_cast<int>(c->heads);
  return AS_OK;
}

// Calls f with an element of the type of an AS_DTYPE_* code.
template <typename F>
int with_float_element(int dtype, F&& f) {
  if (dtype == AS_DTYPE_BF16) return f(Bf16{});
  if (dtype == AS_DTYPE_F16) return f(Fp16{});
  return f(float{});
}

}  // namespace
}  // namespace as
