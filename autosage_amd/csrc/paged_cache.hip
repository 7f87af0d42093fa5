// Keys and values of new tokens into the pages of their sequences, and back.
//
// Tokens stand one behind the other, those of sequence b at token_ptr[b] ..
// token_ptr[b + 1]; the first of them has position start[b] in its sequence.
// Tokens from token_ptr[sequences] on belong to no sequence: a write leaves the
// cache alone for them, a read gives zeros.  A copy (with a rounding to 8 bits
// in a quantised cache): bound by memory, or by the launch for a few tokens.
#include "paged_common.h"

namespace as {

namespace {

struct TokenRows {
  void* data;  // [tokens, heads, width]
  int64_t stride[2];
};

// The place of a token: page id (< 0: none) and the token's place in the page.
struct Place {
  int64_t page;
  int slot;
};
__device__ __forceinline__ Place place_of_token(const PagedCache& c, const int64_t* __restrict__ token_ptr,
                                                const int64_t* __restrict__ start, int64_t t) {
  const int64_t b = wave_row_of_edge(token_ptr, c.sequences, t);
  const int64_t at = t - token_ptr[b];
  if (at < 0 || t >= token_ptr[b + 1]) return Place{-1, 0};
  const int64_t position = start[b] + at;
  const PageList list = page_list(c, static_cast<int>(b));
  const int64_t k = position / c.page_size;
  if (position < 0 || k >= list.count) return Place{-1, 0};
  const int64_t page = c.page_idx[list.begin + k];
  if (page < 0 || page >= c.pages) return Place{-1, 0};
  return Place{page, static_cast<int>(position - k * c.page_size)};
}

// One wave per row of one token, head and tensor.
template <typename T, typename C>
__global__ __launch_bounds__(kBlock) void paged_write_kernel(PagedCache c, TokenRows key, TokenRows value,
                                                             const int64_t* __restrict__ token_ptr,
                                                             const int64_t* __restrict__ start, int64_t tokens) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + wave_in_block();
  if (row >= tokens * c.heads * 2) return;
  const bool is_value = row & 1;
  const int64_t t = (row >> 1) / c.heads;
  const int h = static_cast<int>((row >> 1) - t * c.heads);
  const Place place = place_of_token(c, token_ptr, start, t);
  if (place.page < 0) return;
  const TokenRows& from = is_value ? value : key;
  const PageTensor& to = is_value ? c.value : c.key;
  const T* x = static_cast<const T*>(from.data) + t * from.stride[0] + h * from.stride[1];
  C* y = static_cast<C*>(to.data) + place.page * to.stride[0] + h * to.stride[1] + place.slot * to.stride[2];
  if constexpr (__is_same(T, C)) {
    for (int i = lane_id(); i < to.width; i += kWave) y[i] = x[i];
  } else {
    float largest = 0.0f;
    for (int i = lane_id(); i < to.width; i += kWave) {
      const float v = Elem<T>::at(x, i);
      largest = fmaxf(largest, finite(v) ? fabsf(v) : 0.0f);
    }
    const int e = row_exponent(wave_max_f32(largest));
    const float scale = power_of_two(-e);
    for (int i = lane_id(); i < to.width; i += kWave) {
      y[i].bits = static_cast<uint8_t>(e4m3_pair(Elem<T>::at(x, i) * scale, 0.0f));
    }
    if (lane_id() == 0)
      to.exponents[place.page * to.exponent_stride[0] + h * to.exponent_stride[1] +
                   place.slot * to.exponent_stride[2]] = static_cast<int8_t>(e);
  }
}

template <typename C, typename T>
__global__ __launch_bounds__(kBlock) void paged_read_kernel(PagedCache c, TokenRows key, TokenRows value,
                                                            const int64_t* __restrict__ token_ptr,
                                                            const int64_t* __restrict__ start, int64_t tokens) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + wave_in_block();
  if (row >= tokens * c.heads * 2) return;
  const bool is_value = row & 1;
  const int64_t t = (row >> 1) / c.heads;
  const int h = static_cast<int>((row >> 1) - t * c.heads);
  const Place place = place_of_token(c, token_ptr, start, t);
  const PageTensor& from = is_value ? c.value : c.key;
  const TokenRows& to = is_value ? value : key;
  T* y = static_cast<T*>(to.data) + t * to.stride[0] + h * to.stride[1];
  if (place.page < 0) {
    for (int i = lane_id(); i < from.width; i += kWave) y[i] = T{};
    return;
  }
  const C* x = static_cast<const C*>(from.data) + place.page * from.stride[0] + h * from.stride[1] +
               place.slot * from.stride[2];
  if constexpr (__is_same(T, C)) {
    for (int i = lane_id(); i < from.width; i += kWave) y[i] = x[i];
  } else {
    const int e = from.exponents[place.page * from.exponent_stride[0] + h * from.exponent_stride[1] +
                                 place.slot * from.exponent_stride[2]];
    for (int i = lane_id(); i < from.width; i += kWave) y[i] = rounded<T>(ldexpf(Elem<C>::at(x, i), e));
  }
}

int check_tokens(const PagedCache& c, const void* key, const void* value, const int64_t* token_ptr,
                 const int64_t* start, int64_t tokens, int cache_dtype, int dtype) {
  if (dtype != AS_DTYPE_F32 && dtype != AS_DTYPE_BF16 && dtype != AS_DTYPE_F16)
    return fail(AS_ERR_INVALID_ARGUMENT, "dtype must be AS_DTYPE_F32, AS_DTYPE_BF16 or AS_DTYPE_F16");
  if (cache_dtype != AS_DTYPE_E4M3 && cache_dtype != dtype)
    return fail(AS_ERR_INVALID_ARGUMENT, "a cache that is not quantised holds the type of its tokens");
  if (tokens < 0 || tokens > (int64_t(1) << 40) / c.heads) return fail(AS_ERR_UNSUPPORTED, "too many tokens");
  if (tokens > 0 && c.sequences < 1) return fail(AS_ERR_INVALID_ARGUMENT, "tokens without sequences");
  if (tokens > 0 && (key == nullptr || value == nullptr || token_ptr == nullptr || start == nullptr))
    return fail(AS_ERR_INVALID_ARGUMENT, "null pointer argument");
  const size_t size = dtype == AS_DTYPE_F32 ? 4 : 2;
  if (!aligned(key, size) || !aligned(value, size))
    return fail(AS_ERR_INVALID_ARGUMENT, "key and value must be aligned to their elements");
  return AS_OK;
}

}  // namespace

}  // namespace as

using namespace as;

extern "C" {

int as_paged_cache_write(const as_paged_cache* cache, const void* key, const int64_t* key_strides, const void* value,
                         const int64_t* value_strides, const int64_t* token_ptr, const int64_t* start, int64_t tokens,
                         int dtype, void* stream) {
  clear_error();
  PagedCache c;
  if (const int bad = read_paged_cache(cache, &c)) return bad;
  if (const int bad = check_tokens(c, key, value, token_ptr, start, tokens, cache->dtype, dtype)) return bad;
  if (key_strides == nullptr || value_strides == nullptr) return fail(AS_ERR_INVALID_ARGUMENT, "null strides pointer");
  if (tokens == 0) return AS_OK;
  const TokenRows k{const_cast<void*>(key), {key_strides[0], key_strides[1]}};
  const TokenRows v{const_cast<void*>(value), {value_strides[0], value_strides[1]}};
  const dim3 grid(static_cast<unsigned>((tokens * c.heads * 2 + kWavesPerBlock - 1) / kWavesPerBlock));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_float_element(dtype, [&](auto e) {
    using T = decltype(e);
    if (cache->dtype == AS_DTYPE_E4M3) {
      paged_write_kernel<T, E4m3><<<grid, kBlock, 0, s>>>(c, k, v, token_ptr, start, tokens);
    } else {
      paged_write_kernel<T, T><<<grid, kBlock, 0, s>>>(c, k, v, token_ptr, start, tokens);
    }
    return check_launch("paged_cache_write");
  });
}

int as_paged_cache_read(const as_paged_cache* cache, void* key, void* value, const int64_t* token_ptr,
                        const int64_t* start, int64_t tokens, int dtype, void* stream) {
  clear_error();
  PagedCache c;
  if (const int bad = read_paged_cache(cache, &c)) return bad;
  if (const int bad = check_tokens(c, key, value, token_ptr, start, tokens, cache->dtype, dtype)) return bad;
  if (tokens == 0) return AS_OK;
  const TokenRows k{key, {int64_t(c.heads) * c.key.width, c.key.width}};
  const TokenRows v{value, {int64_t(c.heads) * c.value.width, c.value.width}};
  const dim3 grid(static_cast<unsigned>((tokens * c.heads * 2 + kWavesPerBlock - 1) / kWavesPerBlock));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_float_element(dtype, [&](auto e) {
    using T = decltype(e);
    if (cache->dtype == AS_DTYPE_E4M3) {
      paged_read_kernel<E4m3, T><<<grid, kBlock, 0, s>>>(c, k, v, token_ptr, start, tokens);
    } else {
      paged_read_kernel<T, T><<<grid, kBlock, 0, s>>>(c, k, v, token_ptr, start, tokens);
    }
    return check_launch("paged_cache_read");
  });
}

}  // extern "C"
