// Rotary positions: pairs of a row are turned by the angle of the row's position.
//
//   (a, b) -> m * (a cos t - b sin t,  a sin t + b cos t),   t = position * frequency
//
// Pair i of n is (x[i], x[i + n]), or (x[2i], x[2i + 1]) where neighbours are pairs;
// what a row has behind its 2n first numbers stays.  The gradient is the same with
// -t.
//
// The angle is found in turns in 64 bits (a position of a million leaves fp32 with
// an error of 0.03 in the angle) and its whole turns are dropped before anything is
// rounded to 32.
#include "paged_common.h"

namespace as {

namespace {

struct RotaryRows {
  const void* from;  // [tokens, heads, width]
  void* to;          // the same, contiguous
  int64_t stride[2];
  int heads;
};

struct RotaryArgs {
  RotaryRows rows[2];  // queries and keys
  const int64_t* positions;
  const double* frequencies;  // [pairs]
  int64_t tokens;
  int width;
  int pairs;
  int interleaved;
  float magnitude;
  float sign;
};

constexpr double kPerTurn = 0.15915494309189535;  // 1 / (2 pi)

template <typename T>
__global__ __launch_bounds__(kBlock) void rotary_kernel(RotaryArgs a) {
  const int64_t token = blockIdx.x;
  const double position = static_cast<double>(a.positions[token]);
  const int items = a.width - a.pairs;  // the pairs of a row, then what stays
  const int heads = a.rows[0].heads + a.rows[1].heads;
  for (int i = threadIdx.x; i < items * heads; i += kBlock) {
    const int head = i / items;
    const int pair = i - head * items;
    const bool second = head >= a.rows[0].heads;
    const RotaryRows& r = a.rows[second ? 1 : 0];
    const int h = second ? head - a.rows[0].heads : head;
    const T* x = static_cast<const T*>(r.from) + token * r.stride[0] + h * r.stride[1];
    T* y = static_cast<T*>(r.to) + (token * r.heads + h) * a.width;
    if (pair >= a.pairs) {
      y[pair + a.pairs] = x[pair + a.pairs];
      continue;
    }
    const double turns = position * (a.frequencies[pair] * kPerTurn);
    double sine;
    double cosine;
    sincospi(2.0 * (turns - __builtin_rint(turns)), &sine, &cosine);
    const float s = static_cast<float>(sine) * a.magnitude * a.sign;
    const float c = static_cast<float>(cosine) * a.magnitude;
    const int at = a.interleaved ? 2 * pair : pair;
    const int other = a.interleaved ? at + 1 : at + a.pairs;
    const float u = Elem<T>::at(x, at);
    const float v = Elem<T>::at(x, other);
    y[at] = rounded<T>(u * c - v * s);
    y[other] = rounded<T>(u * s + v * c);
  }
}

}  // namespace

}  // namespace as

using namespace as;

extern "C" {

int as_rotary_positions(const void* query, const int64_t* query_strides, void* query_out, int64_t heads,
                        const void* key, const int64_t* key_strides, void* key_out, int64_t key_heads,
                        const int64_t* positions, const double* frequencies, int64_t tokens, int64_t width,
                        int64_t pairs, int interleaved, int inverse, float magnitude, int dtype, void* stream) {
  clear_error();
  if (dtype != AS_DTYPE_F32 && dtype != AS_DTYPE_BF16 && dtype != AS_DTYPE_F16)
    return fail(AS_ERR_INVALID_ARGUMENT, "dtype must be AS_DTYPE_F32, AS_DTYPE_BF16 or AS_DTYPE_F16");
  if (tokens < 0 || tokens > kMaxBlocksPerLaunch) return fail(AS_ERR_UNSUPPORTED, "at most 2^22 tokens");
  if (heads < 0 || heads > 65535 || key_heads < 0 || key_heads > 65535)
    return fail(AS_ERR_INVALID_ARGUMENT, "heads must lie in [0, 65535]");
  if (width < 1 || width > 1024) return fail(AS_ERR_UNSUPPORTED, "width must lie in [1, 1024]");
  if (pairs < 0 || 2 * pairs > width) return fail(AS_ERR_INVALID_ARGUMENT, "the pairs must fit the width");
  if (tokens == 0 || heads + key_heads == 0) return AS_OK;
  const bool missing = (heads > 0 && (query == nullptr || query_strides == nullptr || query_out == nullptr)) ||
                       (key_heads > 0 && (key == nullptr || key_strides == nullptr || key_out == nullptr));
  if (missing || positions == nullptr || (pairs > 0 && frequencies == nullptr))
    return fail(AS_ERR_INVALID_ARGUMENT, "null pointer argument");
  const size_t size = dtype == AS_DTYPE_F32 ? 4 : 2;
  if (!aligned(query, size) || !aligned(query_out, size) || !aligned(key, size) || !aligned(key_out, size))
    return fail(AS_ERR_INVALID_ARGUMENT, "rows must be aligned to their elements");
  RotaryArgs a{};
  a.rows[0] = RotaryRows{query, query_out, {}, static_cast<int>(heads)};
  a.rows[1] = RotaryRows{key, key_out, {}, static_cast<int>(key_heads)};
  for (int i = 0; i < 2; ++i) {
    a.rows[0].stride[i] = heads > 0 ? query_strides[i] : 0;
    a.rows[1].stride[i] = key_heads > 0 ? key_strides[i] : 0;
  }
  a.positions = positions;
  a.frequencies = frequencies;
  a.tokens = tokens;
  a.width = static_cast<int>(width);
  a.pairs = static_cast<int>(pairs);
  a.interleaved = interleaved != 0;
  a.magnitude = magnitude;
  a.sign = inverse ? -1.0f : 1.0f;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_float_element(dtype, [&](auto e) {
    rotary_kernel<decltype(e)><<<dim3(static_cast<unsigned>(tokens)), kBlock, 0, s>>>(a);
    return check_launch("rotary_positions");
  });
}

}  // extern "C"
