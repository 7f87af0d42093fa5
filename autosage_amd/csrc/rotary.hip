// Rotary positions: pairs of a row are turned by the angle of the row's position.
//
//   (a, b) -> m * (a cos t - b sin t,  a sin t + b cos t),   t = position * frequency
//
// Pair i of n is (x[i], x[i + n]), or (x[2i], x[2i + 1]) where neighbours are pairs;
// what a row has behind its 2n first numbers stays.  The gradient is the same with
// -t.
//
// The angle is found in turns in 64 bits (a position of a million leaves fp32 with
// an error of 0.03 in the angle) and reduced to an eighth of a turn before anything is
// rounded to 32.
//
// Every row is read and written once: bound by memory, so what counts is that the
// angles cost little and the accesses are wide.  A workgroup takes some tokens, finds
// the sines and cosines of their pairs, one for each thread, and keeps them in LDS for
// all heads of queries and keys; then its threads turn V pairs each, 16 bytes of
// either half, neighbours in a row and rows one behind the other.  The rows of its
// first step are asked for before the angles are found.
#include "paged_common.h"

namespace as {

namespace {

struct RotaryRows {
  const void* from;  // [tokens, heads, width]
  void* to;          // the same, contiguous
  int64_t stride[2];
  int heads;
};

// i / d = i * magic >> (31 + shift) for i < 2^31.
struct Divisor {
  int d;
  int shift;
  uint32_t magic;
};
inline Divisor divisor_of(int d) {
  Divisor v{d, 0, 0};
  while ((1 << v.shift) < d) ++v.shift;
  v.magic = static_cast<uint32_t>(((uint64_t(1) << (31 + v.shift)) + d - 1) / static_cast<uint64_t>(d));
  return v;
}
__device__ __forceinline__ int quotient(int i, const Divisor& v) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(i)) * v.magic) >> (31 + v.shift));
}

struct RotaryArgs {
  RotaryRows rows[2];  // queries and keys
  const int64_t* positions;
  const double* frequencies;  // [pairs]
  int64_t tokens;
  int width;
  int pairs;
  int turning;      // units of V pairs in a row, the last of which ends with the pairs
  Divisor units;    // those, and the units of 2V numbers that stay
  Divisor heads;    // of queries and keys
  Divisor by_pairs;
  int each;         // tokens of a workgroup
  float magnitude;
  float sign;
};

constexpr double kPerTurn = 0.15915494309189535;  // 1 / (2 pi)

// Sine and cosine of so many turns.
__device__ __forceinline__ void sine_of_turns(double turns, float* sine, float* cosine) {
  const double quarters = __builtin_rint(4.0 * turns);
  const float rest = static_cast<float>(turns - 0.25 * quarters);  // an eighth of a turn at most
  float s;
  float c;
  sincospif(2.0f * rest, &s, &c);
  const int q = static_cast<int>(static_cast<int64_t>(quarters)) & 3;
  *sine = q & 1 ? c : s;
  *cosine = q & 1 ? s : c;
  *sine = q & 2 ? -*sine : *sine;
  *cosine = (q + 1) & 2 ? -*cosine : *cosine;
}

template <typename T, int V>
__device__ __forceinline__ RawVec<V * sizeof(T)> load_numbers(const T* from) {
  RawVec<V * sizeof(T)> r;
  __builtin_memcpy(&r, from, V * sizeof(T));  // the alignment of an element: the hardware has no other requirement
  return r;
}

constexpr int kRotaryAhead = 2;  // units of a thread whose loads are under way at once

template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kBlock) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float angles[];  // [each * pairs] cosines, the same of sines
  const int64_t first = static_cast<int64_t>(blockIdx.x) * a.each;
  const int count = a.tokens - first < a.each ? static_cast<int>(a.tokens - first) : a.each;
  float* const cosines = angles;
  float* const sines = angles + a.each * a.pairs;
  const int items = count * a.heads.d * a.units.d;

  // a unit: V pairs from `pair` on, or numbers that stay (pair < 0), and where its two runs are read and written
  struct Unit {
    const T* from;
    T* to;
    int token;
    int pair;
    int one, two;
  };
  const auto unit_of = [&](int i) {
    Unit u;
    const int row = quotient(i, a.units);
    const int k = i - row * a.units.d;
    u.token = quotient(row, a.heads);
    int h = row - u.token * a.heads.d;
    const bool second = h >= a.rows[0].heads;
    h = second ? h - a.rows[0].heads : h;
    const int64_t t = first + u.token;
    const int64_t at = second ? t * a.rows[1].stride[0] + h * a.rows[1].stride[1]
                              : t * a.rows[0].stride[0] + h * a.rows[0].stride[1];
    u.from = static_cast<const T*>(second ? a.rows[1].from : a.rows[0].from) + at;
    u.to = static_cast<T*>(second ? a.rows[1].to : a.rows[0].to) +
           (t * (second ? a.rows[1].heads : a.rows[0].heads) + h) * a.width;
    // runs that would pass the end of the pairs, or of the row, end with it: what two units share is the same in both
    if (k < a.turning) {
      u.pair = k * V < a.pairs - V ? k * V : a.pairs - V;
      u.one = INTERLEAVED ? 2 * u.pair : u.pair;
      u.two = INTERLEAVED ? 2 * u.pair + V : u.pair + a.pairs;
    } else {
      const int d = 2 * a.pairs + (k - a.turning) * 2 * V;
      u.pair = -1;
      u.one = d < a.width - V ? d : a.width - V;
      u.two = d + V < a.width - V ? d + V : a.width - V;
    }
    return u;
  };

  for (int base = 0; base < items; base += kRotaryAhead * kBlock) {
    Unit unit[kRotaryAhead];
    RawVec<V * sizeof(T)> one[kRotaryAhead];
    RawVec<V * sizeof(T)> two[kRotaryAhead];
#pragma unroll
    for (int u = 0; u < kRotaryAhead; ++u) {
      const int i = base + u * kBlock + static_cast<int>(threadIdx.x);
      unit[u] = unit_of(i < items ? i : items - 1);
      one[u] = load_numbers<T, V>(unit[u].from + unit[u].one);
      two[u] = load_numbers<T, V>(unit[u].from + unit[u].two);
    }
    if (base == 0) {
      for (int i = threadIdx.x; i < count * a.pairs; i += kBlock) {
        const int t = quotient(i, a.by_pairs);
        const double turns =
            static_cast<double>(a.positions[first + t]) * (a.frequencies[i - t * a.pairs] * kPerTurn);
        float s;
        float c;
        sine_of_turns(turns, &s, &c);
        sines[i] = s * a.magnitude * a.sign;
        cosines[i] = c * a.magnitude;
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kRotaryAhead; ++u) {
      if (base + u * kBlock + static_cast<int>(threadIdx.x) >= items) break;
      if (unit[u].pair >= 0) {
        const int at = unit[u].token * a.pairs + unit[u].pair;
        float x[2 * V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[i] = Elem<T>::get(one[u].w, i);
          x[V + i] = Elem<T>::get(two[u].w, i);
        }
        T y[2 * V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float c = cosines[at + i];
          const float s = sines[at + i];
          const int p = INTERLEAVED ? 2 * i : i;
          const int q = INTERLEAVED ? 2 * i + 1 : V + i;
          y[p] = rounded<T>(x[p] * c - x[q] * s);
          y[q] = rounded<T>(x[p] * s + x[q] * c);
        }
        __builtin_memcpy(&one[u], y, V * sizeof(T));
        __builtin_memcpy(&two[u], y + V, V * sizeof(T));
      }
      __builtin_memcpy(unit[u].to + unit[u].one, &one[u], V * sizeof(T));
      __builtin_memcpy(unit[u].to + unit[u].two, &two[u], V * sizeof(T));
    }
  }
}

// The widest runs that neither the pairs nor what stays is shorter than.
int run_of(int pairs, int rest, int widest) {
  int v = widest;
  while (v > 1 && ((pairs > 0 && pairs < v) || (rest > 0 && rest < v))) v /= 2;
  return v;
}

template <typename T, int V>
void launch_rotary(const RotaryArgs& a, bool interleaved, dim3 grid, size_t lds, hipStream_t s) {
  if (interleaved) {
    rotary_kernel<T, V, true><<<grid, kBlock, lds, s>>>(a);
  } else {
    rotary_kernel<T, V, false><<<grid, kBlock, lds, s>>>(a);
  }
}

constexpr int64_t kMostAngles = 2048;  // of a workgroup: 16 KB of LDS

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
  if (tokens < 0 || tokens > (int64_t(1) << 26)) return fail(AS_ERR_UNSUPPORTED, "at most 2^26 tokens");
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
  a.magnitude = magnitude;
  a.sign = inverse ? -1.0f : 1.0f;
  const int rest = a.width - 2 * a.pairs;
  const int v = run_of(a.pairs, rest, dtype == AS_DTYPE_F32 ? 4 : 8);
  a.turning = (a.pairs + v - 1) / v;
  a.units = divisor_of(a.turning + (rest + 2 * v - 1) / (2 * v));
  a.heads = divisor_of(static_cast<int>(heads + key_heads));
  a.by_pairs = divisor_of(a.pairs > 0 ? a.pairs : 1);
  // Tokens of a workgroup: as many as give each of its threads four units, while 512 workgroups are left and the
  // angles have room
  const int64_t units = int64_t(a.units.d) * a.heads.d;
  a.each = 1;
  while (a.each < 256 && a.each * units < 4 * kBlock && tokens / (2 * a.each) >= 512 &&
         2 * a.each * pairs <= kMostAngles)
    a.each *= 2;
  while (tokens / a.each > kMaxBlocksPerLaunch) a.each *= 2;  // at most 16, and 64 KB of angles
  const dim3 grid(static_cast<unsigned>((tokens + a.each - 1) / a.each));
  const size_t lds = static_cast<size_t>(a.each) * a.pairs * 2 * sizeof(float);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_float_element(dtype, [&](auto e) {
    using T = decltype(e);
    if constexpr (sizeof(T) == 2) {
      if (v == 8) launch_rotary<T, 8>(a, interleaved != 0, grid, lds, s);
    }
    if (v == 4) launch_rotary<T, 4>(a, interleaved != 0, grid, lds, s);
    if (v == 2) launch_rotary<T, 2>(a, interleaved != 0, grid, lds, s);
    if (v == 1) launch_rotary<T, 1>(a, interleaved != 0, grid, lds, s);
    return check_launch("rotary_positions");
  });
}

}  // extern "C"
