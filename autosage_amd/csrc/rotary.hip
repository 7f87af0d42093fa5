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
// rounded to 32: three roundings of 2^-53, less than 2^-51 of the turns, which a sine in
// 32 bits does not show up to 2^24 turns.  The magnitude is rounded to 32 bits and
// multiplied into sine and cosine there, a step more of each (a third product for every
// number, or sines in 64 bits, would save it).
//
// Every row is read and written once: bound by memory, so what counts is that the
// angles cost little and the accesses are wide.  A workgroup takes some tokens, finds
// the sines and cosines of their pairs, one for each thread, and keeps them in LDS for
// all heads of queries and keys; then its threads turn V pairs each, 16 bytes of
// either half, neighbours in a row and rows one behind the other.  The rows of its
// first step are asked for before the angles are found.  16,384 tokens, 40 heads of 128,
// bf16: 57.5 us, 5.8 TB/s; 24 tokens 3.2 us.
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
  int turning;  // units in a row that are turned, the last of which ends with the pairs
  int units;    // those and the units that stay
  int heads;    // of queries and keys
  int each;     // tokens of a workgroup
  int step;     // rows that a workgroup takes at once: a thread has one unit of a row, and that of every step-th
  int step_tokens, step_heads;  // the same as tokens and heads
  Divisor by_units, by_heads, by_pairs;
  float magnitude;
  float sign;
  bool past_caches;  // what is written
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

typedef uint32_t u32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));
template <int V, typename T>
__device__ __forceinline__ void store_numbers(T* to, const RawVec<V * sizeof(T)>& r, bool past_caches) {
  if constexpr (V * sizeof(T) == 16) {
    if (past_caches) {
      __builtin_nontemporal_store(u32x4_a1{r.w[0], r.w[1], r.w[2], r.w[3]}, reinterpret_cast<u32x4_a1*>(to));
      return;
    }
  }
  __builtin_memcpy(to, &r, V * sizeof(T));
}

constexpr int kRotaryAhead = 2;  // units of a thread whose loads are under way at once

template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kBlock) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float angles[];  // [each * pairs] cosines, the same of sines
  const int64_t first = static_cast<int64_t>(blockIdx.x) * a.each;
  const int count = a.tokens - first < a.each ? static_cast<int>(a.tokens - first) : a.each;
  float* const cosines = angles;
  float* const sines = angles + a.each * a.pairs;

  // A thread's unit: two runs of V numbers, a half of what is turned (or stays) apart, so that neighbouring lanes have
  // neighbouring runs (with V = 1 and interleaved pairs, the numbers of a pair).  Runs that would pass the end end with
  // it: what two units share is the same in both.
  const int row0 = quotient(threadIdx.x, a.by_units);
  const int k = static_cast<int>(threadIdx.x) - row0 * a.units + static_cast<int>(blockIdx.y) * kBlock;
  const bool turns = k < a.turning;
  int one;
  int two;
  if (!INTERLEAVED && turns) {
    one = k * V < a.pairs - V ? k * V : a.pairs - V;
    two = a.pairs + one;
  } else if (V == 1 && turns) {
    one = 2 * k;
    two = 2 * k + 1;
  } else {
    const int begin = turns ? 0 : 2 * a.pairs;
    const int last = (turns ? 2 * a.pairs : a.width) - V;
    one = begin + (turns ? k : k - a.turning) * V;
    two = one + (turns ? a.turning : a.units - a.turning) * V;
    one = one < last ? one : last;
    two = two < last ? two : last;
  }
  const bool idle = row0 >= a.step || k >= a.units;  // threads that are no whole row
  int token = quotient(row0, a.by_heads);
  int head = row0 - token * a.heads;
  const int rounds = (count * a.heads + a.step - 1) / a.step;

  for (int r = 0; r < rounds; r += kRotaryAhead) {
    RawVec<V * sizeof(T)> x[kRotaryAhead];
    RawVec<V * sizeof(T)> y[kRotaryAhead];
    T* to[kRotaryAhead];
    int at[kRotaryAhead];
#pragma unroll
    for (int u = 0; u < kRotaryAhead; ++u) {
      const bool second = head >= a.rows[0].heads;
      const int h = second ? head - a.rows[0].heads : head;
      at[u] = idle || token >= count ? -1 : token * a.pairs;
      const int64_t t = first + (at[u] < 0 ? 0 : token);
      const int64_t from = second ? t * a.rows[1].stride[0] + h * a.rows[1].stride[1]
                                  : t * a.rows[0].stride[0] + h * a.rows[0].stride[1];
      const T* row = static_cast<const T*>(second ? a.rows[1].from : a.rows[0].from) + from;
      to[u] = static_cast<T*>(second ? a.rows[1].to : a.rows[0].to) +
              (t * (second ? a.rows[1].heads : a.rows[0].heads) + h) * a.width;
      x[u] = load_numbers<T, V>(row + one);
      y[u] = load_numbers<T, V>(row + two);
      token += a.step_tokens;
      head += a.step_heads;
      const bool over = head >= a.heads;
      token += over ? 1 : 0;
      head -= over ? a.heads : 0;
    }
    if (r == 0) {
      for (int i = threadIdx.x; i < count * a.pairs; i += kBlock) {
        const int t = quotient(i, a.by_pairs);
        const double turned =
            static_cast<double>(a.positions[first + t]) * (a.frequencies[i - t * a.pairs] * kPerTurn);
        float s;
        float c;
        sine_of_turns(turned, &s, &c);
        sines[i] = s * a.magnitude * a.sign;
        cosines[i] = c * a.magnitude;
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kRotaryAhead; ++u) {
      if (at[u] < 0) continue;
      if (turns) {
        T turned[2 * V];
        if constexpr (INTERLEAVED && V > 1) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const RawVec<V * sizeof(T)>& w = half == 0 ? x[u] : y[u];
            const int pair = at[u] + (half == 0 ? one : two) / 2;
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              const float c = cosines[pair + i];
              const float s = sines[pair + i];
              const float p = Elem<T>::get(w.w, 2 * i);
              const float q = Elem<T>::get(w.w, 2 * i + 1);
              turned[half * V + 2 * i] = rounded<T>(p * c - q * s);
              turned[half * V + 2 * i + 1] = rounded<T>(p * s + q * c);
            }
          }
        } else {
          const int pair = at[u] + (INTERLEAVED ? one / 2 : one);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float c = cosines[pair + i];
            const float s = sines[pair + i];
            const float p = Elem<T>::get(x[u].w, i);
            const float q = Elem<T>::get(y[u].w, i);
            turned[i] = rounded<T>(p * c - q * s);
            turned[V + i] = rounded<T>(p * s + q * c);
          }
        }
        __builtin_memcpy(&x[u], turned, V * sizeof(T));
        __builtin_memcpy(&y[u], turned + V, V * sizeof(T));
      }
      store_numbers<V>(to[u] + one, x[u], a.past_caches);
      store_numbers<V>(to[u] + two, y[u], a.past_caches);
    }
  }
}

// The widest runs that neither what is turned (a half of it where halves are pairs) nor what stays is shorter than.
int run_of(int turned, int rest, int widest) {
  int v = widest;
  while (v > 1 && ((turned > 0 && turned < v) || (rest > 0 && rest < v))) v /= 2;
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
  const int v = run_of(interleaved ? 2 * a.pairs : a.pairs, rest, dtype == AS_DTYPE_F32 ? 4 : 8);
  // units of two runs, or of a pair
  const int halves = interleaved && v > 1 ? (a.pairs * 2 + v - 1) / v : 2 * ((a.pairs + v - 1) / v);
  a.turning = (halves + 1) / 2;
  a.units = a.turning + ((rest + v - 1) / v + 1) / 2;
  a.heads = static_cast<int>(heads + key_heads);
  a.step = a.units < kBlock ? kBlock / a.units : 1;
  a.step_tokens = a.step / a.heads;
  a.step_heads = a.step % a.heads;
  a.by_units = divisor_of(a.units);
  // Results go past the caches (16,384 tokens, 40 heads of 128, bf16, with more tokens a workgroup: 61 us, 71 through them), but where what
  // stays leaves runs that are no whole 64 bytes (5,000 tokens, 26 heads of 80, 32 turned, float32: 19 and 16).
  const int run_bytes = (a.units - a.turning) * v * (dtype == AS_DTYPE_F32 ? 4 : 2);
  a.past_caches = rest == 0 || run_bytes % 64 == 0;
  a.by_heads = divisor_of(a.heads);
  a.by_pairs = divisor_of(a.pairs > 0 ? a.pairs : 1);
  // Tokens of a workgroup: as many as give each of its threads a unit, while 512 workgroups are left and the angles
  // have room.  65,536 tokens, 5 heads of 96, 40 turned, float32: 49 us, one token each 79 where 4 heads of 64 in fp16
  // take 16; units for four 60 (16,384 tokens, 40 heads of 128, bf16: 57.5 and 62).  4,096 tokens, 4 heads of 64: 3.2,
  // with 2,048 workgroups 4.7, with 64 6.1.
  const int64_t units = int64_t(a.units) * a.heads;
  a.each = 1;
  while (a.each < 256 && a.each * units < kBlock && tokens / (2 * a.each) >= 512 &&
         2 * a.each * pairs <= kMostAngles)
    a.each *= 2;
  while (tokens / a.each > kMaxBlocksPerLaunch) a.each *= 2;  // at most 16, and 64 KB of angles
  // rows of more units than threads take several workgroups
  const dim3 grid(static_cast<unsigned>((tokens + a.each - 1) / a.each),
                  static_cast<unsigned>((a.units + kBlock - 1) / kBlock));
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
