// Keys and values of new tokens into the pages of their sequences, and back.
//
// Tokens stand one behind the other, those of sequence b at token_ptr[b] ..
// token_ptr[b + 1]; the first of them has position start[b] in its sequence.
// Tokens in front of token_ptr[0] and from token_ptr[sequences] on belong to no
// sequence: a write leaves the cache alone for them, a read gives zeros.
//
// A copy (with a rounding to 8 bits in a quantised cache): bound by memory, or by
// the launch for a few tokens.  A workgroup takes up to 16 tokens: its first wave
// finds their places, then its threads move runs of 8 elements (4 in float32: 16
// bytes of the tokens' type, so that the lanes of a wave are neighbours), all tokens of one
// head before the next head, because the tokens of one head are neighbours in a
// page.  Where a row's maximum is needed its lanes are a power of two, so that it
// takes a few shuffles; else they are as many as the row has runs.
#include "paged_common.h"

namespace as {

namespace {

struct TokenRows {
  void* data;  // [tokens, heads, width]
  int64_t stride[2];
};

constexpr int kMaxTokens = 16;  // of one workgroup
// Elements of one thread, for tokens of T.
template <typename T>
constexpr int kElements = sizeof(T) == 4 ? 4 : 8;
constexpr int kAhead = 4;       // runs of a thread whose loads are under way at once

struct Places {
  int32_t page[kMaxTokens];  // < 0: none
  int32_t slot[kMaxTokens];
};

// The places of tokens first .. first + count - 1, by the first wave.
__device__ __forceinline__ void find_places(const PagedCache& c, const int64_t* __restrict__ token_ptr,
                                            const int64_t* __restrict__ start, int64_t first, int count,
                                            Places& places) {
  if (wave_in_block() == 0) {
    const int64_t row = uniform_i64(wave_row_of_edge(token_ptr, c.sequences, first));
    const int b = block_edge_rows(token_ptr, c.sequences, first, count, row);
    const int64_t t = first + lane_id();
    if (lane_id() < count) {
      const int64_t own = token_ptr[b];
      const int64_t begin = start[b];
      const PageList list = page_list(c, b);
      // A token of the sequence, and a position in front of the sequence or beyond its pages.  `at` stays
      // below 2^62 + 2^26 and begin below what the pages hold, so that no sum wraps whatever the lists hold.
      const bool mine = own >= -(int64_t(1) << 62) && own <= t && t < token_ptr[b + 1];
      const int64_t at = mine ? t - own : 0;
      const int64_t room = list.count * c.page_size;
      const bool outside = begin < -at || begin >= room;
      const int64_t position = mine && !outside ? begin + at : 0;
      const bool none = !mine || outside || position >= room;
      int64_t page = -1;
      int64_t k = 0;
      if (!none) {
        k = position / c.page_size;
        page = c.page_idx[list.begin + k];
      }
      places.page[lane_id()] = page < 0 || page >= c.pages ? -1 : static_cast<int32_t>(page);
      places.slot[lane_id()] = static_cast<int32_t>(none ? 0 : position - k * c.page_size);
    }
  }
  __syncthreads();
}

// Runs of a row: the last one is moved back to end with the row (elements that
// two runs share are moved twice), so that only the elements of rows that are
// shorter than a run are moved one by one.  The accesses ask for the alignment of one byte: the
// hardware has no other requirement.
__device__ __forceinline__ int run_start(int d, int n, int width) {
  const int last = width > n ? width - n : 0;
  return d < last ? d : last;
}
template <int N, typename E>
__device__ __forceinline__ RawVec<N * sizeof(E)> load_elements(const E* from, int width) {
  RawVec<N * sizeof(E)> r;
  static_assert(sizeof(r) == N * sizeof(E));
  if (width >= N) {
    __builtin_memcpy(&r, from, sizeof(r));
  } else {
    E part[N];
#pragma unroll
    for (int i = 0; i < N; ++i) part[i] = from[i < width ? i : width - 1];
    __builtin_memcpy(&r, part, sizeof(r));
  }
  return r;
}
typedef uint32_t u32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));
// STREAM: past the caches, for what a read gives (48 sequences, 8-bit to fp16: 57 us,
// 6.0 TB/s; 95 through them).  What is written to the pages stays: attention reads it next.
template <bool STREAM, int N, typename E>
__device__ __forceinline__ void store_elements(E* to, int width, const RawVec<N * sizeof(E)>& r) {
  static_assert(sizeof(r) == N * sizeof(E));
  if (width >= N) {
    if constexpr (STREAM) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(r)) / 16; ++i)
        __builtin_nontemporal_store(u32x4_a1{r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]},
                                    reinterpret_cast<u32x4_a1*>(to) + i);
    } else {
      __builtin_memcpy(to, &r, sizeof(r));
    }
  } else {
    E part[N];
    __builtin_memcpy(part, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i < width) to[i] = part[i];
    }
  }
}

// How the items of a tensor's rows are told apart: `runs` for each row (i / runs =
// i * magic >> (31 + shift) for i < 2^31, as paged attention divides by the page
// size), then 2^log_tokens tokens of each head.
struct RowItems {
  int runs;
  int shift;
  uint32_t magic;
};
inline RowItems row_items(int width, int elements, bool power_of_two) {
  RowItems it{};
  it.runs = (width + elements - 1) / elements;
  while ((1 << it.shift) < it.runs) ++it.shift;
  if (power_of_two) it.runs = 1 << it.shift;
  it.magic = static_cast<uint32_t>(((uint64_t(1) << (31 + it.shift)) + it.runs - 1) / static_cast<uint64_t>(it.runs));
  return it;
}
// Run, token and head of a thread's item.
struct Item {
  int run;
  int token;
  int head;
};
__device__ __forceinline__ Item item_of(int i, const RowItems& items, int log_tokens) {
  const int r =
      static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(i)) * items.magic) >> (31 + items.shift));
  return Item{i - r * items.runs, r & ((1 << log_tokens) - 1), r >> log_tokens};
}

template <typename T, typename C>
__device__ __forceinline__ void write_rows(const TokenRows& from, const PageTensor& to, const Places& places,
                                           int64_t first, int count, int heads, const RowItems& row, int log_tokens) {
  constexpr int N = kElements<T>;
  const int items = (heads << log_tokens) * row.runs;
  for (int i0 = threadIdx.x; i0 < items; i0 += kAhead * kBlock) {
    RawVec<N * sizeof(T)> raw[kAhead];
    bool active[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const Item it = item_of(i0 + u * kBlock, row, log_tokens);
      active[u] = it.head < heads && it.token < count && it.run * N < to.width && places.page[it.token] >= 0;
      const T* x = static_cast<const T*>(from.data);
      if (active[u])
        raw[u] = load_elements<N>(x + (first + it.token) * from.stride[0] + it.head * from.stride[1] +
                                   run_start(it.run * N, N, to.width), to.width);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const Item it = item_of(i0 + u * kBlock, row, log_tokens);
      int64_t page = 0;
      int64_t slot = 0;
      if (active[u]) {
        page = places.page[it.token];
        slot = places.slot[it.token];
      }
      C* y = static_cast<C*>(to.data) + page * to.stride[0] + it.head * to.stride[1] + slot * to.stride[2] +
             run_start(it.run * N, N, to.width);
      if constexpr (__is_same(T, C)) {
        if (active[u]) store_elements<false, N>(y, to.width, raw[u]);
      } else {
        float x[N];
        float largest = 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          x[k] = active[u] ? Elem<T>::get(raw[u].w, k) : 0.0f;
          largest = fmaxf(largest, finite(x[k]) ? fabsf(x[k]) : 0.0f);
        }
        for (int o = 1; o < row.runs; o <<= 1) largest = fmaxf(largest, __shfl_xor(largest, o, 64));
        const int e = row_exponent(largest);
        const float scale = power_of_two(-e);
        RawVec<N> codes;
#pragma unroll
        for (int k = 0; k < N / 4; ++k)
          codes.w[k] = e4m3_pair(x[4 * k] * scale, x[4 * k + 1] * scale) |
                       e4m3_pair(x[4 * k + 2] * scale, x[4 * k + 3] * scale) << 16;
        if (active[u]) {
          store_elements<false, N>(y, to.width, codes);
          if (it.run == 0)
            to.exponents[page * to.exponent_stride[0] + it.head * to.exponent_stride[1] +
                         slot * to.exponent_stride[2]] = static_cast<int8_t>(e);
        }
      }
    }
  }
}

template <typename C, typename T>
__device__ __forceinline__ void read_rows(const PageTensor& from, const TokenRows& to, const Places& places,
                                          int64_t first, int count, int heads, const RowItems& row, int log_tokens) {
  constexpr int N = kElements<T>;
  const int items = (heads << log_tokens) * row.runs;
  for (int i0 = threadIdx.x; i0 < items; i0 += kAhead * kBlock) {
    RawVec<N * sizeof(C)> raw[kAhead];
    int e[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const Item it = item_of(i0 + u * kBlock, row, log_tokens);
      e[u] = 0;
#pragma unroll
      for (uint32_t& w : raw[u].w) w = 0u;  // zero in every type
      if (it.head < heads && it.token < count && it.run * N < from.width && places.page[it.token] >= 0) {
        const int64_t page = places.page[it.token];
        const int64_t slot = places.slot[it.token];
        raw[u] = load_elements<N>(static_cast<const C*>(from.data) + page * from.stride[0] + it.head * from.stride[1] +
                                   slot * from.stride[2] + run_start(it.run * N, N, from.width), from.width);
        if constexpr (!__is_same(T, C))
          e[u] = from.exponents[page * from.exponent_stride[0] + it.head * from.exponent_stride[1] +
                                slot * from.exponent_stride[2]];
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const Item it = item_of(i0 + u * kBlock, row, log_tokens);
      if (it.head >= heads || it.token >= count || it.run * N >= from.width) continue;
      T* y = static_cast<T*>(to.data) + (first + it.token) * to.stride[0] + it.head * to.stride[1] +
             run_start(it.run * N, N, from.width);
      if constexpr (__is_same(T, C)) {
        store_elements<true, N>(y, from.width, raw[u]);
      } else {
        T values[N];
#pragma unroll
        for (int k = 0; k < N; ++k)
          values[k] = rounded<T>(ldexpf(e4m3_value(static_cast<uint8_t>(raw[u].w[k / 4] >> (8 * (k % 4)))), e[u]));
        RawVec<N * sizeof(T)> r;
        __builtin_memcpy(&r, values, sizeof(r));
        store_elements<true, N>(y, from.width, r);
      }
    }
  }
}

// 4-bit numbers: a lane has 8 elements of a row (16 bytes of a 16-bit type, 4 of codes)
// and four lanes share an exponent, so that neighbouring lanes are neighbours on both
// sides and a group's maximum takes two shuffles.  Rows are cut at whole groups; what
// passes a row's end counts as zeros and is not stored.  Eight numbers are little work,
// so what they need besides counts: a thread has one run of a row, and that of every
// step-th, where a token's rows lie is found once, and a workgroup has keys or values.
// A write goes through the tokens of a head, which
// are neighbours in a page; a read through the heads of a token, which are neighbours
// in the result, so that what goes past the caches fills its lines (20,245 tokens, 10
// heads of 72, fp16, read 21 us; 30 through the tokens of a head).  Keys and values in
// workgroups of their own, whose strides are then the same for all lanes: write and
// read 39.5 us, 42.5 where both are in one; 16 heads of 40 33 and 42.
constexpr int kPairRun = 8;
constexpr int kPairGroup = kGroup / kPairRun;  // lanes that share an exponent
constexpr int64_t kNoPlace = INT64_MIN;
struct PairOffsets {
  int64_t codes[kMaxTokens];  // kNoPlace: none
  int64_t exponents[kMaxTokens];
};
__device__ __forceinline__ void find_offsets(const PageTensor& t, const Places& places, int count, PairOffsets& to) {
  if (threadIdx.x < kMaxTokens) {
    const int token = static_cast<int>(threadIdx.x);
    const int64_t page = token < count ? places.page[token] : -1;
    const int64_t slot = token < count ? places.slot[token] : 0;
    to.codes[token] = page < 0 ? kNoPlace : page * t.stride[0] + slot * t.stride[2];
    to.exponents[token] = page * t.exponent_stride[0] + slot * t.exponent_stride[2];
  }
  __syncthreads();
}

constexpr int kPairAhead = 4;  // runs of a thread whose loads are under way at once
struct PairRows {
  int runs;      // lanes of a row
  int step;      // rows that a workgroup takes at once
  int shift;     // i / runs = i * magic >> (31 + shift)
  uint32_t magic;
  RowItems heads;  // the same for i / heads
};
inline PairRows pair_rows(int width, int heads, int run) {
  const RowItems items = row_items((width + kGroup - 1) / kGroup * (kGroup / run), 1, false);
  return PairRows{items.runs, kBlock / items.runs, items.shift, items.magic, row_items(heads, 1, false)};
}

// Calls f(u, row, token, head, run, whether it is there) for the rows of a tensor, kPairAhead of them at a time, first f
// of all, then g.  HEADS: the heads of a token follow one another, else the tokens of a head.
template <bool HEADS, int RUN, typename F, typename G>
__device__ __forceinline__ void each_row(const PairRows& rows, int width, int heads, int log_tokens, int count, F&& f,
                                         G&& g) {
  const int row0 = static_cast<int>((static_cast<uint64_t>(threadIdx.x) * rows.magic) >> (31 + rows.shift));
  const int run = static_cast<int>(threadIdx.x) - row0 * rows.runs;
  const int all = heads << log_tokens;
  const bool in_row = row0 < rows.step && run * RUN < width;
  for (int r0 = 0; r0 < all; r0 += kPairAhead * rows.step) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int u = 0; u < kPairAhead; ++u) {
        const int at = r0 + u * rows.step + row0;
        int token = at & ((1 << log_tokens) - 1);
        int head = at >> log_tokens;
        if constexpr (HEADS) {
          token = static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(at)) * rows.heads.magic) >>
                                   (31 + rows.heads.shift));
          head = at - token * heads;
        }
        const bool live = in_row && at < all && token < count;
        if (half == 0) {
          f(u, at, token, head, run, live);
        } else {
          g(u, at, token, head, run, live);
        }
      }
    }
  }
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The bits of the largest magnitude of a run, as a float's: those of infinities and NaN are larger than any other's.
template <typename T>
__device__ __forceinline__ uint32_t largest_bits(const uint32_t* w) {
  uint32_t most = 0u;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < kPairRun; ++i) {
      const uint32_t x = w[i] & 0x7fffffffu;
      most = most > x ? most : x;
    }
    return most;
  } else {
#pragma unroll
    for (int i = 0; i < kPairRun / 2; ++i) {
      const uint32_t low = w[i] & 0x7fffu;
      const uint32_t high = (w[i] >> 16) & 0x7fffu;
      most = most > low ? most : low;
      most = most > high ? most : high;
    }
    return __float_as_uint(Elem<T>::get(&most, 0));
  }
}
// Eight numbers over 2^(e - 127), e below 255, rounded to codes, half to even.
template <typename T>
__device__ __forceinline__ uint32_t to_codes(const uint32_t* w, int e) {
  const float scale = __uint_as_float(static_cast<uint32_t>(e) << 23);  // its exponent alone counts: 0 is 2^-127
  uint32_t codes = 0u;
  if constexpr (sizeof(T) == 4) {
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(w[0]), __uint_as_float(w[1]), scale, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(w[2]), __uint_as_float(w[3]), scale, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(w[4]), __uint_as_float(w[5]), scale, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(w[6]), __uint_as_float(w[7]), scale, 3);
  } else if constexpr (__is_same(T, Bf16)) {
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf16x2, w[0]), scale, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf16x2, w[1]), scale, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf16x2, w[2]), scale, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf16x2, w[3]), scale, 3);
  } else {
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(f16x2, w[0]), scale, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(f16x2, w[1]), scale, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(f16x2, w[2]), scale, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(f16x2, w[3]), scale, 3);
  }
  return codes;
}
// What N codes stand for, each number rounded once; NaN for e = 255.
template <typename T, int N>
__device__ __forceinline__ RawVec<N * sizeof(T)> from_codes(uint32_t codes, int e) {
  const float scale = __uint_as_float(static_cast<uint32_t>(e) << 23);
  RawVec<N * sizeof(T)> r;
  static_assert(sizeof(r) == N * sizeof(T));
  if constexpr (sizeof(T) == 4) {
    static_assert(N == 4);
    const f32x2 x[2] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0),
                        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1)};
    __builtin_memcpy(&r, x, sizeof(r));
  } else if constexpr (__is_same(T, Bf16)) {
    const bf16x2 x[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3)};
    __builtin_memcpy(&r, x, sizeof(r));
  } else {
    const f16x2 x[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3)};
    __builtin_memcpy(&r, x, sizeof(r));
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void write_rows_e2m1(const TokenRows& from, const PageTensor& t, const PairOffsets& to,
                                                int64_t first, int count, int heads, const PairRows& rows,
                                                int log_tokens) {
  constexpr int N = kPairRun;
  const T* const tokens = static_cast<const T*>(from.data) + first * from.stride[0];
  uint8_t* const codes_to = static_cast<uint8_t*>(t.data);
  uint8_t* const exponents_to = reinterpret_cast<uint8_t*>(t.exponents);
  RawVec<N * sizeof(T)> raw[kPairAhead];
  const auto load = [&](int u, int, int token, int head, int run, bool live) {
#pragma unroll
    for (uint32_t& w : raw[u].w) w = 0u;
    if (live && to.codes[token] != kNoPlace)
      raw[u] = load_up_to<T, N>(tokens + token * from.stride[0] + head * from.stride[1] + run * N, t.width - run * N);
  };
  const auto store = [&](int u, int, int token, int head, int run, bool live) {
    uint32_t most = largest_bits<T>(raw[u].w);
#pragma unroll
    for (int o = 1; o < kPairGroup; o <<= 1) {
      const uint32_t other = static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), o, 64));
      most = most > other ? most : other;
    }
    const bool odd = most >= 0x7f800000u;
    const int e = odd ? kNanExponent : group_exponent(__uint_as_float(most));
    const uint32_t codes = odd ? 0u : to_codes<T>(raw[u].w, e);
    if (live && to.codes[token] != kNoPlace) {
      uint8_t* y = codes_to + to.codes[token] + head * t.stride[1] + run * (N / 2);
      if (t.width - run * N >= N) {
        __builtin_memcpy(y, &codes, 4);
      } else {
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {
          if (run * N + 2 * k < t.width) y[k] = static_cast<uint8_t>(codes >> (8 * k));
        }
      }
      if (run % kPairGroup == 0)
        exponents_to[to.exponents[token] + head * t.exponent_stride[1] + run / kPairGroup] = static_cast<uint8_t>(e);
    }
  };
  each_row<false, N>(rows, t.width, heads, log_tokens, count, load, store);
}

template <typename T>
__device__ __forceinline__ void read_rows_e2m1(const PageTensor& t, const TokenRows& to, const PairOffsets& from,
                                               int64_t first, int count, int heads, const PairRows& rows,
                                               int log_tokens) {
  constexpr int N = kElements<T>;
  T* const tokens = static_cast<T*>(to.data) + first * to.stride[0];
  const uint8_t* const codes_from = static_cast<const uint8_t*>(t.data);
  const uint8_t* const exponents_from = reinterpret_cast<const uint8_t*>(t.exponents);
  uint32_t codes[kPairAhead];
  int e[kPairAhead];
  const auto load = [&](int u, int, int token, int head, int run, bool live) {
    codes[u] = 0u;
    e[u] = 0;
    if (live && from.codes[token] != kNoPlace) {
      codes[u] = load_up_to<uint8_t, N / 2>(codes_from + from.codes[token] + head * t.stride[1] + run * (N / 2),
                                            (t.width - run * N) / 2).w[0];
      e[u] = exponents_from[from.exponents[token] + head * t.exponent_stride[1] + run / (kGroup / N)];
    }
  };
  const auto store = [&](int u, int row, int, int, int run, bool live) {
    if (!live) return;
    // the results' rows are dense; a row's last run may be a part of one
    store_elements<true, N>(tokens + (row * t.width + run * N), t.width - run * N, from_codes<T, N>(codes[u], e[u]));
  };
  each_row<true, N>(rows, t.width, heads, log_tokens, count, load, store);
}

struct RowShape {
  int log_tokens;
  RowItems key;
  RowItems value;
};

template <typename T, typename C>
__global__ __launch_bounds__(kBlock) void paged_write_kernel(PagedCache c, TokenRows key, TokenRows value,
                                                             const int64_t* __restrict__ token_ptr,
                                                             const int64_t* __restrict__ start, int64_t tokens,
                                                             RowShape shape) {
  __shared__ Places places;
  const int64_t first = static_cast<int64_t>(blockIdx.x) << shape.log_tokens;
  const int64_t left = tokens - first;
  const int count = left < (1 << shape.log_tokens) ? static_cast<int>(left) : 1 << shape.log_tokens;
  find_places(c, token_ptr, start, first, count, places);
  write_rows<T, C>(key, c.key, places, first, count, c.heads, shape.key, shape.log_tokens);
  write_rows<T, C>(value, c.value, places, first, count, c.heads, shape.value, shape.log_tokens);
}

template <typename C, typename T>
__global__ __launch_bounds__(kBlock) void paged_read_kernel(PagedCache c, TokenRows key, TokenRows value,
                                                            const int64_t* __restrict__ token_ptr,
                                                            const int64_t* __restrict__ start, int64_t tokens,
                                                            RowShape shape) {
  __shared__ Places places;
  const int64_t first = static_cast<int64_t>(blockIdx.x) << shape.log_tokens;
  const int64_t left = tokens - first;
  const int count = left < (1 << shape.log_tokens) ? static_cast<int>(left) : 1 << shape.log_tokens;
  find_places(c, token_ptr, start, first, count, places);
  read_rows<C, T>(c.key, key, places, first, count, c.heads, shape.key, shape.log_tokens);
  read_rows<C, T>(c.value, value, places, first, count, c.heads, shape.value, shape.log_tokens);
}

struct PairShape {
  int log_tokens;
  PairRows key;
  PairRows value;
};

template <typename T>
__global__ __launch_bounds__(kBlock) void paged_write_e2m1_kernel(PagedCache c, TokenRows key, TokenRows value,
                                                                  const int64_t* __restrict__ token_ptr,
                                                                  const int64_t* __restrict__ start, int64_t tokens,
                                                                  PairShape shape) {
  __shared__ Places places;
  __shared__ PairOffsets offsets;
  const int64_t first = static_cast<int64_t>(blockIdx.x) << shape.log_tokens;
  const int64_t left = tokens - first;
  const int count = left < (1 << shape.log_tokens) ? static_cast<int>(left) : 1 << shape.log_tokens;
  const PageTensor t = blockIdx.y == 0 ? c.key : c.value;
  const PairRows rows = blockIdx.y == 0 ? shape.key : shape.value;
  find_places(c, token_ptr, start, first, count, places);
  find_offsets(t, places, count, offsets);
  write_rows_e2m1<T>(blockIdx.y == 0 ? key : value, t, offsets, first, count, c.heads, rows, shape.log_tokens);
}

template <typename T>
__global__ __launch_bounds__(kBlock) void paged_read_e2m1_kernel(PagedCache c, TokenRows key, TokenRows value,
                                                                  const int64_t* __restrict__ token_ptr,
                                                                  const int64_t* __restrict__ start, int64_t tokens,
                                                                  PairShape shape) {
  __shared__ Places places;
  __shared__ PairOffsets offsets;
  const int64_t first = static_cast<int64_t>(blockIdx.x) << shape.log_tokens;
  const int64_t left = tokens - first;
  const int count = left < (1 << shape.log_tokens) ? static_cast<int>(left) : 1 << shape.log_tokens;
  const PageTensor t = blockIdx.y == 0 ? c.key : c.value;
  const PairRows rows = blockIdx.y == 0 ? shape.key : shape.value;
  find_places(c, token_ptr, start, first, count, places);
  find_offsets(t, places, count, offsets);
  read_rows_e2m1<T>(t, blockIdx.y == 0 ? key : value, offsets, first, count, c.heads, rows, shape.log_tokens);
}

// Tokens of a workgroup: 16, fewer while that leaves fewer than 1,024 workgroups
// (writes of 2,048 tokens, 8 heads of 128, bf16: 7.1 us; 7.8 with down to 256
// workgroups, 9.0 with 4,096; of 8,192 tokens 12.7, 15.4 and 17.7; of 32,768 tokens
// 44.6, 44.7 and 40.7; reads alike).  Of 4-bit pages fewer than 512 for keys and as many
// for values (4 heads of 64, bf16, up to 16 x 1,700 tokens written and read: 15.0 us;
// 21.2 with 1,024, 14.0 with 256, where 8 heads of 192 and 128 take 20.6, 24.8 and 22.2).
RowShape row_shape(const PagedCache& c, int64_t tokens, int cache_dtype, int dtype, bool write) {
  RowShape s{};
  const int elements = dtype == AS_DTYPE_F32 ? kElements<float> : kElements<Bf16>;
  const bool power_of_two = write && cache_dtype == AS_DTYPE_E4M3;
  s.key = row_items(c.key.width, elements, power_of_two);
  s.value = row_items(c.value.width, elements, power_of_two);
  const int64_t blocks = cache_dtype == AS_DTYPE_E2M1 ? 512 : 1024;
  while ((2 << s.log_tokens) <= kMaxTokens && tokens >> (s.log_tokens + 1) >= blocks) ++s.log_tokens;
  return s;
}

int check_tokens(const PagedCache& c, const void* key, const void* value, const int64_t* token_ptr,
                 const int64_t* start, int64_t tokens, int cache_dtype, int dtype) {
  if (dtype != AS_DTYPE_F32 && dtype != AS_DTYPE_BF16 && dtype != AS_DTYPE_F16)
    return fail(AS_ERR_INVALID_ARGUMENT, "dtype must be AS_DTYPE_F32, AS_DTYPE_BF16 or AS_DTYPE_F16");
  if (!is_coded(cache_dtype) && cache_dtype != dtype)
    return fail(AS_ERR_INVALID_ARGUMENT, "a cache that is not quantised holds the type of its tokens");
  if (tokens < 0 || tokens > kMaxBlocksPerLaunch * kMaxTokens) return fail(AS_ERR_UNSUPPORTED, "at most 2^26 tokens");
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
  const RowShape shape = row_shape(c, tokens, cache->dtype, dtype, true);
  const dim3 grid(static_cast<unsigned>(((tokens - 1) >> shape.log_tokens) + 1));
  const PairShape pairs{shape.log_tokens, pair_rows(c.key.width, c.heads, kPairRun),
                        pair_rows(c.value.width, c.heads, kPairRun)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_float_element(dtype, [&](auto e) {
    using T = decltype(e);
    if (cache->dtype == AS_DTYPE_E2M1) {
      paged_write_e2m1_kernel<T><<<dim3(grid.x, 2), kBlock, 0, s>>>(c, k, v, token_ptr, start, tokens, pairs);
    } else if (cache->dtype == AS_DTYPE_E4M3) {
      paged_write_kernel<T, E4m3><<<grid, kBlock, 0, s>>>(c, k, v, token_ptr, start, tokens, shape);
    } else {
      paged_write_kernel<T, T><<<grid, kBlock, 0, s>>>(c, k, v, token_ptr, start, tokens, shape);
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
  const RowShape shape = row_shape(c, tokens, cache->dtype, dtype, false);
  const dim3 grid(static_cast<unsigned>(((tokens - 1) >> shape.log_tokens) + 1));
  const int run = dtype == AS_DTYPE_F32 ? kElements<float> : kElements<Bf16>;
  const PairShape pairs{shape.log_tokens, pair_rows(c.key.width, c.heads, run), pair_rows(c.value.width, c.heads, run)};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_float_element(dtype, [&](auto e) {
    using T = decltype(e);
    if (cache->dtype == AS_DTYPE_E2M1) {
      paged_read_e2m1_kernel<T><<<dim3(grid.x, 2), kBlock, 0, s>>>(c, k, v, token_ptr, start, tokens, pairs);
    } else if (cache->dtype == AS_DTYPE_E4M3) {
      paged_read_kernel<E4m3, T><<<grid, kBlock, 0, s>>>(c, k, v, token_ptr, start, tokens, shape);
    } else {
      paged_read_kernel<T, T><<<grid, kBlock, 0, s>>>(c, k, v, token_ptr, start, tokens, shape);
    }
    return check_launch("paged_cache_read");
  });
}

}  // extern "C"
