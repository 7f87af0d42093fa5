// Attention of one new token of every sequence over the sequence's pages.
//
//   s[t] = scale * <q, k[t]> + table[bucket(length - 1 - t), h]   for the tokens t that are seen
//   out  = sum_t exp(s[t] - m) v[t] / sum_t exp(s[t] - m),   m = max_t s[t]
//   lse  = m + log(sum_t exp(s[t] - m))
//
// Every key and value is read once, from a page and for all query heads that
// share it: bound by memory from a few thousand tokens on, by the launch below.
//
// The work is cut along the tokens into chunks, one workgroup for each chunk
// and 16 query heads of one key head.  The four waves take turns with tiles of
// 32 tokens (16 in float32) and keep everything in registers: both products are
// matrix instructions of 16 x 16, whose rows are arranged so that the scores
// come out where the second product wants the weights:
//
//   scores   A = keys, B = queries.  Lane (n = lane % 16, g = lane / 16) gets head
//            n and rows g*4 .. g*4+3 of the tile.  Row r of instruction s is token
//            (r/4)*8 + s*4 + r%4, so the lane ends with the tokens g*8 .. g*8+7:
//   out      A = weights: lane (head n, tokens g*8 ..), B = values: lane (column n,
//            the same tokens).  Column n of instruction j is dimension n*8 + j of
//            128, so a lane loads 8 neighbouring numbers of 8 tokens (a row of 128
//            is one contiguous read of 16 lanes) and turns its 8 x 8 block with
//            byte permutes: no shared memory, no shuffle.
//
// With fewer than 16 heads a key head the other rows of the matrix units are
// idle, which costs nothing while memory is the bound.  The maximum is the
// running one, raised only where a score passes it by kSlack, so that most
// tiles rescale nothing; waves and chunks are joined by (maximum, sum,
// weighted sum).  In a call whose sequences have one chunk the workgroup
// writes the result, else a second launch joins the chunks.
//
// Precision: 16-bit products are exact in the matrix units and summed in fp32.
// Weights enter the second product as two 16-bit parts (bf16 keeps 2^-18 of a
// weight, fp16 2^-22), float32 stays float32.  An 8-bit cache is multiplied in
// bf16, which holds its codes exactly; its powers of two are applied to the
// fp32 scores and weights, and queries of other types enter as two (fp16) or
// three (float32) bf16 parts, which hold all of their bits.
//
// A sequence that sees no token, or only scores of -inf, gives zeros and an
// lse of -inf.  A length beyond the sequence's pages or max_length makes its
// results NaN, and so does a page id outside the cache, which is never read.
#include "paged_common.h"
#include "position_map.h"

namespace as {

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kHeads = 16;  // query heads of one workgroup

struct AttentionArgs {
  PagedCache cache;
  const void* query;  // [sequences, heads * group, key width]
  int64_t query_stride[2];
  void* out;           // [sequences, heads * group, value width]
  float* lse;          // [sequences, heads * group], may be null
  const int64_t* lengths;
  const void* table;   // [buckets, heads * group] in the query's type, may be null
  int64_t window;      // 0: every token is seen
  int64_t max_length;  // -1: not known
  int group;
  int head_tiles;      // ceil(group / 16)
  float scale;
  uint32_t page_magic;  // token / page_size = token * page_magic >> (31 + page_shift)
  int page_shift;
  // Chunks.  Their number is known to the host: per_sequence of them for each
  // sequence, or (per_sequence = 0) blocks of pages_per_chunk entries of page_idx,
  // of which sequence b has those from page_ptr[b] / pages_per_chunk + b on.
  int64_t chunks;
  int per_sequence;
  int pages_per_chunk;
  int chunk_tokens;
  float2* part_sum;  // [chunks, heads * group] maximum (in powers of two) and sum
  float* part_out;   // [chunks, heads * group, value width]
};

__device__ __forceinline__ int page_of_token(const AttentionArgs& a, int t) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(t)) * a.page_magic) >> (31 + a.page_shift));
}

struct Seen {
  int begin;
  int end;
  bool bad;  // the length is beyond the pages or max_length: nothing is read
};
__device__ __forceinline__ Seen seen_tokens(const AttentionArgs& a, int b, const PageList& list) {
  int64_t length = a.lengths[b];
  const int64_t room = list.count * a.cache.page_size;
  const int64_t limit = room < (1 << 30) ? room : (1 << 30);
  const bool bad = length > limit || (a.max_length >= 0 && length > a.max_length);
  length = length < 0 || bad ? 0 : length;
  const int64_t begin = a.window > 0 && length > a.window ? length - a.window : 0;
  return Seen{static_cast<int>(begin), static_cast<int>(length), bad};
}

// Chunk k of a sequence covers chunk_tokens tokens from the 8-aligned start of
// what is seen (the start itself where pages are no multiple of 8 tokens).
__device__ __forceinline__ int first_token(const AttentionArgs& a, const Seen& seen) {
  return a.cache.page_size % 8 == 0 ? seen.begin & ~7 : seen.begin;
}
__device__ __forceinline__ int chunk_count(const AttentionArgs& a, const Seen& seen) {
  const int n = seen.end - first_token(a, seen);
  return n <= 0 ? 0 : (n + a.chunk_tokens - 1) / a.chunk_tokens;
}
__device__ __forceinline__ int64_t first_chunk(const AttentionArgs& a, int b) {
  if (a.per_sequence > 0) return static_cast<int64_t>(b) * a.per_sequence;
  const uint32_t begin = static_cast<uint32_t>(page_list(a.cache, b).begin);
  return static_cast<int64_t>(begin / static_cast<uint32_t>(a.pages_per_chunk)) + b;
}
// The sequence of a chunk, by the whole wave: the last whose first chunk is not behind it.
__device__ __forceinline__ int sequence_of_chunk(const AttentionArgs& a, int64_t chunk) {
  if (a.per_sequence > 0) return static_cast<int>(static_cast<uint32_t>(chunk) / static_cast<uint32_t>(a.per_sequence));
  int lo = 0;
  int hi = a.cache.sequences;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int probe = lo + lane_id() * step;
    const uint64_t below = __ballot(probe < hi && first_chunk(a, probe) <= chunk);
    if (below != 0) lo += (63 - __builtin_clzll(below)) * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  return lo;
}

// ---- rows of a page ------------------------------------------------------------
// A lane reads runs of N neighbouring elements.  Where a row does not fill the
// kernel's width, a run that would pass its end is moved back to end with it, so
// that no load needs a guard: the elements it then shares with the run before
// have zeros on the queries' side of the scores, and are the same columns twice
// on the values' side.  NARROW: rows of fewer than 8 elements, one at a time.
__device__ __forceinline__ int run_start(int d, int n, int width) {
  const int last = width > n ? width - n : 0;
  return d < last ? d : last;
}

// The loads ask for the alignment of one byte: the hardware has no other requirement.
template <typename C, int N, bool NARROW>
__device__ __forceinline__ RawVec<N * sizeof(C)> load_run(const C* __restrict__ row, int start, int width) {
  RawVec<N * sizeof(C)> r;
  if constexpr (!NARROW) {
    __builtin_memcpy(&r, row + start, sizeof(r));
  } else {
    C part[N];
#pragma unroll
    for (int i = 0; i < N; ++i) part[i] = row[start + i < width ? start + i : width - 1];
    __builtin_memcpy(&r, part, sizeof(r));
  }
  return r;
}

// ---- element types ---------------------------------------------------------------
// Word pairs of the 16-bit matrix instructions, and how a cache's words get there.
struct Bf16Unit {
  static constexpr float kShift = 0.0f;  // weights are exp2(s - m + kShift)
  __device__ static f32x4 multiply(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
  // two numbers rounded to a word, and what the word holds
  __device__ static uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2));
  }
  __device__ static f32x2 unpack(uint32_t w) { return f32x2{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)}; }
  // infinities and NaN as zeros
  __device__ static uint32_t finite_halves(uint32_t w) {
    return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
  }
};
struct Fp16Unit {
  // weights of at most 2^4 (kSlack) times 2^10: fp16 then keeps those down to 2^-24
  // of the largest with all their bits
  static constexpr float kShift = 10.0f;
  __device__ static f32x4 multiply(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  }
  __device__ static uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, f16x2));
  }
  __device__ static f32x2 unpack(uint32_t w) {
    return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
  }
  __device__ static uint32_t finite_halves(uint32_t w) {
    return ((w & 0x7c00u) == 0x7c00u ? 0u : w & 0xffffu) | ((w & 0x7c000000u) == 0x7c000000u ? 0u : w & 0xffff0000u);
  }
};
template <typename T, typename C>
struct Unit {
  using type = Bf16Unit;
};
template <>
struct Unit<Fp16, Fp16> {
  using type = Fp16Unit;
};

// A running maximum may stay this far (in powers of two) below a score: weights
// are then at most 2^4, which costs no bit of fp32 or bf16.
constexpr float kSlack = 4.0f;

// N 16-bit numbers of a cache as words: what it holds, or its codes in bf16.
template <typename C, int N>
__device__ __forceinline__ void to_words(const RawVec<N * sizeof(C)>& raw, uint32_t* words) {
  if constexpr (__is_same(C, E4m3)) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      words[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw.w[i], 1.0f, false));
      words[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw.w[i], 1.0f, true));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) words[i] = raw.w[i];
  }
}

template <typename T, typename C>
struct Parts {  // 16-bit parts that a query enters the first product in
  static constexpr int value = !__is_same(C, E4m3) ? 1 : (sizeof(T) == 4 ? 3 : (__is_same(T, Fp16) ? 2 : 1));
};
template <typename T, typename C>
struct WeightParts {
  static constexpr int value = sizeof(T) == 4 ? 3 : 2;
};

// ---- one workgroup -----------------------------------------------------------------

template <typename T, typename C, int W, bool NARROW>
__global__ __launch_bounds__(kBlock) void paged_attention_kernel(AttentionArgs a, PositionMap map) {
  constexpr bool kF32 = sizeof(C) == 4;
  constexpr bool kCoded = sizeof(C) == 1;
  constexpr int kTile = kF32 ? 16 : 32;   // tokens of one step of a wave
  constexpr int kOwn = kTile / 4;         // of which a lane weighs this many
  constexpr int kKeyRows = kF32 ? 1 : 2;  // and loads the keys of this many
  constexpr int kKeyRun = kF32 ? 4 : 8;   // dimensions of a key in one load
  constexpr int kKeyRuns = W / (4 * kKeyRun);
  constexpr int kValues = W / 16;         // dimensions of the values a lane holds
  constexpr int kRun = kValues < 8 ? kValues : 8;  // of which neighbours
  constexpr int kBlocks = kValues / kRun;
  constexpr int kQ = Parts<T, C>::value;
  constexpr int kP = WeightParts<T, C>::value;
  using U = typename Unit<T, C>::type;

  __shared__ int32_t border[kMaxBuckets + 1];
  __shared__ float wave_top[kWavesPerBlock][kHeads];
  __shared__ float wave_sum[kWavesPerBlock][kHeads];
  // the bias of the loop, then the waves' sums
  constexpr int kOutFloats = kWavesPerBlock * kHeads * W;
  constexpr int kBiasFloats = kMaxBuckets * kHeads;
  __shared__ float pool[kOutFloats > kBiasFloats ? kOutFloats : kBiasFloats];
  float(*const bias)[kHeads] = reinterpret_cast<float(*)[kHeads]>(pool);
  float(*const wave_out)[kHeads][W] = reinterpret_cast<float(*)[kHeads][W]>(pool);

  const PagedCache& c = a.cache;
  const int lane = lane_id();
  const int n = lane & 15;
  const int g = lane >> 4;
  const int wave = uniform_i32(wave_in_block());
  const int64_t chunk = blockIdx.x;
  const int b = uniform_i32(sequence_of_chunk(a, chunk));
  const int k = uniform_i32(static_cast<int>(chunk - first_chunk(a, b)));
  const int h = static_cast<int>(blockIdx.y) / a.head_tiles;
  const int tile_of_heads = static_cast<int>(blockIdx.y) - h * a.head_tiles;
  const int heads_q = c.heads * a.group;
  const int head0 = h * a.group + tile_of_heads * kHeads;
  const int heads_here = a.group - tile_of_heads * kHeads < kHeads ? a.group - tile_of_heads * kHeads : kHeads;

  const PageList list = page_list(c, b);
  const Seen seen = seen_tokens(a, b, list);
  const int count = chunk_count(a, seen);
  if (k < 0 || (k > 0 && k >= count)) return;  // chunk 0 of a sequence without tokens writes its zeros
  const int base = first_token(a, seen) + k * a.chunk_tokens;
  const int begin = base > seen.begin ? base : seen.begin;
  const int end = base + a.chunk_tokens < seen.end ? base + a.chunk_tokens : seen.end;

  if (a.table != nullptr) {
    const int buckets = map.both_sides ? 2 * map.side : map.side;
    stage_borders(border, map);
    for (int i = threadIdx.x; i < buckets * kHeads; i += kBlock) {
      const int hh = i % kHeads < heads_here ? i % kHeads : 0;
      bias[i / kHeads][i % kHeads] =
          kLog2e * Elem<T>::at(static_cast<const T*>(a.table), static_cast<int64_t>(i / kHeads) * heads_q + head0 + hh);
    }
    __syncthreads();
  }

  // where the lane's runs of a key begin (lane (n, g): dimensions (j*4 + g) * kKeyRun ..), the queries there
  // as operand B, and which elements count (bit i: element i is no repetition)
  int key_at[kKeyRuns];
  uint32_t key_own[kKeyRuns];
  float q32[kF32 ? kKeyRuns : 1][4];
  u32x4 q16[kF32 ? 1 : kKeyRuns][kQ];
  {
    const int head = n < heads_here ? n : 0;
    const T* q_row = static_cast<const T*>(a.query) + b * a.query_stride[0] + (head0 + head) * a.query_stride[1];
#pragma unroll
    for (int j = 0; j < kKeyRuns; ++j) {
      const int d = (j * 4 + g) * kKeyRun;
      key_at[j] = run_start(d, kKeyRun, c.key.width);
      const RawVec<kKeyRun * sizeof(T)> raw = load_run<T, kKeyRun, NARROW>(q_row, key_at[j], c.key.width);
      key_own[j] = 0;
      float q[kKeyRun];
#pragma unroll
      for (int i = 0; i < kKeyRun; ++i) {
        const bool mine = key_at[j] + i >= d && key_at[j] + i < c.key.width;
        key_own[j] |= mine ? 1u << i : 0u;
        q[i] = mine && n < heads_here ? Elem<T>::get(raw.w, i) : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < (kF32 ? 4 : 0); ++i) q32[j][i] = q[i];
#pragma unroll
      for (int i = 0; i < (kF32 ? 0 : 4); ++i) {
#pragma unroll
        for (int p = 0; p < kQ; ++p) {
          const uint32_t w = U::pack(q[(2 * i) % kKeyRun], q[(2 * i + 1) % kKeyRun]);
          q16[j][p][i] = w;
          q[(2 * i) % kKeyRun] -= U::unpack(w)[0];
          q[(2 * i + 1) % kKeyRun] -= U::unpack(w)[1];
        }
      }
    }
  }
  int value_at[kBlocks];
#pragma unroll
  for (int j = 0; j < kBlocks; ++j) value_at[j] = run_start(j * 128 + n * kRun, kRun, c.value.width);

  f32x4 acc[kValues];
  float top;  // of head n, the same in its four lanes
  float sum;  // of head n and the tokens of this lane

  const float to_log2 = a.scale * kLog2e;
  const C* key_base = static_cast<const C*>(c.key.data) + h * c.key.stride[1];
  const C* value_base = static_cast<const C*>(c.value.data) + h * c.value.stride[1];
  const int8_t* key_e_base = kCoded ? c.key.exponents + h * c.key.exponent_stride[1] : nullptr;
  const int8_t* value_e_base = kCoded ? c.value.exponents + h * c.value.exponent_stride[1] : nullptr;
  const int64_t* pages = c.page_idx + list.begin;
  const bool aligned8 = c.page_size % 8 == 0;
  // tokens of this lane: the first of those it loads keys of (the other is 4 further), and of those it weighs
  const int key_token = kF32 ? n : (n >> 2) * 8 + (n & 3);
  const int own_token = g * kOwn;

  // Infinite numbers: a repeated element of a key times zero, or an infinite value
  // times a part of its weight that is zero, would be NaN where the result is
  // infinite.  A wave that ends with NaN runs again without the former, with the
  // parts of the weights for finite values and one for the others.  (8-bit numbers
  // have no infinities.)
  for (bool careful = false;; careful = true) {
#pragma unroll
  for (int j = 0; j < kValues; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  top = -INFINITY;
  sum = 0.0f;
  for (int t0 = base + wave * kTile; t0 < end; t0 += kWavesPerBlock * kTile) {
    // the rows of the lane's tokens; a token outside what is seen stands for one whose place exists
    const C* key_row[kKeyRows];
    const C* value_row[kOwn];
    const int8_t* key_e_at[kCoded ? kOwn : 1];
    const int8_t* value_e_at[kCoded ? kOwn : 1];
    uint32_t bad_tokens = 0;
    const auto place = [&](int t, int& slot, bool& bad) {
      const int e = page_of_token(a, t);
      slot = t - e * c.page_size;
      const int64_t id = pages[e];
      bad = id < 0 || id >= c.pages;
      return bad ? int64_t(0) : id;
    };
    if (aligned8) {
      // blocks of 8 tokens lie in one page
      const int last = (end - 1) & ~7;
      int slot;
      bool bad;
      int t = (t0 + key_token) & ~7;
      int64_t page = place(t < last ? t : last, slot, bad);
#pragma unroll
      for (int s = 0; s < kKeyRows; ++s)
        key_row[s] = key_base + page * c.key.stride[0] + (slot + (key_token & 7) + s * 4) * c.key.stride[2];
      t = (t0 + own_token) & ~7;
      page = place(t < last ? t : last, slot, bad);
      slot += own_token & 7;
      if (bad) bad_tokens = 0xffu;
#pragma unroll
      for (int e = 0; e < kOwn; ++e) {
        value_row[e] = value_base + page * c.value.stride[0] + (slot + e) * c.value.stride[2];
        if constexpr (kCoded) {
          key_e_at[e] = key_e_base + page * c.key.exponent_stride[0] + (slot + e) * c.key.exponent_stride[2];
          value_e_at[e] = value_e_base + page * c.value.exponent_stride[0] + (slot + e) * c.value.exponent_stride[2];
        }
      }
    } else {
      int slot;
      bool bad;
#pragma unroll
      for (int s = 0; s < kKeyRows; ++s) {
        const int t = t0 + key_token + s * 4;
        const int64_t page = place(t < end ? t : end - 1, slot, bad);
        key_row[s] = key_base + page * c.key.stride[0] + slot * c.key.stride[2];
      }
#pragma unroll
      for (int e = 0; e < kOwn; ++e) {
        const int t = t0 + own_token + e;
        const int64_t page = place(t < end ? t : end - 1, slot, bad);
        if (bad) bad_tokens |= 1u << e;
        value_row[e] = value_base + page * c.value.stride[0] + slot * c.value.stride[2];
        if constexpr (kCoded) {
          key_e_at[e] = key_e_base + page * c.key.exponent_stride[0] + slot * c.key.exponent_stride[2];
          value_e_at[e] = value_e_base + page * c.value.exponent_stride[0] + slot * c.value.exponent_stride[2];
        }
      }
    }

    RawVec<kKeyRun * sizeof(C)> key_raw[kKeyRows][kKeyRuns];
#pragma unroll
    for (int s = 0; s < kKeyRows; ++s) {
#pragma unroll
      for (int j = 0; j < kKeyRuns; ++j) key_raw[s][j] = load_run<C, kKeyRun, NARROW>(key_row[s], key_at[j], c.key.width);
    }
    RawVec<kRun * sizeof(C)> value_raw[kBlocks][kOwn];
#pragma unroll
    for (int e = 0; e < kOwn; ++e) value_raw[0][e] = load_run<C, kRun, NARROW>(value_row[e], value_at[0], c.value.width);
    int key_e[kOwn], value_e[kOwn];
#pragma unroll
    for (int e = 0; e < (kCoded ? kOwn : 0); ++e) {
      key_e[e] = *key_e_at[e];
      value_e[e] = *value_e_at[e];
    }

    f32x4 score[kKeyRows];
#pragma unroll
    for (int s = 0; s < kKeyRows; ++s) {
      score[s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < kKeyRuns; ++j) {
        if constexpr (kF32) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w = key_raw[s][j].w[i];
            if (careful && !((key_own[j] >> i) & 1)) w = 0u;
            score[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w), q32[j][i], score[s], 0, 0, 0);
          }
        } else {
          uint32_t w[4];
          to_words<C, 8>(key_raw[s][j], w);
          if (!kCoded && careful) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t two = key_own[j] >> (2 * i);
              w[i] &= (two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
            }
          }
#pragma unroll
          for (int p = 0; p < kQ; ++p) score[s] = U::multiply(u32x4{w[0], w[1], w[2], w[3]}, q16[j][p], score[s]);
        }
      }
    }

    // scores in powers of two
    float s2[kOwn];
    float most = -INFINITY;
#pragma unroll
    for (int e = 0; e < kOwn; ++e) {
      s2[e] = score[e / 4][e % 4] * to_log2;
      if constexpr (kCoded) s2[e] = ldexpf(s2[e], key_e[e]);
    }
    if (a.table != nullptr) {
      // every token of the tile farther than the last border: one number a head
      if (seen.end - t0 - kTile >= border[map.side - 1]) {
        const float far = bias[map.side - 1][n];
#pragma unroll
        for (int e = 0; e < kOwn; ++e) s2[e] += far;
      } else {
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
          const int away = seen.end - 1 - (t0 + own_token + e);
          s2[e] += bias[bucket_of_distance(border, map, away < 0 ? 0 : away)][n];
        }
      }
    }
    const bool edge = t0 < begin || t0 + kTile > end;
    if (edge || __any(bad_tokens != 0)) {
#pragma unroll
      for (int e = 0; e < kOwn; ++e) {
        const int t = t0 + own_token + e;
        const bool out_of_sight = t < begin || t >= end;
        if ((bad_tokens >> e) & 1) s2[e] = NAN;
        if (out_of_sight) s2[e] = -INFINITY;
      }
    }
#pragma unroll
    for (int e = 0; e < kOwn; ++e) most = fmaxf(most, s2[e]);

    if (__any(most > top + kSlack)) {
      most = fmaxf(most, __shfl_xor(most, 16, 64));
      most = fmaxf(most, __shfl_xor(most, 32, 64));
      const float next = fmaxf(top, most);
      const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - next);
      top = next;
      sum *= keep;
      // lane (n, g) holds the heads g*4 .. g*4+3 of its columns
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = __shfl(keep, g * 4 + i, 64);
#pragma unroll
        for (int j = 0; j < kValues; ++j) acc[j][i] *= f;
      }
    }
    const float from = top == -INFINITY ? 0.0f : top - U::kShift;
    float weight[kOwn];
#pragma unroll
    for (int e = 0; e < kOwn; ++e) {
      weight[e] = __builtin_amdgcn_exp2f(s2[e] - from);
      sum += weight[e];
      if constexpr (kCoded) weight[e] = ldexpf(weight[e], value_e[e]);
    }
    u32x4 w16[kP];
    u32x4 one16;
    if (!kF32 && !kCoded && careful) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = weight[(2 * i) % kOwn];
        const float y = weight[(2 * i + 1) % kOwn];
        one16[i] = U::pack(x > 0.0f ? 1.0f : x, y > 0.0f ? 1.0f : y);
      }
    }
#pragma unroll
    for (int p = 0; p < (kF32 ? 0 : kP); ++p) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = U::pack(weight[(2 * i) % kOwn], weight[(2 * i + 1) % kOwn]);
        w16[p][i] = w;
        weight[(2 * i) % kOwn] -= U::unpack(w)[0];
        weight[(2 * i + 1) % kOwn] -= U::unpack(w)[1];
      }
    }

#pragma unroll
    for (int jb = 0; jb < kBlocks; ++jb) {
      if (jb + 1 < kBlocks) {
#pragma unroll
        for (int e = 0; e < kOwn; ++e)
          value_raw[jb + 1][e] = load_run<C, kRun, NARROW>(value_row[e], value_at[jb + 1], c.value.width);
      }
      if (edge) {
        // a value out of sight may be anything; its weight is zero, and so has to be the product
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
          const int t = t0 + own_token + e;
#pragma unroll
          for (uint32_t& w : value_raw[jb][e].w) w = t < begin || t >= end ? 0u : w;
        }
      }
      if constexpr (kF32) {
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
#pragma unroll
          for (int j = 0; j < kRun; ++j)
            acc[jb * kRun + j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                weight[e], __uint_as_float(value_raw[jb][e].w[j]), acc[jb * kRun + j], 0, 0, 0);
        }
      } else {
        uint32_t words[8][kRun / 2];
#pragma unroll
        for (int e = 0; e < 8; ++e) to_words<C, kRun>(value_raw[jb][e % kOwn], words[e]);
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
          u32x4 column;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            column[i] = __builtin_amdgcn_perm(words[2 * i + 1][j / 2], words[2 * i][j / 2],
                                              j % 2 == 0 ? 0x05040100u : 0x07060302u);
          if (!kCoded && careful) {
            u32x4 others;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              others[i] = column[i] ^ U::finite_halves(column[i]);
              column[i] ^= others[i];
            }
            acc[jb * kRun + j] = U::multiply(one16, others, acc[jb * kRun + j]);
          }
#pragma unroll
          for (int p = 0; p < kP; ++p) acc[jb * kRun + j] = U::multiply(w16[p], column, acc[jb * kRun + j]);
        }
      }
    }
  }
  if (kCoded || careful) break;
  bool odd = sum != sum;
#pragma unroll
  for (int j = 0; j < kValues; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) odd = odd || acc[j][i] != acc[j][i];
  }
  if (!__any(odd)) break;
  }

  // join the waves
  sum += __shfl_xor(sum, 16, 64);
  sum += __shfl_xor(sum, 32, 64);
  if (g == 0) {
    wave_top[wave][n] = top;
    wave_sum[wave][n] = sum;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int hh = g * 4 + i;
    if (hh < heads_here) {
      float most = wave_top[0][hh];
#pragma unroll
      for (int w = 1; w < kWavesPerBlock; ++w) most = fmaxf(most, wave_top[w][hh]);
      const float mine = wave_top[wave][hh];
      const float f = mine == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mine - most);
#pragma unroll
      for (int j = 0; j < kValues; ++j) {
        const int d = value_at[j / kRun] + j % kRun;
        if (!NARROW || d < c.value.width) wave_out[wave][hh][d] = acc[j][i] * f;
      }
    }
  }
  __syncthreads();
  const int width = c.value.width;
  const bool last = count <= 1;  // the whole sequence is here
  for (int i = threadIdx.x; i < heads_here * width; i += kBlock) {
    const int hh = i / width;
    const int d = i - hh * width;
    float most = wave_top[0][hh];
#pragma unroll
    for (int w = 1; w < kWavesPerBlock; ++w) most = fmaxf(most, wave_top[w][hh]);
    float total = 0.0f;
    float x = 0.0f;
#pragma unroll
    for (int w = 0; w < kWavesPerBlock; ++w) {
      const float mine = wave_top[w][hh];
      total += (mine == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mine - most)) * wave_sum[w][hh];
      x += wave_out[w][hh][d];
    }
    if (last) {
      const int64_t row = static_cast<int64_t>(b) * heads_q + head0 + hh;
      const bool none = total == 0.0f;
      static_cast<T*>(a.out)[row * width + d] = rounded<T>(seen.bad ? NAN : (none ? 0.0f : x / total));
      if (a.lse != nullptr && d == 0)
        a.lse[row] = seen.bad ? NAN : (none ? -INFINITY : (most - U::kShift + __builtin_amdgcn_logf(total)) * kLn2);
    } else {
      const int64_t row = chunk * heads_q + head0 + hh;
      a.part_out[row * width + d] = x;
      if (d == 0) a.part_sum[row] = make_float2(most, total);
    }
  }
}

// Joins the chunks of one sequence and query head: one workgroup, whose waves
// take turns with the chunks and whose lanes hold the width.
template <typename T>
__global__ __launch_bounds__(kBlock) void paged_attention_join_kernel(AttentionArgs a, float shift) {
  __shared__ float2 wave_sums[kWavesPerBlock];
  __shared__ float wave_out[kWavesPerBlock][kMaxWidth];
  const PagedCache& c = a.cache;
  const int heads_q = c.heads * a.group;
  const int b = blockIdx.y;
  const int hq = blockIdx.x;
  const PageList list = page_list(c, b);
  const Seen seen = seen_tokens(a, b, list);
  const int count = chunk_count(a, seen);
  if (count <= 1) return;
  const int64_t first = first_chunk(a, b);
  const int lane = lane_id();
  const int wave = wave_in_block();
  const int width = c.value.width;
  constexpr int kParts = kMaxWidth / kWave;
  float acc[kParts];
#pragma unroll
  for (int i = 0; i < kParts; ++i) acc[i] = 0.0f;
  float top = -INFINITY;
  float sum = 0.0f;
  for (int k = wave; k < count && first + k < a.chunks; k += kWavesPerBlock) {
    const int64_t row = (first + k) * heads_q + hq;
    const float2 part = a.part_sum[row];
    const float next = fmaxf(top, part.x);
    const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - next);
    const float f = part.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(part.x - next);
    top = next;
    sum = sum * keep + part.y * f;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int d = lane + i * kWave;
      if (d < width) acc[i] = acc[i] * keep + a.part_out[row * width + d] * f;
    }
  }
  if (lane == 0) wave_sums[wave] = make_float2(top, sum);
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    if (lane + i * kWave < width) wave_out[wave][lane + i * kWave] = acc[i];
  }
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= width) return;
  float most = wave_sums[0].x;
#pragma unroll
  for (int w = 1; w < kWavesPerBlock; ++w) most = fmaxf(most, wave_sums[w].x);
  float total = 0.0f;
  float x = 0.0f;
#pragma unroll
  for (int w = 0; w < kWavesPerBlock; ++w) {
    const float f = wave_sums[w].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(wave_sums[w].x - most);
    total += wave_sums[w].y * f;
    x += wave_out[w][d] * f;
  }
  const int64_t row = static_cast<int64_t>(b) * heads_q + hq;
  const bool none = total == 0.0f;
  static_cast<T*>(a.out)[row * width + d] = rounded<T>(none ? 0.0f : x / total);
  if (a.lse != nullptr && d == 0)
    a.lse[row] = none ? -INFINITY : (most - shift + __builtin_amdgcn_logf(total)) * kLn2;
}

// ---- launch --------------------------------------------------------------------------

// Workgroups that a call is cut into at least, while a chunk keeps kMinChunk tokens.
constexpr int64_t kTargetBlocks = 2048;
constexpr int64_t kMinChunk = 128;
constexpr int64_t kMaxChunk = 4096;

struct Split {
  int64_t chunks;
  int64_t per_sequence;
  int64_t pages_per_chunk;
  int64_t chunk_tokens;
};
Split split_of(const as_paged_cache* c, int64_t group, int64_t window, int64_t max_length) {
  const int64_t units = c->heads * ((group + kHeads - 1) / kHeads);
  // tokens of one sequence at most, and of all of them
  int64_t longest = c->page_idx_len * c->page_size;
  if (max_length >= 0 && max_length < longest) longest = max_length;
  if (window > 0 && window + 8 < longest) longest = window + 8;
  if (longest < 1) longest = 1;
  int64_t all = c->page_idx_len * c->page_size;
  if (all > longest * c->sequences) all = longest * c->sequences;
  int64_t tokens = all * units / kTargetBlocks;
  tokens = tokens < kMinChunk ? kMinChunk : (tokens > kMaxChunk ? kMaxChunk : tokens);
  tokens = (tokens + kMinChunk - 1) / kMinChunk * kMinChunk;
  Split s{};
  const int64_t each = (longest + tokens - 1) / tokens;
  if (max_length >= 0 || each == 1) {
    s.per_sequence = each;
    s.chunk_tokens = tokens;
    s.chunks = each * c->sequences;
  } else {
    s.pages_per_chunk = (tokens + c->page_size - 1) / c->page_size;
    s.chunk_tokens = s.pages_per_chunk * c->page_size;
    s.chunks = c->page_idx_len / s.pages_per_chunk + c->sequences;
  }
  return s;
}

size_t part_bytes(const Split& s, int64_t heads_q, int64_t width) {
  if (s.per_sequence == 1) return 8;
  return align_up(static_cast<size_t>(s.chunks) * heads_q * sizeof(float2), 256) +
         static_cast<size_t>(s.chunks) * heads_q * width * sizeof(float);
}

template <typename T, typename C, int W>
void launch_width(const AttentionArgs& a, const PositionMap& map, dim3 grid, hipStream_t s) {
  if (a.cache.key.width >= 8 && a.cache.value.width >= 8) {
    paged_attention_kernel<T, C, W, false><<<grid, kBlock, 0, s>>>(a, map);
  } else {
    paged_attention_kernel<T, C, W, true><<<grid, kBlock, 0, s>>>(a, map);
  }
}

template <typename T, typename C>
int launch_attention(const AttentionArgs& a, const PositionMap& map, hipStream_t s) {
  const int width = a.cache.key.width > a.cache.value.width ? a.cache.key.width : a.cache.value.width;
  const dim3 grid(static_cast<unsigned>(a.chunks), static_cast<unsigned>(a.cache.heads * a.head_tiles));
  if (width <= 64) {
    launch_width<T, C, 64>(a, map, grid, s);
  } else if (width <= 128) {
    launch_width<T, C, 128>(a, map, grid, s);
  } else {
    launch_width<T, C, 256>(a, map, grid, s);
  }
  if (const int bad = check_launch("paged_attention")) return bad;
  if (a.per_sequence == 1) return AS_OK;
  paged_attention_join_kernel<T><<<dim3(static_cast<unsigned>(a.cache.heads * a.group),
                                       static_cast<unsigned>(a.cache.sequences)),
                                   kBlock, 0, s>>>(a, Unit<T, C>::type::kShift);
  return check_launch("paged_attention (join)");
}

}  // namespace

}  // namespace as

using namespace as;

extern "C" {

size_t as_paged_attention_workspace_bytes(const as_paged_cache* cache, int64_t group, int64_t window,
                                          int64_t max_length) {
  PagedCache c;
  if (read_paged_cache(cache, &c) != AS_OK || group < 1) return 8;
  return part_bytes(split_of(cache, group, window, max_length), cache->heads * group, cache->value_width);
}

int as_paged_attention(const as_paged_cache* cache, const void* query, const int64_t* query_strides, void* out,
                       float* lse, const int64_t* lengths, int64_t group, float scale, int64_t window,
                       const void* table, int64_t buckets, const int32_t* borders, int both_sides, int64_t max_length,
                       int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  AttentionArgs a{};
  if (const int bad = read_paged_cache(cache, &a.cache)) return bad;
  if (dtype != AS_DTYPE_F32 && dtype != AS_DTYPE_BF16 && dtype != AS_DTYPE_F16)
    return fail(AS_ERR_INVALID_ARGUMENT, "dtype must be AS_DTYPE_F32, AS_DTYPE_BF16 or AS_DTYPE_F16");
  if (cache->dtype != AS_DTYPE_E4M3 && cache->dtype != dtype)
    return fail(AS_ERR_INVALID_ARGUMENT, "a cache that is not quantised holds the type of the queries");
  if (group < 1 || group * a.cache.heads > 65535)
    return fail(AS_ERR_INVALID_ARGUMENT, "query heads must lie in [1, 65535]");
  if (window < 0 || max_length < -1) return fail(AS_ERR_INVALID_ARGUMENT, "window and max_length must be positive");
  PositionMap map{};
  if (table != nullptr) {
    if (const int bad = fill_position_map(&map, borders, buckets, both_sides)) return bad;
  }
  const Split split = split_of(cache, group, window, max_length);
  const size_t need = part_bytes(split, cache->heads * group, cache->value_width);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(AS_ERR_WORKSPACE, "paged attention needs %zu workspace bytes", need);
  if (a.cache.sequences == 0) return AS_OK;
  if (a.cache.sequences > 65535 || split.chunks > kMaxBlocksPerLaunch || cache->page_idx_len > INT32_MAX)
    return fail(AS_ERR_UNSUPPORTED, "at most 65535 sequences, 2^31 - 1 list entries and 2^22 chunks");
  if (query == nullptr || query_strides == nullptr || out == nullptr || lengths == nullptr)
    return fail(AS_ERR_INVALID_ARGUMENT, "null pointer argument");
  const size_t size = dtype == AS_DTYPE_F32 ? 4 : 2;
  if (!aligned(query, size) || !aligned(out, size) || !aligned(table, size))
    return fail(AS_ERR_INVALID_ARGUMENT, "query, out and table must be aligned to their elements");
  a.query = query;
  a.query_stride[0] = query_strides[0];
  a.query_stride[1] = query_strides[1];
  a.out = out;
  a.lse = lse;
  a.lengths = lengths;
  a.table = table;
  a.window = window;
  a.max_length = max_length;
  a.group = static_cast<int>(group);
  a.head_tiles = static_cast<int>((group + kHeads - 1) / kHeads);
  a.scale = scale;
  // t / S for t < 2^31: M = ceil(2^(31 + s) / S) with s = ceil(log2 S) is below 2^32, and t * M >> (31 + s) is exact
  while ((1 << a.page_shift) < a.cache.page_size) ++a.page_shift;
  a.page_magic = static_cast<uint32_t>(((uint64_t(1) << (31 + a.page_shift)) + a.cache.page_size - 1) /
                                       static_cast<uint64_t>(a.cache.page_size));
  a.chunks = split.chunks;
  a.per_sequence = static_cast<int>(split.per_sequence);
  a.pages_per_chunk = static_cast<int>(split.pages_per_chunk);
  a.chunk_tokens = static_cast<int>(split.chunk_tokens);
  a.part_sum = static_cast<float2*>(workspace);
  a.part_out = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                        align_up(static_cast<size_t>(split.chunks) * cache->heads * group *
                                                     sizeof(float2), 256));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_float_element(dtype, [&](auto e) {
    using T = decltype(e);
    if (cache->dtype == AS_DTYPE_E4M3) return launch_attention<T, E4m3>(a, map, s);
    return launch_attention<T, T>(a, map, s);
  });
}

}  // extern "C"
