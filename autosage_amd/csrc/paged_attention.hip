// Attention of one new token of every sequence over the sequence's pages.
//
//   s[t] = scale * <q, k[t]> + table[bucket(length - 1 - t), h]   for the tokens t that are seen
//   out  = sum_t exp(s[t] - m) v[t] / sum_t exp(s[t] - m),   m = max_t s[t]
//   lse  = m + log(sum_t exp(s[t] - m))
//
// Every key and value is read once, from a page and for all query heads that
// share it: bound by memory from a few thousand tokens on, by the launch below.
//
// The work is cut into equal shares: the tiles of 32 tokens of all sequences, one
// sequence behind the other, are dealt out evenly to the workgroups of 16 query
// heads of one key head, which find their share from the lengths on the device
// (the host knows neither the lengths nor, in a captured graph, the batch they
// belong to).  A share may end inside a sequence and reach over several; each
// part of a sequence in a share gives a partial result.  One workgroup's four
// waves take turns with the tiles of a part (16 tokens in float32) and keep
// everything in registers: both products are
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
//            byte permutes: no shared memory, no shuffle.  (Rows of 64 and 192: 4 numbers.)
//
// With fewer than 16 heads a key head the other rows of the matrix units are
// idle, which costs nothing while memory is the bound.  The maximum is the
// running one, raised only where a score passes it by kSlack, so that most
// tiles rescale nothing; waves and parts are joined by (maximum, sum,
// weighted sum).  A part that is all of a sequence writes the result itself; a
// second launch joins the parts of the others, and is left out where the host
// knows that the sequences are short (kSingle tokens: one workgroup each).
//
// Measured: 64 sequences of up to 8,192 tokens, 32 query heads over 8 of width 128,
// bf16: 219 us, 5.5 TB/s (a large copy reaches 4.9 on this card); two of 131,072
// from an 8-bit cache: 111 us, 4.9 TB/s; one of 17 tokens: 6 us, the latency of six
// dependent reads.
//
// Precision: 16-bit products are exact in the matrix units and summed in fp32.
// Weights enter the second product as two 16-bit parts (bf16 keeps 2^-18 of a
// weight, fp16 2^-22), float32 stays float32.  An 8-bit cache is multiplied in
// bf16, which holds its codes exactly; its powers of two are applied to the
// fp32 scores and weights, and queries of other types enter as two (fp16) or
// three (float32) bf16 parts, which hold all of their bits.  (Rows of values below
// 2^-105 bring weights into the range where bf16 has fewer bits: off by 6e-5 of the
// result at 1e-34, 5e-3 at 1e-37.)
//
// A sequence that sees no token, or only scores of -inf, gives zeros and an
// lse of -inf.  A length beyond the sequence's pages or max_length makes its
// results NaN, and so does a page id outside the cache, which is never read.

#include "paged_shares.h"

namespace as {

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// How a call reaches the rows of its tokens.  kBlocks8: pages are a multiple of 8
// tokens, so that the blocks of 8 which a lane works on lie in one page each, and
// the exponents of a page's tokens are neighbours.  kTokens: every token is looked
// up.  kNarrow: so it is, and rows of fewer than 8 elements are read one at a time.
enum Mode { kBlocks8, kTokens, kNarrow };

// ---- rows of a page ------------------------------------------------------------
// A lane reads runs of N neighbouring elements.  Where a row does not fill the
// kernel's width, a run that would pass its end is moved back to end with it, so
// that no load needs a guard: the elements it then shares with the run before
// have zeros on the queries' side of the scores, and are the same columns twice
// on the values' side.
__device__ __forceinline__ int run_start(int d, int n, int width) {
  const int last = width > n ? width - n : 0;
  return d < last ? d : last;
}

// The loads ask for the alignment of one byte: the hardware has no other requirement.
template <typename C, int N, int MODE>
__device__ __forceinline__ RawVec<N * sizeof(C)> load_run(const C* __restrict__ row, int start, int width) {
  RawVec<N * sizeof(C)> r;
  static_assert(sizeof(r) == N * sizeof(C));
  if constexpr (MODE != kNarrow) {
    __builtin_memcpy(&r, row + start, sizeof(r));
  } else {
    // zeros behind the row: an infinite number there would make NaN of the queries' zeros
    C part[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const C x = row[start + i < width ? start + i : width - 1];
      part[i] = start + i < width ? x : C{};
    }
    __builtin_memcpy(&r, part, sizeof(r));
  }
  return r;
}

// ---- element types ---------------------------------------------------------------
// Word pairs of the 16-bit matrix instructions, and how a cache's words get there.
struct Bf16Unit {
  static constexpr float kShift = 0.0f;  // weights are exp2((s - m) * kLog2e + kShift)
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

// A running maximum may stay this far below a score: weights are then at most
// 2^4, which costs no bit of fp32 or bf16.
constexpr float kSlack = 4.0f * kLn2;

// exp(d) for the difference d of two scores.  Scores stay as they are and only
// differences are brought to powers of two: a score of -3e38 (a mask) times kLog2e
// would be infinite.
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

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

template <typename T, typename C, int W, int MODE>
__global__ __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(W > 128 && MODE != kNarrow ? 2 : 1))) void
paged_attention_kernel(AttentionArgs a, PositionMap map) {
  constexpr bool kF32 = sizeof(C) == 4;
  constexpr bool kCoded = sizeof(C) == 1;
  constexpr int kTile = kF32 ? 16 : 32;   // tokens of one step of a wave
  constexpr int kOwn = kTile / 4;         // of which a lane weighs this many
  constexpr int kKeyRows = kF32 ? 1 : 2;  // and loads the keys of this many
  constexpr int kKeyRun = kF32 ? 4 : 8;   // dimensions of a key in one load
  constexpr int kKeyRuns = W / (4 * kKeyRun);
  constexpr int kValues = W / 16;         // dimensions of the values a lane holds
  constexpr int kRun = kValues % 8 == 0 ? 8 : 4;  // of which neighbours
  constexpr int kBlocks = kValues / kRun;
  // rows beyond 128 take too many registers to ask for keys and values at once
  constexpr bool kLater = kBlocks > 1;
  constexpr int kQ = Parts<T, C>::value;
  constexpr int kP = WeightParts<T, C>::value;
  using U = typename Unit<T, C>::type;

  __shared__ int32_t border[kMaxBuckets + 1];
  __shared__ ShareSums share_sums;
  __shared__ float wave_top[kWavesPerBlock][kHeads];
  __shared__ float wave_sum[kWavesPerBlock][kHeads];
  __shared__ float bias[kMaxBuckets][kHeads];  // of the keys in front of the query
  constexpr int kOutWaves = kLater ? 2 : kWavesPerBlock;
  __shared__ float wave_out[kOutWaves][kHeads][W];
  __shared__ u32x4 q_shared[kLater ? kKeyRuns : 1][kQ][kLater ? kWave : 1];

  const PagedCache& c = a.cache;
  const int lane = lane_id();
  const int n = lane & 15;
  const int g = lane >> 4;
  const int wave = uniform_i32(wave_in_block());
  // the heads of a share follow one another: they share its pages
  const int units = c.heads * a.head_tiles;
  const int share_index = static_cast<int>(blockIdx.x / static_cast<unsigned>(units));
  const int unit = static_cast<int>(blockIdx.x) - share_index * units;
  const int h = unit / a.head_tiles;
  const int tile_of_heads = unit - h * a.head_tiles;
  const int heads_q = c.heads * a.group;
  const int head0 = h * a.group + tile_of_heads * kHeads;
  const int heads_here = a.group - tile_of_heads * kHeads < kHeads ? a.group - tile_of_heads * kHeads : kHeads;

  if (a.table != nullptr) {
    stage_borders(border, map);
    for (int i = threadIdx.x; i < map.side * kHeads; i += kBlock) {
      const int hh = i % kHeads < heads_here ? i % kHeads : 0;
      bias[i / kHeads][i % kHeads] =
          Elem<T>::at(static_cast<const T*>(a.table), static_cast<int64_t>(i / kHeads) * heads_q + head0 + hh);
    }
  }
  Share share{0, 1, 1, 0, share_index};
  if (a.shares > 0) {
    share = share_of(a, share_index, share_sums);
    if (share.first >= share.end) return;
  } else if (a.table != nullptr) {
    __syncthreads();
  }

  const C* key_base = static_cast<const C*>(c.key.data) + h * c.key.stride[1];
  const C* value_base = static_cast<const C*>(c.value.data) + h * c.value.stride[1];
  const int64_t key_step = c.key.stride[2];
  const int64_t value_step = c.value.stride[2];
  // tokens of this lane: the first of those it loads keys of (the other is 4 further), and of those it weighs
  const int key_token = kF32 ? n : (n >> 2) * 8 + (n & 3);
  const int own_token = g * kOwn;
  int value_at[kBlocks];
#pragma unroll
  for (int j = 0; j < kBlocks; ++j) value_at[j] = run_start((j * 16 + n) * kRun, kRun, c.value.width);

  int64_t at = share.at;
  for (int b = uniform_i32(share.b); b < c.sequences && at < share.end; ++b) {
    const PageList list = page_list(c, b);
    const Seen seen = seen_tokens(a, b, list);
    const int pieces = a.shares > 0 ? piece_count(a, seen) : 1;
    // pieces from .. to - 1 of this sequence are in the share
    const int from_piece = share.first > at ? static_cast<int>(share.first - at) : 0;
    const int to_piece = share.end < at + pieces ? static_cast<int>(share.end - at) : pieces;
    const bool whole = from_piece == 0 && to_piece == pieces;
    const int64_t part = static_cast<int64_t>(share_index) + b;
    if (a.shares > 0 && unit == 0 && from_piece == 0 && threadIdx.x == 0)
      a.plan[b] = make_int2(static_cast<int>(part),
                            static_cast<int>((at + pieces - 1) / share.size - at / share.size) + 1);
    at += pieces;
    const int origin = first_token(a, seen);
    const int base = origin + from_piece * kPiece;
    const int begin = base > seen.begin ? base : seen.begin;
    const int stop = a.shares > 0 ? origin + to_piece * kPiece : seen.end;
    const int end = stop < seen.end ? stop : seen.end;
    const int64_t* pages = c.page_idx + list.begin;

    // where the lane's runs of a key begin (lane (n, g): dimensions (j*4 + g) * kKeyRun ..), the queries there
    // as operand B
    int key_at[kKeyRuns];
    // (in LDS with rows beyond 128: all waves hold the same)
    u32x4 q_own[kLater ? 1 : kKeyRuns][kQ];
    const auto q_of = [&](int j, int p) { return kLater ? q_shared[j][p][lane] : q_own[kLater ? 0 : j][p]; };
    {
      const int head = n < heads_here ? n : 0;
      const T* q_row = static_cast<const T*>(a.query) + b * a.query_stride[0] + (head0 + head) * a.query_stride[1];
#pragma unroll
      for (int j = 0; j < kKeyRuns; ++j) {
        const int d = (j * 4 + g) * kKeyRun;
        key_at[j] = run_start(d, kKeyRun, c.key.width);
        const RawVec<kKeyRun * sizeof(T)> raw = load_run<T, kKeyRun, MODE>(q_row, key_at[j], c.key.width);
        float q[kKeyRun];
#pragma unroll
        for (int i = 0; i < kKeyRun; ++i) {
          const bool mine = key_at[j] + i >= d && key_at[j] + i < c.key.width;
          q[i] = mine && n < heads_here ? Elem<T>::get(raw.w, i) : 0.0f;
        }
#pragma unroll
        for (int p = 0; p < kQ; ++p) {
          u32x4 words;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (kF32) {
              words[i] = __float_as_uint(q[i]);
            } else {
              words[i] = U::pack(q[(2 * i) % kKeyRun], q[(2 * i + 1) % kKeyRun]);
              // what the next part holds; nothing is left of an infinite number
              const f32x2 held = U::unpack(words[i]);
              q[(2 * i) % kKeyRun] = finite(held[0]) ? q[(2 * i) % kKeyRun] - held[0] : 0.0f;
              q[(2 * i + 1) % kKeyRun] = finite(held[1]) ? q[(2 * i + 1) % kKeyRun] - held[1] : 0.0f;
            }
          }
          if constexpr (!kLater) {
            q_own[j][p] = words;
          } else if (wave == 0) {
            q_shared[j][p][lane] = words;
          }
        }
      }
      if constexpr (kLater) __syncthreads();
    }
    f32x4 acc[kValues];
    float top;  // of head n, the same in its four lanes
    float sum;  // of head n and the tokens of this lane

    // What a tile needs from memory.
    struct Tile {
      RawVec<kKeyRun * sizeof(C)> key[kKeyRows][kKeyRuns];
      RawVec<kRun * sizeof(C)> value[kLater ? 1 : kOwn];
      const C* value_row[kLater && MODE != kBlocks8 ? kOwn : 1];  // where they are, for later
      RawVec<8> key_e, value_e;                        // exponents of the tokens this lane weighs, a byte each
      uint32_t bad_tokens;                             // tokens whose page is outside the cache, a bit each
    };
    const auto is_bad = [&](int64_t id) { return id < 0 || id >= c.pages; };
    const auto load_rows = [&](Tile& tile, int s, const C* key_row) {
#pragma unroll
      for (int j = 0; j < kKeyRuns; ++j) tile.key[s][j] = load_run<C, kKeyRun, MODE>(key_row, key_at[j], c.key.width);
    };
    // The page ids of what a lane loads keys of and weighs in a tile: of two blocks
    // with kBlocks8 (asked for a tile ahead), where a block behind what is seen
    // stands for its last one, else of every token, where the last token does.
    const int last = (end - 1) & ~7;
    const auto key_block = [&](int t0) {
      const int t = (t0 + key_token) & ~7;
      return t < last ? t : last;
    };
    const auto own_block = [&](int t0) {
      const int t = (t0 + own_token) & ~7;
      return t < last ? t : last;
    };
    constexpr bool kIdsAhead = MODE == kBlocks8;
    struct Ids {
      int64_t key[MODE == kBlocks8 ? 1 : kKeyRows];
      int64_t own[MODE == kBlocks8 ? 1 : kOwn];
    };
    const auto seen_token = [&](int t) { return t < end ? t : end - 1; };
    const auto ids_of = [&](int t0) {
      Ids ids;
      if constexpr (MODE == kBlocks8) {
        ids.key[0] = pages[page_of_token(a, key_block(t0))];
        ids.own[0] = pages[page_of_token(a, own_block(t0))];
      } else {
#pragma unroll
        for (int s = 0; s < kKeyRows; ++s) ids.key[s] = pages[page_of_token(a, seen_token(t0 + key_token + s * 4))];
#pragma unroll
        for (int e = 0; e < kOwn; ++e) ids.own[e] = pages[page_of_token(a, seen_token(t0 + own_token + e))];
      }
      return ids;
    };
    const auto load_tile = [&](Tile& tile, int t0, const Ids& ids) {
      if constexpr (MODE == kBlocks8) {
        int t = key_block(t0);
        int slot = t - page_of_token(a, t) * c.page_size + (key_token & 7);
        int64_t page = is_bad(ids.key[0]) ? 0 : ids.key[0];
        const C* row = key_base + page * c.key.stride[0] + slot * key_step;
#pragma unroll
        for (int s = 0; s < kKeyRows; ++s) load_rows(tile, s, row + s * 4 * key_step);
        t = own_block(t0);
        slot = t - page_of_token(a, t) * c.page_size + (own_token & 7);
        const bool bad = is_bad(ids.own[0]);
        page = bad ? 0 : ids.own[0];
        tile.bad_tokens = bad ? 0xffu : 0u;
        row = value_base + page * c.value.stride[0] + slot * value_step;
#pragma unroll
        for (int e = 0; e < (kLater ? 0 : kOwn); ++e)
          tile.value[e] = load_run<C, kRun, MODE>(row + e * value_step, value_at[0], c.value.width);
        tile.value_row[0] = row;
        if constexpr (kCoded) {
          __builtin_memcpy(&tile.key_e, c.key.exponents + page * c.key.exponent_stride[0] +
                                            h * c.key.exponent_stride[1] + slot, 8);
          __builtin_memcpy(&tile.value_e, c.value.exponents + page * c.value.exponent_stride[0] +
                                              h * c.value.exponent_stride[1] + slot, 8);
        }
      } else {
        const auto slot_of = [&](int t) {
          t = seen_token(t);
          return t - page_of_token(a, t) * c.page_size;
        };
#pragma unroll
        for (int s = 0; s < kKeyRows; ++s) {
          const int64_t page = is_bad(ids.key[s]) ? 0 : ids.key[s];
          load_rows(tile, s, key_base + page * c.key.stride[0] + slot_of(t0 + key_token + s * 4) * key_step);
        }
        tile.bad_tokens = 0;
        uint32_t key_e[2] = {0u, 0u};
        uint32_t value_e[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
          const bool bad = is_bad(ids.own[e]);
          const int64_t page = bad ? 0 : ids.own[e];
          const int slot = slot_of(t0 + own_token + e);
          if (bad) tile.bad_tokens |= 1u << e;
          const C* row = value_base + page * c.value.stride[0] + slot * value_step;
          if constexpr (kLater) {
            tile.value_row[e] = row;
          } else {
            tile.value[e] = load_run<C, kRun, MODE>(row, value_at[0], c.value.width);
          }
          if constexpr (kCoded) {
            key_e[e / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(
                                c.key.exponents[page * c.key.exponent_stride[0] + h * c.key.exponent_stride[1] +
                                                slot * c.key.exponent_stride[2]])) << (8 * (e % 4));
            value_e[e / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(
                                  c.value.exponents[page * c.value.exponent_stride[0] + h * c.value.exponent_stride[1] +
                                                    slot * c.value.exponent_stride[2]])) << (8 * (e % 4));
          }
        }
        tile.key_e.w[0] = key_e[0];
        tile.key_e.w[1] = key_e[1];
        tile.value_e.w[0] = value_e[0];
        tile.value_e.w[1] = value_e[1];
      }
    };

    // Infinite numbers: a repeated element of a key times zero, or an infinite value
    // times a part of its weight that is zero, would be NaN where the result is
    // infinite.  A wave that ends with NaN runs again without the former, with the
    // parts of the weights for finite values and one for the others.  (8-bit numbers
    // have no infinities.)
    bool careful = false;
    const auto work_on = [&](const Tile& tile, int t0) {
      f32x4 score[kKeyRows];
#pragma unroll
      for (int s = 0; s < kKeyRows; ++s) {
        score[s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kKeyRuns; ++j) {
          if constexpr (kF32) {
            const u32x4 q = q_of(j, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t w = tile.key[s][j].w[i];
              if (careful && key_at[j] + i < (j * 4 + g) * kKeyRun) w = 0u;
              score[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w), __uint_as_float(q[i]), score[s], 0, 0, 0);
            }
          } else {
            uint32_t w[4];
            to_words<C, 8>(tile.key[s][j], w);
            if (!kCoded && careful) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int repeated = (j * 4 + g) * kKeyRun - key_at[j] - 2 * i;
                w[i] = repeated <= 0 ? w[i] : (repeated == 1 ? w[i] & 0xffff0000u : 0u);
              }
            }
#pragma unroll
            for (int p = 0; p < kQ; ++p) score[s] = U::multiply(u32x4{w[0], w[1], w[2], w[3]}, q_of(j, p), score[s]);
          }
        }
      }

      RawVec<kRun * sizeof(C)> value[kBlocks][kOwn];
      const auto load_values = [&](int jb) {
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
          const C* row = MODE == kBlocks8 ? tile.value_row[0] + e * value_step
                                          : tile.value_row[kLater && MODE != kBlocks8 ? e : 0];
          value[jb][e] = load_run<C, kRun, MODE>(row, value_at[jb], c.value.width);
        }
      };
      if constexpr (kLater) {
        load_values(0);
      } else {
#pragma unroll
        for (int e = 0; e < kOwn; ++e) value[0][e] = tile.value[e];
      }

      float scores[kOwn];
      float most = -INFINITY;
#pragma unroll
      for (int e = 0; e < kOwn; ++e) {
        scores[e] = score[e / 4][e % 4] * a.scale;
        if constexpr (kCoded) scores[e] = ldexpf(scores[e], static_cast<int8_t>(tile.key_e.w[e / 4] >> (8 * (e % 4))));
      }
      if (a.table != nullptr) {
        // every token of the tile farther than the last border: one number a head
        if (seen.end - t0 - kTile >= border[map.side - 1]) {
          const float far = bias[map.side - 1][n];
#pragma unroll
          for (int e = 0; e < kOwn; ++e) scores[e] += far;
        } else {
#pragma unroll
          for (int e = 0; e < kOwn; ++e) {
            const int away = seen.end - 1 - (t0 + own_token + e);
            scores[e] += bias[bucket_of_distance(border, map, away < 0 ? 0 : away)][n];
          }
        }
      }
      const bool edge = t0 < begin || t0 + kTile > end;
      if (edge || __any(tile.bad_tokens != 0)) {
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
          const int t = t0 + own_token + e;
          const bool out_of_sight = t < begin || t >= end;
          if ((tile.bad_tokens >> e) & 1) scores[e] = NAN;
          if (out_of_sight) scores[e] = -INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < kOwn; ++e) most = fmaxf(most, scores[e]);

      if (__any(most > top + kSlack)) {
        most = fmaxf(most, __shfl_xor(most, 16, 64));
        most = fmaxf(most, __shfl_xor(most, 32, 64));
        // each head decides for itself, so that its result does not depend on the others'
        const float next = most > top + kSlack ? most : top;
        const float keep = top == -INFINITY ? 0.0f : exp_of(top - next);
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
      const float from = top == -INFINITY ? 0.0f : top;
      float weight[kOwn];
#pragma unroll
      for (int e = 0; e < kOwn; ++e) {
        weight[e] = __builtin_amdgcn_exp2f(fmaf(scores[e] - from, kLog2e, U::kShift));
        sum += weight[e];
        if constexpr (kCoded) weight[e] = ldexpf(weight[e], static_cast<int8_t>(tile.value_e.w[e / 4] >> (8 * (e % 4))));
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
        if (jb + 1 < kBlocks) load_values(jb + 1);
        if (edge) {
          // a value out of sight may be anything; its weight is zero, and so has to be the product
#pragma unroll
          for (int e = 0; e < kOwn; ++e) {
            const int t = t0 + own_token + e;
#pragma unroll
            for (uint32_t& w : value[jb][e].w) w = t < begin || t >= end ? 0u : w;
          }
        }
        if constexpr (kF32) {
#pragma unroll
          for (int e = 0; e < kOwn; ++e) {
#pragma unroll
            for (int j = 0; j < kRun; ++j)
              acc[jb * kRun + j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  weight[e], __uint_as_float(value[jb][e].w[j]), acc[jb * kRun + j], 0, 0, 0);
          }
        } else {
          uint32_t words[8][kRun / 2];
#pragma unroll
          for (int e = 0; e < 8; ++e) to_words<C, kRun>(value[jb][e % kOwn], words[e]);
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
    };

    constexpr int kStride = kWavesPerBlock * kTile;
    for (;; careful = true) {
#pragma unroll
      for (int j = 0; j < kValues; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      top = -INFINITY;
      sum = 0.0f;
      int t0 = base + wave * kTile;
      Ids ids{};
      if (kIdsAhead && t0 < end) ids = ids_of(t0);
      for (; t0 < end; t0 += kStride) {
        // the queries in LDS are read for every tile: kept, they would take the registers they are spared
        if constexpr (kLater) asm volatile("" ::: "memory");
        Tile tile;
        if constexpr (!kIdsAhead) ids = ids_of(t0);
        load_tile(tile, t0, ids);
        if constexpr (kIdsAhead) ids = ids_of(t0 + kStride);
        work_on(tile, t0);
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
      float most = wave_top[0][hh];
#pragma unroll
      for (int w = 1; w < kWavesPerBlock; ++w) most = fmaxf(most, wave_top[w][hh]);
      const float mine = wave_top[wave][hh];
      const float f = mine == -INFINITY ? 0.0f : exp_of(mine - most);
#pragma unroll
      for (int j = 0; j < kValues; ++j) acc[j][i] *= f;
    }
    const auto each_out = [&](auto&& f) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int hh = g * 4 + i;
#pragma unroll
        for (int j = 0; j < kValues; ++j) {
          const int d = value_at[j / kRun] + j % kRun;
          if (hh < heads_here && (MODE != kNarrow || d < c.value.width)) acc[j][i] = f(wave_out[wave % kOutWaves][hh][d], acc[j][i]);
        }
      }
    };
    const auto put = [](float& to, float x) { return to = x; };
    if constexpr (kLater) {
      // two waves hand their sums to the other two; lanes that hold the same column
      // read it before either writes
      if (wave >= kOutWaves) each_out(put);
      __syncthreads();
      if (wave < kOutWaves) each_out([](float& to, float x) { return x + to; });
      __syncthreads();
      if (wave < kOutWaves) each_out(put);
    } else {
      each_out(put);
    }
    __syncthreads();
    const int width = c.value.width;
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
        total += (mine == -INFINITY ? 0.0f : exp_of(mine - most)) * wave_sum[w][hh];
        if (w < kOutWaves) x += wave_out[w % kOutWaves][hh][d];
      }
      if (whole) {
        const int64_t row = static_cast<int64_t>(b) * heads_q + head0 + hh;
        const bool none = total == 0.0f;
        static_cast<T*>(a.out)[row * width + d] = rounded<T>(seen.bad ? NAN : (none ? 0.0f : x / total));
        if (a.lse != nullptr && d == 0)
          a.lse[row] = seen.bad ? NAN : (none ? -INFINITY : fmaf(__builtin_amdgcn_logf(total) - U::kShift, kLn2, most));
      } else {
        const int64_t row = part * heads_q + head0 + hh;
        a.part_out[row * width + d] = x;
        if (d == 0) a.part_sum[row] = make_float2(most, total);
      }
    }
    __syncthreads();  // the next part's results go where these were
  }
}

// Joins the parts of a sequence and query head: TEAM waves for each (one where
// there are many; 2,048 rows of two parts: 6 us, 10 with eight).  Every wave
// finds the maximum and the sum of all parts, lane l those with index l mod 64;
// then the waves of a team take turns with the parts, four at once, and the lanes
// hold the width.
constexpr int kJoinWaves = 8;
constexpr int kJoinAhead = 4;
template <typename T, int TEAM>
__global__ __launch_bounds__(kJoinWaves* kWave) void paged_attention_join_kernel(AttentionArgs a, float shift) {
  __shared__ float wave_out[TEAM][kMaxWidth];
  const PagedCache& c = a.cache;
  const int heads_q = c.heads * a.group;
  const int lane = lane_id();
  const int wave = uniform_i32(wave_in_block()) % TEAM;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kJoinWaves / TEAM) + uniform_i32(wave_in_block()) / TEAM;
  if (row >= static_cast<int64_t>(c.sequences) * heads_q) return;
  const int b = static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(heads_q));
  const int hq = static_cast<int>(row) - b * heads_q;
  const int64_t first = a.plan[b].x;
  const int count = a.plan[b].y;
  if (count <= 1) return;
  const int width = c.value.width;
  const float2* const sums = a.part_sum + first * heads_q + hq;
  const float* const rows = a.part_out + (first * heads_q + hq) * width;
  float top = -INFINITY;
  float sum = 0.0f;
  for (int k = lane; k < count; k += kWave) {
    const float2 part = sums[static_cast<int64_t>(k) * heads_q];
    const float next = fmaxf(top, part.x);
    const float base = next == -INFINITY ? 0.0f : next;
    sum = sum * exp_of(top - base) + part.y * exp_of(part.x - base);
    top = next;
  }
  const float most = wave_max_f32(top);
  const float base = most == -INFINITY ? 0.0f : most;
  const float total = wave_sum_f32(sum * exp_of(top - base));

  constexpr int kParts = kMaxWidth / kWave;
  float acc[kParts];
#pragma unroll
  for (int i = 0; i < kParts; ++i) acc[i] = 0.0f;
  for (int k0 = wave; k0 < count; k0 += TEAM * kJoinAhead) {
    float f[kJoinAhead];
    float x[kJoinAhead][kParts];
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
      const int k = k0 + u * TEAM;
      const int64_t at = static_cast<int64_t>(k < count ? k : count - 1) * heads_q;
      f[u] = k < count ? exp_of(sums[at].x - base) : 0.0f;
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        const int d = lane + i * kWave;
        x[u][i] = k < count && d < width ? rows[at * width + d] : 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < kJoinAhead; ++u) {
#pragma unroll
      for (int i = 0; i < kParts; ++i) acc[i] = fmaf(f[u], x[u][i], acc[i]);
    }
  }
  const bool none = total == 0.0f;
  T* const out = static_cast<T*>(a.out) + row * width;
  if constexpr (TEAM == 1) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int d = lane + i * kWave;
      if (d < width) out[d] = rounded<T>(none ? 0.0f : acc[i] / total);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kParts; ++i) wave_out[wave][lane + i * kWave] = acc[i];
    __syncthreads();
    const int d = threadIdx.x;
    if (d < width) {
      float x = 0.0f;
#pragma unroll
      for (int w = 0; w < TEAM; ++w) x += wave_out[w][d];
      out[d] = rounded<T>(none ? 0.0f : x / total);
    }
  }
  if (a.lse != nullptr && wave == 0 && lane == 0)
    a.lse[row] = none ? -INFINITY : fmaf(__builtin_amdgcn_logf(total) - shift, kLn2, most);
}

// ---- launch --------------------------------------------------------------------------

// Sequences of at most this many tokens have a workgroup each, and no second launch
// (8 key heads of 128 for 32, bf16, one launch and two: one sequence of 256 tokens 9.7
// and 12.8 us, of 512 12.0 and 12.9, of 1,024 16.7 and 13.0; 8 of 512 12.2 and 13.1, of
// 1,024 18.2 and 16.8; 64 of 512 26 and 30, of 1,024 46 and 49).
constexpr int64_t kSingle = 512;

// Shares: two workgroups a CU in one round (64 sequences of 4,096 tokens, 8 key
// heads, bf16: 5.5 TB/s; 5.1 in three rounds), also where sequences are many and
// short: 1,000 of 50 to 700 tokens 331 us, 375 with eight times the shares; 20,000
// of up to 520, one key head, 468 and 899; 2,000 of up to 9 197 and 231.
// (4-bit pages: three workgroups of some kernels.)  dtype: of the queries, < 0 where it is not known yet.
int64_t share_count(const as_paged_cache* c, const PagedCache& laid_out, int64_t group, int64_t window,
                    int64_t max_length, int dtype) {
  const int64_t units = c->heads * ((group + kHeads - 1) / kHeads);
  // tokens of one sequence at most
  int64_t longest = c->page_idx_len * c->page_size;
  if (max_length >= 0 && max_length < longest) longest = max_length;
  if (window > 0 && window < longest) longest = window;
  if (longest <= kSingle) return 0;
  const int64_t all = c->dtype == AS_DTYPE_E2M1 ? paged_shares_e2m1(laid_out, dtype) : 512;
  return all / units < 1 ? 1 : all / units;
}

struct Workspace {
  size_t sums, out, bytes;  // where the parts' sums and results begin behind the plan, and the size of all
};
Workspace workspace_of(const as_paged_cache* c, int64_t group, int64_t shares) {
  if (shares == 0) return Workspace{0, 0, 0};
  const size_t rows = static_cast<size_t>(shares + c->sequences) * c->heads * group;
  Workspace w;
  w.sums = align_up(static_cast<size_t>(c->sequences) * sizeof(int2), 256);
  w.out = w.sums + align_up(rows * sizeof(float2), 256);
  w.bytes = w.out + rows * c->value_width * sizeof(float);
  return w;
}

template <typename T, typename C, int W>
void launch_width(const AttentionArgs& a, const PositionMap& map, dim3 grid, hipStream_t s) {
  const PagedCache& c = a.cache;
  const bool neighbours = sizeof(C) > 1 || (c.key.exponent_stride[2] == 1 && c.value.exponent_stride[2] == 1);
  if (c.key.width < 8 || c.value.width < 8) {
    paged_attention_kernel<T, C, W, kNarrow><<<grid, kBlock, 0, s>>>(a, map);
  } else if (c.page_size % 8 == 0 && neighbours) {
    paged_attention_kernel<T, C, W, kBlocks8><<<grid, kBlock, 0, s>>>(a, map);
  } else {
    paged_attention_kernel<T, C, W, kTokens><<<grid, kBlock, 0, s>>>(a, map);
  }
}

template <typename T, typename C>
int launch_attention(const AttentionArgs& a, const PositionMap& map, hipStream_t s) {
  const int width = a.cache.key.width > a.cache.value.width ? a.cache.key.width : a.cache.value.width;
  const dim3 grid(static_cast<unsigned>((a.shares > 0 ? a.shares : a.cache.sequences) * a.cache.heads * a.head_tiles));
  // the narrowest rows that hold both widths: what a row does not fill is loaded and
  // multiplied all the same (width 160 in float32, 20 sequences to 4,000: 69 us in
  // rows of 192, 82 in rows of 256; width 144 in 8 bits 31 and 36)
  if (width <= 64) {
    launch_width<T, C, 64>(a, map, grid, s);
  } else if (width <= 128) {
    launch_width<T, C, 128>(a, map, grid, s);
  } else if (width <= 192) {
    launch_width<T, C, 192>(a, map, grid, s);
  } else {
    launch_width<T, C, 256>(a, map, grid, s);
  }
  return check_launch("paged_attention");
}

template <typename T>
int launch_join(const AttentionArgs& a, float shift, hipStream_t s) {
  const int64_t rows = int64_t(a.cache.sequences) * a.cache.heads * a.group;
  if (rows >= 1024) {
    paged_attention_join_kernel<T, 1>
        <<<dim3(static_cast<unsigned>((rows + kJoinWaves - 1) / kJoinWaves)), kJoinWaves * kWave, 0, s>>>(a, shift);
  } else {
    paged_attention_join_kernel<T, kJoinWaves>
        <<<dim3(static_cast<unsigned>(rows)), kJoinWaves * kWave, 0, s>>>(a, shift);
  }
  return check_launch("paged_attention (join)");
}

}  // namespace

}  // namespace as

using namespace as;

extern "C" {

size_t as_paged_attention_workspace_bytes(const as_paged_cache* cache, int64_t group, int64_t window,
                                          int64_t max_length) {
  PagedCache c;
  if (read_paged_cache(cache, &c) != AS_OK || group < 1 || group > 65535 / c.heads) return 0;
  return workspace_of(cache, group, share_count(cache, c, group, window, max_length, -1)).bytes;
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
  if (!is_coded(cache->dtype) && cache->dtype != dtype)
    return fail(AS_ERR_INVALID_ARGUMENT, "a cache that is not quantised holds the type of the queries");
  if (group < 1 || group > 65535 / a.cache.heads)
    return fail(AS_ERR_INVALID_ARGUMENT, "query heads must lie in [1, 65535]");
  if (window < 0 || max_length < -1) return fail(AS_ERR_INVALID_ARGUMENT, "window and max_length must be positive");
  PositionMap map{};
  if (table != nullptr) {
    if (const int bad = fill_position_map(&map, borders, buckets, both_sides)) return bad;
  }
  const int64_t shares = share_count(cache, a.cache, group, window, max_length, dtype);
  const Workspace parts = workspace_of(cache, group, shares);
  if (workspace_bytes < parts.bytes || (parts.bytes > 0 && workspace == nullptr))
    return fail(AS_ERR_WORKSPACE, "paged attention needs %zu workspace bytes", parts.bytes);
  if (!aligned(workspace, 16)) return fail(AS_ERR_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
  if (a.cache.sequences == 0) return AS_OK;
  if (a.cache.sequences > 65535 || group * a.cache.heads * a.cache.sequences > kMaxBlocksPerLaunch)
    return fail(AS_ERR_UNSUPPORTED, "at most 65535 sequences, and 2^22 query heads of all sequences");
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
  a.shares = static_cast<int>(shares);
  char* const ws = static_cast<char*>(workspace);
  a.plan = reinterpret_cast<int2*>(ws);
  a.part_sum = reinterpret_cast<float2*>(ws + parts.sums);
  a.part_out = reinterpret_cast<float*>(ws + parts.out);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_float_element(dtype, [&](auto e) {
    using T = decltype(e);
    const bool coded = is_coded(cache->dtype);
    const int bad = cache->dtype == AS_DTYPE_E2M1 ? launch_paged_attention_e2m1(a, map, dtype, s)
                    : coded                       ? launch_attention<T, E4m3>(a, map, s)
                                                  : launch_attention<T, T>(a, map, s);
    if (bad != AS_OK || a.shares == 0) return bad;
    return launch_join<T>(a, coded ? Unit<T, E4m3>::type::kShift : Unit<T, T>::type::kShift, s);
  });
}

}  // extern "C"
