// Attention of one new token of every sequence over pages of 4-bit numbers.
//
// The sums, shares, parts and matrix instructions are those of the other pages
// (paged_attention.hip): the scores of 16 tokens and 16 query heads come out of the
// first product where the second one wants the weights.  What differs is what four
// bits make of the loads and what they take to become operands:
//
//   * a lane reads 16 bytes of a key: 32 neighbouring numbers, which share one
//     exponent.  Products of 32 run over any order of a row's numbers, as long as the
//     queries have it too; so the lanes of a token (g = lane / 16) take runs
//     (j*4 + g) of 32 (16 where a row of 64 or 192 has no more for each), and step i of
//     a run is its numbers 8i .. 8i+7.
//   * a lane holds the columns 8n .. 8n+7 (n = lane % 16) of the values of 8 tokens, 4
//     bytes of each.  They are brought to bf16 and turned 8 x 8 by byte permutes.
//   * the conversion to bf16 multiplies with the exponent on the way.  A code times a
//     power of two is a number of bf16, so that neither scores nor weights are scaled
//     afterwards, and an exponent of NaN makes NaN.  Numbers below 2^-126 count as zeros.
//   * queries enter in bf16 parts: one for bf16, two for fp16, three for float32, which
//     hold all of their bits and have one sign; weights in two (2^-18 of a weight), or
//     three for float32.  So a key that is held as 2^128 makes an infinite score, and such
//     a value NaN.
//
// A row of 128 is 68 bytes, half of an 8-bit one, and each of its numbers costs a vector
// instruction or so: what bounds the kernel is how many loads are on the way while they
// run.  Hence the next tile of a wave is asked for before this one is worked on, its rows
// taking over the registers of this one's as they are used up, and the page ids of the
// one after it.
//
// Measured with the join, 8 key heads, 4 query heads each: 64 sequences of 8,192 tokens of
// 128, bf16, 571 MB: 117 us, 4.9 TB/s (5.9 TB/s is what another 8,192 tokens each come in
// at; the rest is launches, first loads and joins); of up to 8,192, 322 MB: 76; rows of 256,
// 4,096 tokens: 109, 5.2 TB/s; of 64, 16,384 tokens: 132 to 136, 4.2 TB/s.  One sequence of
// 17: 5.4 us.
//
// A token's page may be any, its length may end anywhere and its pages may hold
// anything behind it: see the other kernel.

#include "paged_shares.h"

namespace as {

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 multiply(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Two numbers rounded to a word, and what the word holds.
__device__ __forceinline__ uint32_t pack(float x, float y) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2));
}
__device__ __forceinline__ f32x2 unpack(uint32_t w) {
  return f32x2{__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
}
// The same cut to the word's bits (a NaN has its highest bit set after any product, and stays one).
__device__ __forceinline__ uint32_t cut(float x, float y) {
  return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
}
// What is left of x for the next part.  All parts have to make one infinity of a number that is held as 2^128: so they are
// cut, which leaves the rest with x's sign, and where nothing is left, or x is infinite itself, the rest is 2^-40 of the
// first part (a zero only for a zero, and for queries below 2^-86).
constexpr float kLeast = 1.0f / (1024.0f * 1024.0f * 1024.0f * 1024.0f);
__device__ __forceinline__ float next_part(float x, float held, float least) {
  const float rest = x - held;
  return __builtin_islessgreater(rest, 0.0f) ? rest : least;
}
// The numbers 2i and 2i + 1 of a word of codes, times 2^(e - 127) for scale = e << 23; NaN for e = 255.
template <int I>
__device__ __forceinline__ uint32_t bf16_pair(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, I));
}
__device__ __forceinline__ float as_scale(uint32_t e) { return __uint_as_float(e << 23); }

// A running maximum may stay this far below a score: weights are then at most 2^4.
constexpr float kSlack = 4.0f * kLn2;
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// How a call reaches its rows.  kWhole: pages are a multiple of 8 tokens and rows of 32
// numbers, so that the blocks of 8 tokens which a lane works on lie in one page each,
// and no run passes a row's end.  kDense: besides, rows fill the kernel's width and the
// tokens of a head follow one another, so that the rows of a block are constants
// apart.  kTokens: every token is looked up, and the last word
// of a row is read where it ends with the row, and shifted.  kBytes: so it is, and words
// are read a byte at a time, for rows of fewer than 4 bytes.
//
// 64 sequences of up to 8,192 tokens, 8 key heads, bf16.  kDense, rows of 128: 79 us on a floor
// of 64, bound by memory.  kWhole, rows of 96: 99 on 48; addresses that are no constants apart
// and columns that are not there make 28M vector instructions of 23M (46 us of the ALUs), and
// leave registers for two workgroups a CU, not three.  kTokens, rows of 80 in pages of 16: 144
// on 40, of 128 in pages of 12: 152 on 64; ten tokens a lane that are looked up one by one, and
// shifted words, make 50M (82 us) and 2.9M loads of 1.7M (75 us of the address units).  Of the
// two conditions that lead there a block of 8 tokens needs the page's alone: rows that are no
// multiple of 32 in pages of 8 only share the mode.
enum Mode { kDense, kWhole, kTokens, kBytes };
constexpr bool in_blocks(int mode) { return mode == kDense || mode == kWhole; }

// Where a word (or half of one) of a row is read, and how far it is shifted then.
struct Word {
  int at;
  int shift;
};
template <int BYTES, int MODE>
__device__ __forceinline__ Word word_of(int at, int row_bytes) {
  if constexpr (MODE == kDense || MODE == kBytes) return Word{at, 0};
  if (MODE == kWhole || at >= row_bytes) return Word{at < row_bytes ? at : 0, 0};
  const int last = row_bytes - BYTES;
  return Word{at < last ? at : last, at < last ? 0 : 8 * (at - last)};
}
// The same for a byte permute, of a key's words: those behind the row are zeros, for whatever is read in their place may
// stand for an infinite number, which a query's zero makes NaN.  (Nobody asks for such columns of a value.)
struct KeyWord {
  int at;
  uint32_t bytes;  // 0x0c is a zero
};
template <int MODE>
__device__ __forceinline__ KeyWord key_word_of(int at, int row_bytes) {
  constexpr uint32_t kAll = 0x03020100u;
  constexpr uint32_t kNone = 0x0c0c0c0cu;
  const Word w = word_of<4, MODE>(at, row_bytes);
  if (MODE != kTokens) return KeyWord{w.at, kAll};
  return KeyWord{w.at, at < row_bytes ? static_cast<uint32_t>(((uint64_t(kNone) << 32) | kAll) >> w.shift) : kNone};
}
template <int BYTES, int MODE>
__device__ __forceinline__ uint32_t load_word(const uint8_t* __restrict__ row, int at, int row_bytes) {
  if constexpr (MODE == kBytes) {
    uint32_t x = 0u;
#pragma unroll
    for (int i = 0; i < BYTES; ++i) x |= at + i < row_bytes ? uint32_t(row[at + i]) << (8 * i) : 0u;
    return x;
  } else if constexpr (BYTES == 2) {
    uint16_t x;
    __builtin_memcpy(&x, row + at, 2);
    return x;
  } else {
    uint32_t x;
    __builtin_memcpy(&x, row + at, 4);
    return x;
  }
}

template <int I>
struct Constant {
  static constexpr int value = I;
};
// 16 bytes at once, at any address of memory, and at a multiple of 16 in LDS.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1), may_alias));
typedef uint32_t u32x4_16 __attribute__((ext_vector_type(4), aligned(16), may_alias));
__device__ __forceinline__ u32x4 load_16(const uint8_t* p) { return *reinterpret_cast<const u32x4_any*>(p); }
__device__ __forceinline__ void store_16(uint8_t* p, u32x4 x) { *reinterpret_cast<u32x4_16*>(p) = x; }

template <typename T>
constexpr int kQueryParts = sizeof(T) == 4 ? 3 : (__is_same(T, Fp16) ? 2 : 1);
template <typename T>
constexpr int kWeightParts = sizeof(T) == 4 ? 3 : 2;

// Workgroups of a CU: three where rows are dense and a wave needs at most 168 registers (paged_shares_e2m1 deals the
// work out to as many).  64 sequences of up to 8,192 tokens, 8 key heads of 128, bf16: 76 us with three, 80 with two, 90
// with four (which spill); 20 of up to 4,000 in float32 33 and 30, rows of 256 43 and 28.
template <typename T, int W, int MODE>
constexpr int kWavesPerSimd = MODE == kDense && (W == 64 || (W == 128 && sizeof(T) == 2)) ? 3 : (MODE == kBytes ? 1 : 2);

constexpr int kTile = 32;  // tokens of one step of a wave
constexpr int kOwn = 8;    // of which a lane weighs this many

// BIASED: with a table, or without one all the same.
template <typename T, int W, int MODE, bool BIASED>
__global__ __launch_bounds__(kBlock) __attribute__((amdgpu_waves_per_eu(kWavesPerSimd<T, W, MODE>))) void paged_attention_e2m1_kernel(AttentionArgs a, PositionMap map) {
  constexpr int kKeyRun = W % 128 == 0 ? 32 : 16;  // numbers of a key in one load
  constexpr int kKeyRuns = W / (4 * kKeyRun);
  constexpr int kKeyWords = kKeyRun / 8;
  constexpr int kSteps = kKeyRuns * kKeyWords;
  constexpr int kValues = W / 16;  // columns that a lane holds
  constexpr int kRun = kValues % 8 == 0 ? 8 : 4;  // of which neighbours
  constexpr int kBlocks = kValues / kRun;
  constexpr bool kShared = W > 128;  // queries in LDS: rows beyond 128 leave no registers for them
  constexpr int kQ = kQueryParts<T>;
  constexpr int kP = kWeightParts<T>;
  constexpr int kOutWaves = 2;

  __shared__ int32_t border[BIASED ? kMaxBuckets + 1 : 1];
  __shared__ ShareSums share_sums;
  __shared__ float wave_top[kWavesPerBlock][kHeads];
  __shared__ float wave_sum[kWavesPerBlock][kHeads];
  __shared__ float bias[BIASED ? kMaxBuckets : 1][kHeads];  // of the keys in front of the query
  __shared__ float wave_out[kOutWaves][kHeads][W];
  __shared__ u32x4 q_shared[kShared ? kSteps : 1][kQ][kShared ? kWave : 1];
  // kStaged: a wave's tile on its way into registers.  Values of a block of 8 tokens, and a gap so that the four blocks
  // of a read lie in banks of their own; exponents of the keys' tokens, then of the values'.
  constexpr bool kStaged = MODE == kDense && W == 64;
  constexpr int kBlockBytes = 4 * W + 32;
  __shared__ __attribute__((aligned(16))) uint8_t staged_values[kStaged ? kWavesPerBlock : 1][kStaged ? 4 * kBlockBytes : 1];
  __shared__ __attribute__((aligned(16))) uint8_t staged_e[kStaged ? kWavesPerBlock : 1][kStaged ? 2 * W : 1];

  const PagedCache& c = a.cache;
  const int lane = lane_id();
  const int n = lane & 15;
  const int g = lane >> 4;
  const int wave = uniform_i32(wave_in_block());
  // The heads of a share follow one another: they share its pages.  Of two neighbouring heads the exponents of a
  // page may share lines, so they are given to workgroups 8 apart, which the hardware gives to one of its 8 dies.
  const int units = c.heads * a.head_tiles;
  int block = static_cast<int>(blockIdx.x);
  int in_pair = 0;
  const bool paired = units % 2 == 0 && gridDim.x % 16 == 0;
  if (paired) {
    in_pair = (block >> 3) & 1;
    block = ((block >> 4) << 3) + (block & 7);
  }
  const int unit_count = paired ? units / 2 : units;
  const int share_index = static_cast<int>(static_cast<unsigned>(block) / static_cast<unsigned>(unit_count));
  int unit = block - share_index * unit_count;
  if (paired) unit = 2 * unit + in_pair;
  const int h = unit / a.head_tiles;
  const int tile_of_heads = unit - h * a.head_tiles;
  const int heads_q = c.heads * a.group;
  const int head0 = h * a.group + tile_of_heads * kHeads;
  const int heads_here = a.group - tile_of_heads * kHeads < kHeads ? a.group - tile_of_heads * kHeads : kHeads;

  const bool biased = BIASED && a.table != nullptr;
  if (biased) {
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
  } else if (biased) {
    __syncthreads();
  }

  // the queries have the scale's sign, or are multiplied with it where it is zero
  const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale);
  const float q_sign = a.scale == 0.0f ? 0.0f : copysignf(1.0f, a.scale);
  const float left = biased ? 1.0f : scale;  // what scores are still to be multiplied with
  const uint8_t* key_base = static_cast<const uint8_t*>(c.key.data) + h * c.key.stride[1];
  const uint8_t* value_base = static_cast<const uint8_t*>(c.value.data) + h * c.value.stride[1];
  const uint8_t* key_e_base = reinterpret_cast<const uint8_t*>(c.key.exponents) + h * c.key.exponent_stride[1];
  const uint8_t* value_e_base = reinterpret_cast<const uint8_t*>(c.value.exponents) + h * c.value.exponent_stride[1];
  // from a token to the next, and (by the page's number) to a page
  const int64_t key_step = MODE == kDense ? W / 2 : c.key.stride[2];
  const int64_t value_step = MODE == kDense ? W / 2 : c.value.stride[2];
  const int64_t key_e_step = MODE == kDense ? W / kGroup : c.key.exponent_stride[2];
  const int64_t value_e_step = MODE == kDense ? W / kGroup : c.value.exponent_stride[2];
  const auto page_offset = [](int64_t page, int64_t stride) {
    return MODE == kDense ? static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(page)) *
                                                 static_cast<uint32_t>(stride))
                          : page * stride;
  };
  const int key_bytes = c.key.width / 2;
  const int value_bytes = c.value.width / 2;
  // tokens of this lane: the first of those it loads keys of (the other is 4 further), and of those it weighs
  const int key_token = (n >> 2) * 8 + (n & 3);
  const int own_token = g * kOwn;
  // Words of a key and of a value, and their exponents.  A lane behind a row's end reads its beginning: it has zeros on
  // the queries' side (and codes of zero here, or an exponent that leaves them finite), and columns that nobody asks for
  // on the values'.
  KeyWord key_word[in_blocks(MODE) ? kKeyRuns : kSteps];
  int key_e_at[kKeyRuns];
  bool key_there[kKeyRuns];
#pragma unroll
  for (int j = 0; j < kKeyRuns; ++j) {
    const int d = (j * 4 + g) * kKeyRun;
    key_there[j] = d < c.key.width;
    key_e_at[j] = MODE == kDense || d < c.key.width ? d / kGroup : 0;
    if constexpr (in_blocks(MODE)) {
      key_word[j] = key_word_of<MODE>(d / 2, key_bytes);
    } else {
#pragma unroll
      for (int i = 0; i < kKeyWords; ++i) key_word[j * kKeyWords + i] = key_word_of<MODE>(d / 2 + 4 * i, key_bytes);
    }
  }
  Word value_word[kBlocks];
  int value_e_at[kBlocks];
#pragma unroll
  for (int j = 0; j < kBlocks; ++j) {
    const int d = (j * 16 + n) * kRun;
    value_word[j] = word_of<kRun / 2, MODE>(d / 2, value_bytes);
    value_e_at[j] = MODE == kDense || d < c.value.width ? d / kGroup : 0;
  }

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

    // the queries as operand B: step j*kKeyWords + i has the numbers 8i .. of run j
    u32x4 q_own[kShared ? 1 : kSteps][kQ];
    const auto q_of = [&](int j, int p) { return kShared ? q_shared[j][p][lane] : q_own[kShared ? 0 : j][p]; };
    {
      const int head = n < heads_here ? n : 0;
      // not known to be the same for every sequence: the masks of its comparisons would be kept for all of them
      int key_width = c.key.width;
      asm("" : "+s"(key_width));
      const T* q_row = static_cast<const T*>(a.query) + b * a.query_stride[0] + (head0 + head) * a.query_stride[1];
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        const int d0 = (j / kKeyWords * 4 + g) * kKeyRun + j % kKeyWords * 8;
        float q[8];
        if constexpr (MODE == kDense) {
          RawVec<8 * sizeof(T)> raw;
          __builtin_memcpy(&raw, q_row + d0, sizeof(raw));
#pragma unroll
          for (int i = 0; i < 8; ++i) q[i] = n < heads_here ? Elem<T>::get(raw.w, i) * q_sign : 0.0f;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int d = d0 + i;
            const float x = Elem<T>::at(q_row, d < key_width ? d : 0);
            q[i] = d < key_width && n < heads_here ? x * q_sign : 0.0f;
          }
        }
        f32x2 least[4];
#pragma unroll
        for (int p = 0; p < kQ; ++p) {
          u32x4 words;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            words[i] = kQ == 1 ? pack(q[2 * i], q[2 * i + 1]) : cut(q[2 * i], q[2 * i + 1]);
            const f32x2 held = unpack(words[i]);
            if (p == 0) least[i] = f32x2{held[0] * kLeast, held[1] * kLeast};
            q[2 * i] = next_part(q[2 * i], held[0], least[i][0]);
            q[2 * i + 1] = next_part(q[2 * i + 1], held[1], least[i][1]);
          }
          if constexpr (!kShared) {
            q_own[j][p] = words;
          } else if (wave == 0) {
            q_shared[j][p][lane] = words;
          }
        }
      }
      if constexpr (kShared) __syncthreads();
    }
    f32x4 acc[kValues];
    float top;  // of head n, the same in its four lanes
    float sum;  // of head n and the tokens of this lane

    // What a tile needs from memory.
    struct Keys {
      uint32_t codes[2][kSteps];
      uint32_t e[2][kKeyRuns];
    };
    struct Values {
      uint32_t codes[kBlocks][kOwn];
      uint32_t e[kBlocks][kOwn];
      uint32_t bad_tokens;  // tokens whose page is outside the cache, a bit each
    };
    struct Ids {
      int64_t key[in_blocks(MODE) ? 1 : 2];
      int64_t own[in_blocks(MODE) ? 1 : kOwn];
    };
    const auto is_bad = [&](int64_t id) { return id < 0 || id >= c.pages; };
    // Blocks (or tokens) behind what is seen stand for the last one: their loads need no guard.
    const int last = (end - 1) & ~7;
    const auto block_of = [&](int t) { return (t & ~7) < last ? t & ~7 : last; };
    const auto seen_token = [&](int t) { return t < end ? t : end - 1; };
    const auto ids_of = [&](int t0) {
      Ids ids;
      if constexpr (in_blocks(MODE)) {
        ids.key[0] = pages[page_of_token(a, block_of(t0 + key_token))];
        ids.own[0] = pages[page_of_token(a, block_of(t0 + own_token))];
      } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) ids.key[s] = pages[page_of_token(a, seen_token(t0 + key_token + s * 4))];
#pragma unroll
        for (int e = 0; e < kOwn; ++e) ids.own[e] = pages[page_of_token(a, seen_token(t0 + own_token + e))];
      }
      return ids;
    };
    const auto load_key = [&](Keys& keys, int s, const uint8_t* row, const uint8_t* row_e) {
#pragma unroll
      for (int j = 0; j < kKeyRuns; ++j) {
        if constexpr (in_blocks(MODE)) {
          __builtin_memcpy(&keys.codes[s][j * kKeyWords], row + key_word[j].at, 4 * kKeyWords);
        } else {
#pragma unroll
          for (int i = 0; i < kKeyWords; ++i)
            keys.codes[s][j * kKeyWords + i] = load_word<4, MODE>(row, key_word[j * kKeyWords + i].at, key_bytes);
        }
        keys.e[s][j] = row_e[key_e_at[j]];
      }
    };
    const auto load_value = [&](Values& values, int e, const uint8_t* row, const uint8_t* row_e) {
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) {
        const uint32_t x = load_word<kRun / 2, MODE>(row, value_word[j].at, value_bytes);
        values.codes[j][e] = MODE == kTokens ? x >> value_word[j].shift : x;
        values.e[j][e] = row_e[value_e_at[j]];
      }
    };
    const auto slot_of = [&](int t) { return t - page_of_token(a, t) * c.page_size; };
    const auto load_keys = [&](Keys& keys, int t0, const Ids& ids) {
      if constexpr (in_blocks(MODE)) {
        const int slot = slot_of(block_of(t0 + key_token)) + (key_token & 7);
        const int64_t page = is_bad(ids.key[0]) ? 0 : ids.key[0];
        const uint8_t* row = key_base + page_offset(page, c.key.stride[0]) + slot * key_step;
        const uint8_t* row_e = key_e_base + page_offset(page, c.key.exponent_stride[0]) + slot * key_e_step;
#pragma unroll
        for (int s = 0; s < 2; ++s) load_key(keys, s, row + s * 4 * key_step, row_e + s * 4 * key_e_step);
      } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int64_t page = is_bad(ids.key[s]) ? 0 : ids.key[s];
          const int slot = slot_of(seen_token(t0 + key_token + s * 4));
          load_key(keys, s, key_base + page_offset(page, c.key.stride[0]) + slot * key_step,
                   key_e_base + page_offset(page, c.key.exponent_stride[0]) + slot * key_e_step);
        }
      }
    };
    const auto load_values = [&](Values& values, int t0, const Ids& ids) {
      if constexpr (in_blocks(MODE)) {
        const int slot = slot_of(block_of(t0 + own_token));
        const bool bad = is_bad(ids.own[0]);
        const int64_t page = bad ? 0 : ids.own[0];
        values.bad_tokens = bad ? 0xffu : 0u;
        const uint8_t* row = value_base + page_offset(page, c.value.stride[0]) + slot * value_step;
        const uint8_t* row_e = value_e_base + page_offset(page, c.value.exponent_stride[0]) + slot * value_e_step;
#pragma unroll
        for (int e = 0; e < kOwn; ++e) load_value(values, e, row + e * value_step, row_e + e * value_e_step);
      } else {
        values.bad_tokens = 0;
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
          const bool bad = is_bad(ids.own[e]);
          const int64_t page = bad ? 0 : ids.own[e];
          const int slot = slot_of(seen_token(t0 + own_token + e));
          if (bad) values.bad_tokens |= 1u << e;
          load_value(values, e, value_base + page_offset(page, c.value.stride[0]) + slot * value_step,
                     value_e_base + page_offset(page, c.value.exponent_stride[0]) + slot * value_e_step);
        }
      }
    };

    // kStaged: loads of 16 bytes a lane, whose order is the memory's, and the turn to the lanes that use them in LDS
    // (a few loads a tile where a lane that fetches its own takes 22, at 16 cycles of the address unit each).  64
    // sequences of 16,384 tokens, 8 heads of 64: 136 us where direct loads take 152.  Rows of 128 have twice the work
    // for each load: 64 sequences of 8,192 took 119 us both ways, uneven ones 77 against 75, and rows of 256 30 us
    // against 28, so they load directly.  Lane l knows the page of block l % 4.
    struct Staged {
      u32x4 values;
      u32x4 e;
      uint32_t bad_tokens;
    };
    struct BlockId {
      int64_t id;
      int slot;
    };
    const auto block_id = [&](int t0) {
      const int t = block_of(t0 + (lane & 3) * 8);
      const int entry = page_of_token(a, t);
      return BlockId{pages[entry], t - entry * c.page_size};
    };
    // (page, or -1, and slot) of a block
    const auto page_and_slot = [&](const BlockId& b, int block) {
      return make_int2(__shfl(is_bad(b.id) ? -1 : static_cast<int>(b.id), block, kWave), __shfl(b.slot, block, kWave));
    };
    const auto load_staged = [&](Staged& to, const BlockId& b) {
      // the values of a block are 16 times 16 bytes, its exponents are 16 bytes
      const int2 v = page_and_slot(b, lane >> 4);
      to.values = load_16(value_base + page_offset(v.x < 0 ? 0 : v.x, c.value.stride[0]) + v.y * (W / 2) +
                          (lane & 15) * 16);
      const bool second = lane & 4;
      const int2 e = page_and_slot(b, lane & 3);
      to.e = load_16((second ? value_e_base : key_e_base) +
                     page_offset(e.x < 0 ? 0 : e.x, second ? c.value.exponent_stride[0] : c.key.exponent_stride[0]) +
                     e.y * (W / kGroup));
      to.bad_tokens = page_and_slot(b, g).x < 0 ? 0xffu : 0u;
    };
    const auto load_dense_keys = [&](Keys& keys, const BlockId& b) {
      const int2 p = page_and_slot(b, n >> 2);
      const uint8_t* row = key_base + page_offset(p.x < 0 ? 0 : p.x, c.key.stride[0]) + (p.y + (n & 3)) * (W / 2);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int j = 0; j < kKeyRuns; ++j)
          __builtin_memcpy(&keys.codes[s][j * kKeyWords], row + s * 4 * (W / 2) + key_word[j].at, 4 * kKeyWords);
      }
    };
    const auto stage = [&](const Staged& from) {
      store_16(&staged_values[wave][(lane >> 4) * kBlockBytes + (lane & 15) * 16], from.values);
      store_16(&staged_e[wave][(lane & 7) * 16], from.e);  // lanes that have the same write the same
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };
    const auto unstage_keys = [&](Keys& keys) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int j = 0; j < kKeyRuns; ++j)
          keys.e[s][j] = staged_e[wave][(key_token + 4 * s) * (W / kGroup) + key_e_at[j]];
      }
    };
    const auto unstage_values = [&](Values& values) {
#pragma unroll
      for (int e = 0; e < kOwn; ++e) {
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) {
          const uint8_t* from = &staged_values[wave][g * kBlockBytes + e * (W / 2) + (j * 16 + n) * (kRun / 2)];
          values.codes[j][e] = 0u;
          __builtin_memcpy(&values.codes[j][e], from, kRun / 2);
          values.e[j][e] = staged_e[wave][W + (own_token + e) * (W / kGroup) + value_e_at[j]];
        }
      }
    };

    const auto products = [&](const Keys& keys, f32x4 (&score)[2]) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        score[s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          // where it is used: in front of that it would be waited for
          uint32_t w = keys.codes[s][j];
          if constexpr (MODE == kTokens) w = __builtin_amdgcn_perm(0u, w, key_word[j].bytes);
          const uint32_t e = keys.e[s][j / kKeyWords];
          const float scale = as_scale(MODE == kWhole && !key_there[j / kKeyWords] ? 127u : e);
          const u32x4 k{bf16_pair<0>(w, scale), bf16_pair<1>(w, scale), bf16_pair<2>(w, scale), bf16_pair<3>(w, scale)};
#pragma unroll
          for (int p = 0; p < kQ; ++p) score[s] = multiply(k, q_of(j, p), score[s]);
        }
      }
    };
    const auto weigh = [&](Values& values, const f32x4 (&score)[2], int t0) {
      // Scores, and the products that they are scale times of where there is no bias: one fused step less then for
      // each weight, and their maximum is the scores' (scale is not negative, the queries have its sign).
      float scores[kOwn];
      float most = -INFINITY;
#pragma unroll
      for (int e = 0; e < kOwn; ++e) scores[e] = score[e / 4][e % 4];
      if (biased) {
        // every token of the tile farther than the last border: one number a head
        if (seen.end - t0 - kTile >= border[map.side - 1]) {
          const float far = bias[map.side - 1][n];
#pragma unroll
          for (int e = 0; e < kOwn; ++e) scores[e] = fmaf(scores[e], scale, far);
        } else {
#pragma unroll
          for (int e = 0; e < kOwn; ++e) {
            const int away = seen.end - 1 - (t0 + own_token + e);
            scores[e] = fmaf(scores[e], scale, bias[bucket_of_distance(border, map, away < 0 ? 0 : away)][n]);
          }
        }
      }
      if (t0 < begin || t0 + kTile > end || __any(values.bad_tokens != 0)) {
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
          const int t = t0 + own_token + e;
          const bool out_of_sight = t < begin || t >= end;
          if ((values.bad_tokens >> e) & 1) scores[e] = NAN;
          if (out_of_sight) scores[e] = -INFINITY;
          // a value out of sight may be anything; its weight is zero, and so has to be the product
#pragma unroll
          for (int j = 0; j < kBlocks; ++j) {
            values.codes[j][e] = out_of_sight ? 0u : values.codes[j][e];
            values.e[j][e] = out_of_sight ? 127u : values.e[j][e];
          }
        }
      }
#pragma unroll
      for (int e = 0; e < kOwn; ++e) most = fmaxf(most, scores[e]);

      most *= left;
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
        weight[e] = exp_of(fmaf(scores[e], left, -from));
        sum += weight[e];
      }
      u32x4 w16[kP];
#pragma unroll
      for (int p = 0; p < kP; ++p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = pack(weight[2 * i], weight[2 * i + 1]);
          w16[p][i] = w;
          weight[2 * i] -= unpack(w)[0];
          weight[2 * i + 1] -= unpack(w)[1];
        }
      }

#pragma unroll
      for (int jb = 0; jb < kBlocks; ++jb) {
        // two columns at a time, so that few converted numbers are held at once
        const auto columns = [&](auto pair) {
          constexpr int I = decltype(pair)::value;
          uint32_t words[kOwn];
#pragma unroll
          for (int e = 0; e < kOwn; ++e) words[e] = bf16_pair<I>(values.codes[jb][e], as_scale(values.e[jb][e]));
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            u32x4 column;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              column[i] = __builtin_amdgcn_perm(words[2 * i + 1], words[2 * i], j == 0 ? 0x05040100u : 0x07060302u);
            f32x4& to = acc[jb * kRun + 2 * I + j];
#pragma unroll
            for (int p = 0; p < kP; ++p) to = multiply(w16[p], column, to);
          }
          __builtin_amdgcn_sched_barrier(0);
        };
        columns(Constant<0>{});
        columns(Constant<1>{});
        if constexpr (kRun == 8) {
          columns(Constant<2>{});
          columns(Constant<3>{});
        }
      }
    };

    constexpr int kStride = kWavesPerBlock * kTile;
#pragma unroll
    for (int j = 0; j < kValues; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    top = -INFINITY;
    sum = 0.0f;
    int t0 = base + wave * kTile;
    if (t0 < end) {
      // each kind of row takes the registers of the last tile's as soon as those are used up
      Keys keys;
      Values values;
      if constexpr (kStaged) {
        Staged staged;
        BlockId ids = block_id(t0);
        load_dense_keys(keys, ids);
        load_staged(staged, ids);
        ids = block_id(t0 + kStride);
        for (;;) {
          stage(staged);
          values.bad_tokens = staged.bad_tokens;
          load_staged(staged, ids);
          unstage_keys(keys);
          f32x4 score[2];
          products(keys, score);
          __builtin_amdgcn_sched_barrier(0);
          load_dense_keys(keys, ids);
          ids = block_id(t0 + 2 * kStride);
          unstage_values(values);
          weigh(values, score, t0);
          __builtin_amdgcn_sched_barrier(0);
          t0 += kStride;
          if (t0 >= end) break;
        }
      } else {
        Ids ids = ids_of(t0);
        load_keys(keys, t0, ids);
        load_values(values, t0, ids);
        ids = ids_of(t0 + kStride);
        for (;;) {
          // the queries in LDS are read for every tile: kept, they would take the registers they are spared
          if constexpr (kShared) asm volatile("" ::: "memory");
          f32x4 score[2];
          products(keys, score);
          __builtin_amdgcn_sched_barrier(0);
          load_keys(keys, t0 + kStride, ids);
          weigh(values, score, t0);
          __builtin_amdgcn_sched_barrier(0);
          load_values(values, t0 + kStride, ids);
          ids = ids_of(t0 + 2 * kStride);
          t0 += kStride;
          if (t0 >= end) break;
        }
      }
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
#pragma unroll
        for (int j = 0; j < kValues; ++j)
          acc[j][i] = f(wave_out[wave % kOutWaves][g * 4 + i][(j / kRun * 16 + n) * kRun + j % kRun], acc[j][i]);
      }
    };
    // two waves hand their sums to the other two
    const auto put = [](float& to, float x) { return to = x; };
    if (wave >= kOutWaves) each_out(put);
    __syncthreads();
    if (wave < kOutWaves) {
      each_out([](float& to, float x) { return x + to; });
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
#pragma unroll
      for (int w = 0; w < kWavesPerBlock; ++w) {
        const float mine = wave_top[w][hh];
        total += (mine == -INFINITY ? 0.0f : exp_of(mine - most)) * wave_sum[w][hh];
      }
      const float x = wave_out[0][hh][d] + wave_out[1][hh][d];
      if (whole) {
        const int64_t row = static_cast<int64_t>(b) * heads_q + head0 + hh;
        const bool none = total == 0.0f;
        static_cast<T*>(a.out)[row * width + d] = rounded<T>(seen.bad ? NAN : (none ? 0.0f : x / total));
        if (a.lse != nullptr && d == 0)
          a.lse[row] = seen.bad ? NAN : (none ? -INFINITY : fmaf(__builtin_amdgcn_logf(total), kLn2, most));
      } else {
        const int64_t row = part * heads_q + head0 + hh;
        a.part_out[row * width + d] = x;
        if (d == 0) a.part_sum[row] = make_float2(most, total);
      }
    }
    __syncthreads();  // the next part's results go where these were
  }
}

// The narrowest rows that hold both widths: what a row does not fill is loaded and multiplied all the same.
int row_width(const PagedCache& c) {
  const int width = c.key.width > c.value.width ? c.key.width : c.value.width;
  return width <= 64 ? 64 : (width <= 128 ? 128 : (width <= 192 ? 192 : 256));
}
// Whether the rows of a tensor are those of kDense.
bool dense(const PageTensor& t, int width) {
  const auto near = [](int64_t stride) { return stride >= 0 && stride <= INT32_MAX; };
  return t.width == width && t.stride[2] == width / 2 && t.exponent_stride[2] == width / kGroup && near(t.stride[0]) &&
         near(t.exponent_stride[0]);
}
Mode mode_of(const PagedCache& c) {
  if (c.key.width < 8 || c.value.width < 8) return kBytes;
  if (c.page_size % 8 != 0 || c.key.width % kGroup != 0 || c.value.width % kGroup != 0) return kTokens;
  return dense(c.key, row_width(c)) && dense(c.value, row_width(c)) ? kDense : kWhole;
}

template <typename T, int W>
void launch_width(const AttentionArgs& a, const PositionMap& map, dim3 grid, hipStream_t s) {
  switch (mode_of(a.cache)) {
    case kBytes:
      paged_attention_e2m1_kernel<T, W, kBytes, true><<<grid, kBlock, 0, s>>>(a, map);
      break;
    case kTokens:
      paged_attention_e2m1_kernel<T, W, kTokens, true><<<grid, kBlock, 0, s>>>(a, map);
      break;
    case kWhole:
      paged_attention_e2m1_kernel<T, W, kWhole, true><<<grid, kBlock, 0, s>>>(a, map);
      break;
    case kDense:
      if (a.table == nullptr) {
        paged_attention_e2m1_kernel<T, W, kDense, false><<<grid, kBlock, 0, s>>>(a, map);
      } else {
        paged_attention_e2m1_kernel<T, W, kDense, true><<<grid, kBlock, 0, s>>>(a, map);
      }
  }
}

}  // namespace

int64_t paged_shares_e2m1(const PagedCache& c, int dtype) {
  if (mode_of(c) != kDense) return 512;
  const int width = row_width(c);
  return width == 64 || (width == 128 && dtype != AS_DTYPE_F32) ? 768 : 512;
}

int launch_paged_attention_e2m1(const AttentionArgs& a, const PositionMap& map, int dtype, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.shares > 0 ? a.shares : a.cache.sequences) * a.cache.heads * a.head_tiles));
  return with_float_element(dtype, [&](auto e) {
    using T = decltype(e);
    switch (row_width(a.cache)) {
      case 64:
        launch_width<T, 64>(a, map, grid, s);
        break;
      case 128:
        launch_width<T, 128>(a, map, grid, s);
        break;
      case 192:
        launch_width<T, 192>(a, map, grid, s);
        break;
      default:
        launch_width<T, 256>(a, map, grid, s);
    }
    return check_launch("paged_attention");
  });
}

}  // namespace as
