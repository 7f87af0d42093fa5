// What the kernels of paged attention share: their arguments, which tokens of a
// sequence are seen, and how the work is dealt out to the workgroups.
#pragma once

#include "paged_common.h"
#include "position_map.h"

namespace as {

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
  int shares;         // workgroups of each 16 heads of a key head; 0: one per sequence
  int2* plan;         // [sequences] of each sequence: its first part's number, and how many it has
  float2* part_sum;   // [parts, heads * group] maximum and sum
  float* part_out;    // [parts, heads * group, value width]
};

// Pages of 4-bit numbers (paged_attention4.hip).  dtype: of the queries.  Workgroups in
// one round (dtype < 0: of those queries that have the most); attention without the
// join of the parts that its shares leave.
int64_t paged_shares_e2m1(const PagedCache& c, int dtype);
int launch_paged_attention_e2m1(const AttentionArgs& a, const PositionMap& map, int dtype, hipStream_t s);

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kHeads = 16;  // query heads of one workgroup

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

constexpr int kPiece = 32;  // tokens; what is dealt out
constexpr int kMinShare = 4;  // pieces of a share at least, one for each wave

// The first token of a sequence's pieces: the 8-aligned start of what is seen (the
// start itself where pages are no multiple of 8 tokens).
__device__ __forceinline__ int first_token(const AttentionArgs& a, const Seen& seen) {
  return a.cache.page_size % 8 == 0 ? seen.begin & ~7 : seen.begin;
}
// Every sequence has a piece, so that one without tokens is visited too.
__device__ __forceinline__ int piece_count(const AttentionArgs& a, const Seen& seen) {
  const int n = seen.end - first_token(a, seen);
  return n <= kPiece ? 1 : (n + kPiece - 1) / kPiece;
}
__device__ __forceinline__ int piece_count(const AttentionArgs& a, int b) {
  const PageList list = page_list(a.cache, b);
  return piece_count(a, seen_tokens(a, b, list));
}

__device__ __forceinline__ int64_t wave_incl_scan_i64(int64_t v) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int64_t t = __shfl_up(v, o, kWave);
    if (lane_id() >= o) v += t;
  }
  return v;
}

// A workgroup's share: pieces first .. end - 1 of all, `size` of them in every
// share but the last; sequence b holds the first one and begins at piece `at`.
struct Share {
  int64_t first, end, size;
  int64_t at;
  int b;
};
// By the whole workgroup: thread t sums the pieces of `each` sequences from t * each
// on; then the sequences of the thread that holds `first` are gone through, 64 at
// a time.  Leaves the workgroup synchronised.
struct ShareSums {
  int64_t wave[kWavesPerBlock];
  int64_t at;
  int b;
};
__device__ __forceinline__ Share share_of(const AttentionArgs& a, int i, ShareSums& sums) {
  const int n = a.cache.sequences;
  const int each = (n + kBlock - 1) / kBlock;
  const int from = threadIdx.x * each;
  int64_t mine = 0;
#pragma unroll 4
  for (int j = 0; j < each; ++j) {
    if (from + j < n) mine += piece_count(a, from + j);
  }
  int64_t before = wave_incl_scan_i64(mine) - mine;
  if (lane_id() == kWave - 1) sums.wave[wave_in_block()] = before + mine;
  __syncthreads();
  int64_t all = 0;
#pragma unroll
  for (int w = 0; w < kWavesPerBlock; ++w) {
    if (w < wave_in_block()) before += sums.wave[w];
    all += sums.wave[w];
  }
  Share s;
  s.size = (all + a.shares - 1) / a.shares;
  s.size = s.size < kMinShare ? kMinShare : s.size;
  s.first = s.size * i;
  s.end = s.first + s.size < all ? s.first + s.size : all;
  if (before <= s.first && s.first < before + mine) {
    sums.at = before;
    sums.b = from;
  }
  __syncthreads();
  s.at = sums.at;
  s.b = sums.b;
  for (int b0 = s.b; each > 1 && s.first < all; b0 += kWave) {
    const int b = b0 + lane_id();
    const int64_t own = b < n ? piece_count(a, b) : 0;
    const int64_t upto = s.at + wave_incl_scan_i64(own);
    if (__shfl(upto, kWave - 1, kWave) > s.first || b0 + kWave >= n) {
      const int last = 63 - __builtin_clzll(__ballot(b < n && upto - own <= s.first) | 1);
      s.at = __shfl(upto - own, last, kWave);
      s.b = b0 + last;
      break;
    }
    s.at = __shfl(upto, kWave - 1, kWave);
  }
  // the same in every lane
  s.size = uniform_i64(s.size);
  s.first = uniform_i64(s.first);
  s.end = uniform_i64(s.end);
  s.at = uniform_i64(s.at);
  s.b = uniform_i32(s.b);
  return s;
}

}  // namespace
}  // namespace as
