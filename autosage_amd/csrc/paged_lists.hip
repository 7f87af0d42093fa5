// Page lists that grow and shrink with their sequences.
//
// Sequence b has lengths[b] tokens in the pages table[b][0 .. ceil(length / page_size)).
// It gives up its last -change[b] tokens, or gets room for change[b] more; pages come
// from the top of a stack of free ones and go back there.
//
// With D pages given back in all (sequences ascending, pages of a sequence ascending),
// number k of them goes to free[count + D - 1 - k]; then number k of the pages that
// are taken, in the same order, is free[count + D - 1 - k].  So a drop undoes a
// growth, bit for bit.  Sequences are served in order while the stack holds the sum of
// what they need; one that needs more than is left, or than its list has room for,
// keeps its length.
//
// All of it is prefix sums and copies.  The sums run over the sequences (pages that go
// back, pages that are needed, tokens); from them every page and every token finds its
// sequence by itself, 64 at a time, so that it does not matter how many of them a
// sequence has.  (A wave whose 64 belong to sequences far apart walks over those between
// them, 64 a step: of 8,192 sequences the first and the last alone take 80 us a call where
// all take 15, of 2^20 8,900 where all take 85.)  A small call is one workgroup, which keeps the sums in LDS: bound by
// the latency of its dependent reads (64 sequences, a token each: 5 us).  Others sum in
// tiles of 256 sequences, first each tile, then all, and do the pages that go back, and
// then those that are taken and the tokens, in two more launches (8,192 sequences
// that grow by 24,576 tokens: 18 us in four launches; 24 by 505,668: 15).
#include "as_device.h"
#include "as_internal.h"

namespace as {

namespace {

constexpr int kListThreads = 1024;
constexpr int kListWaves = kListThreads / kWave;
// Changes are cut to what no list holds, so that no sum passes 64 bits.
constexpr int64_t kMostTokens = int64_t(1) << 40;

struct ListArgs {
  int64_t* table;  // [sequences, room]
  int64_t table_stride;
  int64_t room;
  const int64_t* lengths;
  const int64_t* change;
  int64_t* free_pages;
  int64_t free_len;
  int64_t* free_count;
  int64_t page_size;
  int64_t* new_lengths;
  int64_t* token_ptr;  // [sequences + 1]
  int64_t* positions;  // [tokens]
  int64_t* slots;      // [tokens]
  int64_t tokens;
  int64_t sequences;
  int64_t* sums;   // kSums numbers of the whole call
  struct Sums* totals;  // [tiles]
  int64_t* taken;       // [tiles]
  int64_t* back;   // [sequences + 1] pages that go back in front of a sequence
  int64_t* need;   // the same of pages that are needed
  double per_page;  // 1 / page_size
};
enum { kCount, kBack, kNeed, kTokens, kSums };  // count: of the stack, before the call

// t / page_size for 0 <= t < 2^52: the rounded quotient is off by less than one, and is put right.
__device__ __forceinline__ int64_t page_of(const ListArgs& a, int64_t t) {
  const int64_t q = static_cast<int64_t>(static_cast<double>(t) * a.per_page);
  const int64_t rest = t - q * a.page_size;
  return q + (rest >= a.page_size ? 1 : 0) - (rest < 0 ? 1 : 0);
}
// Pages of so many tokens, more than a list has room for where it has no room.
__device__ __forceinline__ int64_t pages_of(const ListArgs& a, int64_t tokens) {
  return tokens > a.room * a.page_size ? a.room + 1 : page_of(a, tokens + a.page_size - 1);
}

struct Change {
  int64_t length, change;
  int64_t held;   // pages it has
  int64_t after;  // tokens, if it is served
  int64_t back;   // pages it gives up
  int64_t need;   // pages it needs more
  bool fits;      // its list has room
};
__device__ __forceinline__ Change change_of(const ListArgs& a, int64_t length, int64_t change) {
  Change c{};
  c.length = length < 0 ? 0 : (length > kMostTokens ? kMostTokens : length);
  c.change = change < -kMostTokens ? -kMostTokens : (change > kMostTokens ? kMostTokens : change);
  c.held = pages_of(a, c.length);
  c.held = c.held < a.room ? c.held : a.room;
  c.after = c.length + c.change;
  c.after = c.after < 0 ? 0 : c.after;
  const int64_t pages = pages_of(a, c.after);
  c.fits = pages <= a.room;
  if (c.change < 0) c.back = pages < c.held ? c.held - pages : 0;
  if (c.change > 0 && c.fits) c.need = pages > c.held ? pages - c.held : 0;
  return c;
}
// What the pages and tokens look up about the sequences: in memory, or in LDS where one workgroup does it all.
struct Lists {
  const int64_t* lengths;
  const int64_t* change;
  const int64_t* back;
  const int64_t* need;
  const int64_t* token_ptr;
};
__device__ __forceinline__ Change change_of(const ListArgs& a, const Lists& l, int64_t b) {
  return change_of(a, l.lengths[b], l.change[b]);
}
// How far the stack reaches when all pages are back.
__device__ __forceinline__ int64_t top_of(const ListArgs& a, int64_t count, int64_t back) {
  return count + back < a.free_len ? count + back : a.free_len;
}
__device__ __forceinline__ bool is_served(const Change& c, int64_t need_before, int64_t top) {
  return c.change <= 0 || (c.fits && (c.need == 0 || need_before + c.need <= top));
}

__device__ __forceinline__ int64_t wave_scan(int64_t v) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int64_t t = __shfl_up(v, o, kWave);
    if (lane_id() >= o) v += t;
  }
  return v;
}
// What is summed over the sequences: pages that go back, pages that are needed, tokens.
struct Sums {
  int64_t v[3];
};
__device__ __forceinline__ Sums sums_of(const Change& c) {
  return Sums{{c.back, c.need, c.change > 0 ? c.change : 0}};
}
__device__ __forceinline__ Sums plus(const Sums& x, const Sums& y) {
  return Sums{{x.v[0] + y.v[0], x.v[1] + y.v[1], x.v[2] + y.v[2]}};
}
template <int WAVES>
struct Scan {
  Sums waves[WAVES + 1];
};
// The sums of the threads before this one, and of all, by the whole workgroup; `any`: the wave has something to add.
template <int WAVES>
__device__ __forceinline__ Sums block_before(const Sums& mine, bool any, Scan<WAVES>& scan, Sums* all) {
  static_assert(WAVES <= kWave);
  Sums upto{};
  if (any) {
#pragma unroll
    for (int i = 0; i < 3; ++i) upto.v[i] = wave_scan(mine.v[i]);
  }
  if (lane_id() == kWave - 1) scan.waves[wave_in_block()] = upto;
  __syncthreads();
  if (threadIdx.x < kWave) {
    const Sums own = lane_id() < WAVES ? scan.waves[lane_id() < WAVES ? lane_id() : 0] : Sums{};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      int64_t x = own.v[i];
#pragma unroll
      for (int o = 1; o < WAVES; o <<= 1) {
        const int64_t t = __shfl_up(x, o, kWave);
        if (lane_id() >= o) x += t;
      }
      if (lane_id() < WAVES) scan.waves[lane_id()].v[i] = x - own.v[i];
      if (lane_id() == WAVES - 1) scan.waves[WAVES].v[i] = x;
    }
  }
  __syncthreads();
  *all = scan.waves[WAVES];
  Sums before = scan.waves[wave_in_block()];
#pragma unroll
  for (int i = 0; i < 3; ++i) before.v[i] += upto.v[i] - mine.v[i];
  return before;
}
__device__ __forceinline__ int64_t wave_max_i64(int64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const int64_t t = __shfl_xor(v, o, kWave);
    v = v > t ? v : t;
  }
  return v;
}
__device__ __forceinline__ int64_t stack_count(const ListArgs& a) {
  const int64_t found = *a.free_count;
  return found < 0 ? 0 : (found > a.free_len ? a.free_len : found);
}

// The sequences of 64 pages or tokens from i on, one for each lane, by the sums in front of the sequences.
__device__ __forceinline__ int sequence_of(const int64_t* __restrict__ before, int64_t n, int64_t i, int64_t end) {
  const int64_t row = uniform_i64(wave_row_of_edge(before, n, i));
  return block_edge_rows(before, n, i, end - i < kWave ? static_cast<int>(end - i) : kWave, row);
}

// Wave `wave` of `waves`: pages that go back.
__device__ __forceinline__ void give_back(const ListArgs& a, const Lists& l, const int64_t (&sums)[kSums], int64_t wave, int64_t waves) {
  for (int64_t k0 = wave * kWave; k0 < sums[kBack]; k0 += waves * kWave) {
    const int b = sequence_of(l.back, a.sequences, k0, sums[kBack]);
    const int64_t k = k0 + lane_id();
    if (k < sums[kBack]) {
      const Change c = change_of(a, l, b);
      int64_t* const entry = a.table + b * a.table_stride + c.held - c.back + (k - l.back[b]);
      const int64_t to = sums[kCount] + sums[kBack] - 1 - k;
      if (to < a.free_len) a.free_pages[to] = *entry;
      *entry = -1;
    }
  }
}

// Pages that are taken.
__device__ __forceinline__ void take(const ListArgs& a, const Lists& l, const int64_t (&sums)[kSums], int64_t wave, int64_t waves) {
  const int64_t top = top_of(a, sums[kCount], sums[kBack]);
  const int64_t all = sums[kNeed] < top ? sums[kNeed] : top;  // nobody who needs a page behind these is served
  for (int64_t k0 = wave * kWave; k0 < all; k0 += waves * kWave) {
    const int b = sequence_of(l.need, a.sequences, k0, all);
    const int64_t k = k0 + lane_id();
    if (k < all) {
      const Change c = change_of(a, l, b);
      const int64_t before = l.need[b];
      if (is_served(c, before, top)) a.table[b * a.table_stride + c.held + (k - before)] = a.free_pages[top - 1 - k];
    }
  }
}

// Positions and places of the tokens, which read the pages that were held from the table and the others from the stack.
__device__ __forceinline__ void place_tokens(const ListArgs& a, const Lists& l, const int64_t (&sums)[kSums], int64_t wave, int64_t waves) {
  const int64_t top = top_of(a, sums[kCount], sums[kBack]);
  for (int64_t t0 = wave * kWave; t0 < a.tokens; t0 += waves * kWave) {
    const int64_t t = t0 + lane_id();
    int64_t position = -1;
    int64_t slot = -1;
    if (t0 < sums[kTokens]) {
      const int b = sequence_of(l.token_ptr, a.sequences, t0, sums[kTokens]);
      const Change c = change_of(a, l, b);
      const int64_t before = l.need[b];
      if (t < sums[kTokens] && is_served(c, before, top)) {
        position = c.length + (t - l.token_ptr[b]);
        const int64_t k = page_of(a, position);
        const int64_t page = k < c.held ? a.table[b * a.table_stride + k] : a.free_pages[top - 1 - before - (k - c.held)];
        slot = page < 0 ? -1 : page * a.page_size + (position - k * a.page_size);
      }
    }
    if (t < a.tokens) {
      a.positions[t] = position;
      a.slots[t] = slot;
    }
  }
}

// All of it by one workgroup, a sequence for each thread.
struct Kept {
  int64_t lengths[kListThreads], change[kListThreads];
  int64_t back[kListThreads + 1], need[kListThreads + 1], token_ptr[kListThreads + 1];
};
__global__ __launch_bounds__(kListThreads) void paged_lists_kernel(ListArgs a) {
  __shared__ Kept kept;
  __shared__ Scan<kListWaves> scan;
  __shared__ int64_t wave_taken[kListWaves];
  const int wave = uniform_i32(wave_in_block());
  const int64_t b = threadIdx.x;
  const bool any = wave * kWave < a.sequences;
  const int64_t count = stack_count(a);
  Change c{};
  if (any && b < a.sequences) {
    const int64_t length = a.lengths[b];
    const int64_t change = a.change[b];
    kept.lengths[b] = length;
    kept.change[b] = change;
    c = change_of(a, length, change);
  }
  Sums all;
  const Sums before = block_before<kListWaves>(sums_of(c), any, scan, &all);
  const int64_t top = top_of(a, count, all.v[0]);
  int64_t taken = 0;
  if (any && b < a.sequences) {
    const bool served = is_served(c, before.v[1], top);
    a.new_lengths[b] = served ? c.after : c.length;
    a.token_ptr[b] = before.v[2];
    kept.back[b] = before.v[0];
    kept.need[b] = before.v[1];
    kept.token_ptr[b] = before.v[2];
    if (served && c.need > 0) taken = before.v[1] + c.need;
  }
  if (any) taken = wave_max_i64(taken);
  if (lane_id() == 0) wave_taken[wave] = taken;
  if (threadIdx.x == 0) {
    kept.back[a.sequences] = all.v[0];
    kept.need[a.sequences] = all.v[1];
    kept.token_ptr[a.sequences] = all.v[2];
    a.token_ptr[a.sequences] = all.v[2];
  }
  __syncthreads();
  if (wave == 0) {
    // the last one that is served has the largest sum
    taken = wave_max_i64(lane_id() < kListWaves ? wave_taken[lane_id()] : 0);
    if (lane_id() == 0) *a.free_count = top - taken;
  }
  const int64_t sums[kSums] = {count, all.v[0], all.v[1], all.v[2]};
  const Lists l{kept.lengths, kept.change, kept.back, kept.need, kept.token_ptr};
  if (all.v[0] > 0) {
    give_back(a, l, sums, wave, kListWaves);
    __syncthreads();
  }
  constexpr int kHalf = kListWaves / 2;
  if (wave < kHalf) {
    take(a, l, sums, wave, kHalf);
  } else {
    place_tokens(a, l, sums, wave - kHalf, kHalf);
  }
}

// Sums of a tile's sequences, one for each thread.
__global__ __launch_bounds__(kBlock) void paged_lists_totals_kernel(ListArgs a) {
  __shared__ Scan<kWavesPerBlock> scan;
  const int64_t b = int64_t(blockIdx.x) * kBlock + threadIdx.x;
  Change c{};
  if (b < a.sequences) c = change_of(a, a.lengths[b], a.change[b]);
  Sums all;
  block_before<kWavesPerBlock>(sums_of(c), true, scan, &all);
  if (threadIdx.x == 0) a.totals[blockIdx.x] = all;
}

// The sums in front of every sequence, who is served, and for each tile the sum of the last one that takes pages.
__global__ __launch_bounds__(kBlock) void paged_lists_sums_kernel(ListArgs a, int tiles) {
  __shared__ Scan<kWavesPerBlock> scan;
  __shared__ Scan<kWavesPerBlock> scan_of_tiles;
  __shared__ int64_t wave_taken[kWavesPerBlock];
  const int64_t count = stack_count(a);
  const int64_t b = int64_t(blockIdx.x) * kBlock + threadIdx.x;
  Change c{};
  if (b < a.sequences) c = change_of(a, a.lengths[b], a.change[b]);
  Sums own;
  Sums before = block_before<kWavesPerBlock>(sums_of(c), true, scan, &own);
  Sums all = own;
  if (tiles > 1) {
    Sums front{};
    Sums rest{};
    for (int i = threadIdx.x; i < tiles; i += kBlock) {
      const Sums t = a.totals[i];
      rest = plus(rest, t);
      if (i < static_cast<int>(blockIdx.x)) front = plus(front, t);
    }
    block_before<kWavesPerBlock>(front, true, scan_of_tiles, &all);
    before = plus(before, all);
    __syncthreads();
    block_before<kWavesPerBlock>(rest, true, scan_of_tiles, &all);
  }
  const int64_t top = top_of(a, count, all.v[0]);
  int64_t taken = 0;
  if (b < a.sequences) {
    const bool served = is_served(c, before.v[1], top);
    a.new_lengths[b] = served ? c.after : c.length;
    a.back[b] = before.v[0];
    a.need[b] = before.v[1];
    a.token_ptr[b] = before.v[2];
    if (served && c.need > 0) taken = before.v[1] + c.need;
  }
  taken = wave_max_i64(taken);
  if (lane_id() == 0) wave_taken[wave_in_block()] = taken;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWavesPerBlock; ++w) taken = taken > wave_taken[w] ? taken : wave_taken[w];
    a.taken[blockIdx.x] = taken;
    if (blockIdx.x == 0) {
      a.back[a.sequences] = all.v[0];
      a.need[a.sequences] = all.v[1];
      a.token_ptr[a.sequences] = all.v[2];
      a.sums[kCount] = count;
      a.sums[kBack] = all.v[0];
      a.sums[kNeed] = all.v[1];
      a.sums[kTokens] = all.v[2];
    }
  }
}

__device__ __forceinline__ Lists in_memory(const ListArgs& a) {
  return Lists{a.lengths, a.change, a.back, a.need, a.token_ptr};
}
__device__ __forceinline__ void read_sums(const ListArgs& a, int64_t (&sums)[kSums]) {
#pragma unroll
  for (int i = 0; i < kSums; ++i) sums[i] = a.sums[i];
}

__global__ __launch_bounds__(kBlock) void paged_lists_back_kernel(ListArgs a) {
  int64_t sums[kSums];
  read_sums(a, sums);
  give_back(a, in_memory(a), sums, int64_t(blockIdx.x) * kWavesPerBlock + uniform_i32(wave_in_block()), int64_t(gridDim.x) * kWavesPerBlock);
}

// The first `takers` workgroups write the pages, the others the tokens; one of their waves the number of pages left.
__global__ __launch_bounds__(kBlock) void paged_lists_take_kernel(ListArgs a, int tiles, int takers) {
  int64_t sums[kSums];
  read_sums(a, sums);
  const int block = static_cast<int>(blockIdx.x);
  const int wave = uniform_i32(wave_in_block());
  if (block == 0 && wave == 0) {
    int64_t taken = 0;
    for (int i = lane_id(); i < tiles; i += kWave) taken = taken > a.taken[i] ? taken : a.taken[i];
    taken = wave_max_i64(taken);
    if (lane_id() == 0) *a.free_count = top_of(a, sums[kCount], sums[kBack]) - taken;
  }
  if (block < takers) {
    take(a, in_memory(a), sums, int64_t(block) * kWavesPerBlock + wave, int64_t(takers) * kWavesPerBlock);
  } else {
    place_tokens(a, in_memory(a), sums, int64_t(block - takers) * kWavesPerBlock + wave,
                 int64_t(gridDim.x - takers) * kWavesPerBlock);
  }
}

// What one workgroup does alone.  64 sequences, a token each: 11.4 us of a captured run of calls, three launches 16.5;
// 1,024 sequences 25 and 39; 64 with 2,048 tokens 14 and 17, but with 4,096 16 and 15, 16 with 8,192 tokens 20 and 15.
constexpr int64_t kAloneSequences = kListThreads;
constexpr int64_t kAloneTokens = 2048;
// How many pages go back the host does not know, but how many entries the lists have.  4 of 64 lists of 256 pages that
// end: 5.0 us, in three launches 7.5; all 64 of 64 pages 9.5 and 7.8, of 256 pages 28 and 7.6, of 1,024 pages 103 and
// 7.9; 20 of 1,000 lists of 64 pages 8 and 13, all 1,000 115 and 14.
constexpr int64_t kAloneEntries = int64_t(1) << 15;
constexpr int64_t kMostBlocks = 1024;

int64_t tiles_of(int64_t sequences) { return sequences > 0 ? (sequences + kBlock - 1) / kBlock : 1; }

}  // namespace

}  // namespace as

using namespace as;

extern "C" {

size_t as_paged_cache_resize_workspace_bytes(int64_t sequences) {
  return sequences < 0 ? 0 : static_cast<size_t>(2 * (sequences + 1) + kSums + 4 * tiles_of(sequences)) * sizeof(int64_t);
}

int as_paged_cache_resize(int64_t* table, int64_t table_stride, int64_t room, const int64_t* lengths,
                          const int64_t* change, int64_t* free_pages, int64_t free_len, int64_t* free_count,
                          int64_t page_size, int64_t* new_lengths, int64_t* token_ptr, int64_t* positions,
                          int64_t* slots, int64_t sequences, int64_t tokens, void* workspace, size_t workspace_bytes,
                          void* stream) {
  clear_error();
  if (sequences < 0 || sequences > (1 << 20)) return fail(AS_ERR_UNSUPPORTED, "at most 2^20 sequences");
  if (page_size < 1 || page_size > (1 << 20))
    return fail(AS_ERR_INVALID_ARGUMENT, "a page holds 1 to 2^20 tokens");
  if (room < 0 || room > kMostTokens / 2 / page_size || table_stride < 0)
    return fail(AS_ERR_INVALID_ARGUMENT, "a list has room for less than 2^39 tokens, and a non-negative stride");
  if (free_len < 0) return fail(AS_ERR_INVALID_ARGUMENT, "the free list must have a non-negative size");
  if (tokens < 0 || tokens > (int64_t(1) << 26)) return fail(AS_ERR_UNSUPPORTED, "at most 2^26 tokens");
  if (free_count == nullptr || token_ptr == nullptr || (sequences > 0 && (lengths == nullptr || change == nullptr ||
      new_lengths == nullptr)) || (sequences > 0 && room > 0 && table == nullptr) ||
      (free_len > 0 && free_pages == nullptr) || (tokens > 0 && (positions == nullptr || slots == nullptr)))
    return fail(AS_ERR_INVALID_ARGUMENT, "null pointer argument");
  const size_t bytes = as_paged_cache_resize_workspace_bytes(sequences);
  if (workspace_bytes < bytes || (bytes > 0 && workspace == nullptr))
    return fail(AS_ERR_WORKSPACE, "page lists need %zu workspace bytes", bytes);
  if (!aligned(workspace, 8)) return fail(AS_ERR_INVALID_ARGUMENT, "the workspace must be 8-byte aligned");
  // later launches read lengths and changes again
  for (const int64_t* const from : {lengths, change}) {
    const auto apart = [&](const int64_t* to, int64_t count, int64_t read) {
      return count == 0 || read == 0 || to + count <= from || from + read <= to;
    };
    if (!apart(new_lengths, sequences, sequences) || !apart(token_ptr, sequences + 1, sequences) ||
        !apart(positions, tokens, sequences) || !apart(slots, tokens, sequences))
      return fail(AS_ERR_INVALID_ARGUMENT, "the results must lie apart from lengths and change");
  }
  int64_t* const ws = static_cast<int64_t*>(workspace);
  const int tiles = static_cast<int>(tiles_of(sequences));
  ListArgs a{};
  a.table = table;
  a.table_stride = table_stride;
  a.room = room;
  a.lengths = lengths;
  a.change = change;
  a.free_pages = free_pages;
  a.free_len = free_len;
  a.free_count = free_count;
  a.page_size = page_size;
  a.new_lengths = new_lengths;
  a.token_ptr = token_ptr;
  a.positions = positions;
  a.slots = slots;
  a.tokens = tokens;
  a.sequences = sequences;
  a.sums = ws;
  a.totals = reinterpret_cast<Sums*>(a.sums + kSums);
  a.taken = a.sums + kSums + 3 * tiles;
  a.back = a.taken + tiles;
  a.need = a.back + sequences + 1;
  a.per_page = 1.0 / static_cast<double>(page_size);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t entries = sequences * room;
  const bool alone = sequences <= kAloneSequences && tokens <= kAloneTokens && entries <= kAloneEntries;
  if (alone) {
    paged_lists_kernel<<<1, kListThreads, 0, s>>>(a);
    return check_launch("paged_cache_resize");
  }
  if (tiles > 1) {
    paged_lists_totals_kernel<<<static_cast<unsigned>(tiles), kBlock, 0, s>>>(a);
    if (const int bad = check_launch("paged_cache_resize (totals)")) return bad;
  }
  paged_lists_sums_kernel<<<static_cast<unsigned>(tiles), kBlock, 0, s>>>(a, tiles);
  if (const int bad = check_launch("paged_cache_resize (sums)")) return bad;
  // a page that goes back is in a list, and one that is taken on the stack
  const auto blocks = [](int64_t items) {
    const int64_t n = (items + kBlock - 1) / kBlock;
    return static_cast<int>(n < 1 ? 1 : (n < kMostBlocks ? n : kMostBlocks));
  };
  paged_lists_back_kernel<<<static_cast<unsigned>(blocks(entries)), kBlock, 0, s>>>(a);
  if (const int bad = check_launch("paged_cache_resize (pages that go back)")) return bad;
  const int takers = blocks(entries < free_len ? entries : free_len);
  paged_lists_take_kernel<<<static_cast<unsigned>(takers + blocks(tokens)), kBlock, 0, s>>>(
      a, tiles, takers);
  return check_launch("paged_cache_resize (pages that are taken)");
}

}  // extern "C"
