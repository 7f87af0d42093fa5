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
// All of it is prefix sums and copies.  One workgroup sums over the sequences (pages
// that go back, pages that are needed, tokens); from the sums every page and every
// token finds its sequence by itself, 64 at a time, so that it does not matter how they
// are spread over the sequences.  Small calls are that one workgroup alone, which is
// bound by the latency of its dependent reads; others do the pages that go back, and
// then those that are taken and the tokens, in two more launches (8,192 sequences,
// 24,576 tokens: AAA us; the workgroup alone BBB).
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
  int64_t* back;   // [sequences + 1] pages that go back in front of a sequence
  int64_t* need;   // the same of pages that are needed
  uint32_t page_magic;  // t / page_size = t * page_magic >> (31 + page_shift) for t < 2^31
  int page_shift;       // -1: tokens of a list may be more
};
enum { kCount, kBack, kNeed, kTokens, kSums };  // count: of the stack, before the call

__device__ __forceinline__ int64_t page_of(const ListArgs& a, int64_t t) {
  if (a.page_shift < 0) return static_cast<int64_t>(static_cast<uint64_t>(t) / static_cast<uint64_t>(a.page_size));
  return static_cast<int64_t>((static_cast<uint64_t>(static_cast<uint32_t>(t)) * a.page_magic) >> (31 + a.page_shift));
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
__device__ __forceinline__ Change change_of(const ListArgs& a, int64_t b) {
  return change_of(a, a.lengths[b], a.change[b]);
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
// What the threads before this one have, and what all have (by the whole workgroup).
__device__ __forceinline__ int64_t block_before(int64_t mine, int64_t* waves, int64_t* all) {
  const int64_t upto = wave_scan(mine);
  __syncthreads();
  if (lane_id() == kWave - 1) waves[wave_in_block()] = upto;
  __syncthreads();
  int64_t before = upto - mine;
  *all = 0;
#pragma unroll
  for (int w = 0; w < kListWaves; ++w) {
    if (w < wave_in_block()) before += waves[w];
    *all += waves[w];
  }
  return before;
}

// By one workgroup: thread t sums over `each` sequences, then writes the sums in front of them.
__device__ __forceinline__ void sum_up(const ListArgs& a, int64_t (&sums)[kSums]) {
  __shared__ int64_t waves[kListWaves];
  const int64_t n = a.sequences;
  const int64_t each = (n + kListThreads - 1) / kListThreads;
  const int64_t from = threadIdx.x * each;
  const int64_t to = from + each < n ? from + each : n;
  int64_t count = *a.free_count;
  count = count < 0 ? 0 : (count > a.free_len ? a.free_len : count);
  int64_t back = 0;
  int64_t need = 0;
  int64_t tokens = 0;
#pragma unroll 4
  for (int64_t b = from; b < to; ++b) {
    const Change c = change_of(a, b);
    back += c.back;
    need += c.need;
    tokens += c.change > 0 ? c.change : 0;
  }
  back = block_before(back, waves, &sums[kBack]);
  need = block_before(need, waves, &sums[kNeed]);
  tokens = block_before(tokens, waves, &sums[kTokens]);
  sums[kCount] = count;
  const int64_t top = top_of(a, count, sums[kBack]);
  int64_t taken = 0;
#pragma unroll 4
  for (int64_t b = from; b < to; ++b) {
    const Change c = change_of(a, b);
    const bool served = is_served(c, need, top);
    a.new_lengths[b] = served ? c.after : c.length;
    a.back[b] = back;
    a.need[b] = need;
    a.token_ptr[b] = tokens;
    if (served && c.need > 0) taken = need + c.need;
    back += c.back;
    need += c.need;
    tokens += c.change > 0 ? c.change : 0;
  }
  // the last one that is served has the largest sum
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const int64_t t = __shfl_xor(taken, o, kWave);
    taken = taken > t ? taken : t;
  }
  __syncthreads();
  if (lane_id() == 0) waves[wave_in_block()] = taken;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < kListWaves; ++w) taken = taken > waves[w] ? taken : waves[w];
    a.back[n] = sums[kBack];
    a.need[n] = sums[kNeed];
    a.token_ptr[n] = sums[kTokens];
    *a.free_count = top - taken;
  }
}

// The sequences of 64 pages or tokens from i on, one for each lane, by the sums in front of the sequences.  (Each lane
// reads sums of its own: what this workgroup has just written must not come through the scalar cache.)
__device__ __forceinline__ int sequence_of(const int64_t* __restrict__ before, int64_t n, int64_t i, int64_t end) {
  const int64_t row = uniform_i64(wave_row_of_edge(before, n, i));
  return block_edge_rows(before, n, i, end - i < kWave ? static_cast<int>(end - i) : kWave, row);
}

// Wave `wave` of `waves`: pages that go back.
__device__ __forceinline__ void give_back(const ListArgs& a, const int64_t (&sums)[kSums], int64_t wave, int64_t waves) {
  for (int64_t k0 = wave * kWave; k0 < sums[kBack]; k0 += waves * kWave) {
    const int b = sequence_of(a.back, a.sequences, k0, sums[kBack]);
    const int64_t k = k0 + lane_id();
    if (k < sums[kBack]) {
      const Change c = change_of(a, b);
      int64_t* const entry = a.table + b * a.table_stride + c.held - c.back + (k - a.back[b]);
      const int64_t to = sums[kCount] + sums[kBack] - 1 - k;
      if (to < a.free_len) a.free_pages[to] = *entry;
      *entry = -1;
    }
  }
}

// Pages that are taken.
__device__ __forceinline__ void take(const ListArgs& a, const int64_t (&sums)[kSums], int64_t wave, int64_t waves) {
  const int64_t top = top_of(a, sums[kCount], sums[kBack]);
  const int64_t all = sums[kNeed] < top ? sums[kNeed] : top;  // nobody who needs a page behind these is served
  for (int64_t k0 = wave * kWave; k0 < all; k0 += waves * kWave) {
    const int b = sequence_of(a.need, a.sequences, k0, all);
    const int64_t k = k0 + lane_id();
    if (k < all) {
      const Change c = change_of(a, b);
      const int64_t before = a.need[b];
      if (is_served(c, before, top)) a.table[b * a.table_stride + c.held + (k - before)] = a.free_pages[top - 1 - k];
    }
  }
}

// Positions and places of the tokens, which read the pages that were held from the table and the others from the stack.
__device__ __forceinline__ void place_tokens(const ListArgs& a, const int64_t (&sums)[kSums], int64_t wave, int64_t waves) {
  const int64_t top = top_of(a, sums[kCount], sums[kBack]);
  for (int64_t t0 = wave * kWave; t0 < a.tokens; t0 += waves * kWave) {
    const int64_t t = t0 + lane_id();
    int64_t position = -1;
    int64_t slot = -1;
    if (t0 < sums[kTokens]) {
      const int b = sequence_of(a.token_ptr, a.sequences, t0, sums[kTokens]);
      const Change c = change_of(a, b);
      const int64_t before = a.need[b];
      if (t < sums[kTokens] && is_served(c, before, top)) {
        position = c.length + (t - a.token_ptr[b]);
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

__global__ __launch_bounds__(kListThreads) void paged_lists_kernel(ListArgs a, bool alone) {
  int64_t sums[kSums];
  sum_up(a, sums);
  if (!alone) {
    if (threadIdx.x == 0) {
#pragma unroll
      for (int i = 0; i < kSums; ++i) a.sums[i] = sums[i];
    }
    return;
  }
  __syncthreads();
  if (sums[kBack] > 0) {
    give_back(a, sums, uniform_i32(wave_in_block()), kListWaves);
    __syncthreads();
  }
  take(a, sums, uniform_i32(wave_in_block()), kListWaves);
  place_tokens(a, sums, uniform_i32(wave_in_block()), kListWaves);
}

__device__ __forceinline__ void read_sums(const ListArgs& a, int64_t (&sums)[kSums]) {
#pragma unroll
  for (int i = 0; i < kSums; ++i) sums[i] = a.sums[i];
}

__global__ __launch_bounds__(kBlock) void paged_lists_back_kernel(ListArgs a) {
  int64_t sums[kSums];
  read_sums(a, sums);
  give_back(a, sums, int64_t(blockIdx.x) * kWavesPerBlock + uniform_i32(wave_in_block()), int64_t(gridDim.x) * kWavesPerBlock);
}

// The first `takers` workgroups write the pages, the others the tokens.
__global__ __launch_bounds__(kBlock) void paged_lists_take_kernel(ListArgs a, int takers) {
  int64_t sums[kSums];
  read_sums(a, sums);
  const int block = static_cast<int>(blockIdx.x);
  if (block < takers) {
    take(a, sums, int64_t(block) * kWavesPerBlock + uniform_i32(wave_in_block()), int64_t(takers) * kWavesPerBlock);
  } else {
    place_tokens(a, sums, int64_t(block - takers) * kWavesPerBlock + uniform_i32(wave_in_block()),
                 int64_t(gridDim.x - takers) * kWavesPerBlock);
  }
}

// What one workgroup does alone: with more the other two launches pay.
constexpr int64_t kAloneSequences = 1024;
constexpr int64_t kAloneTokens = 2048;
constexpr int64_t kMostBlocks = 1024;

}  // namespace

}  // namespace as

using namespace as;

extern "C" {

size_t as_paged_cache_resize_workspace_bytes(int64_t sequences) {
  return sequences < 0 ? 0 : static_cast<size_t>(2 * (sequences + 1) + kSums) * sizeof(int64_t);
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
  int64_t* const ws = static_cast<int64_t*>(workspace);
  ListArgs a{table,       table_stride, room,      lengths, change, free_pages, free_len, free_count,      page_size,
             new_lengths, token_ptr,    positions, slots,   tokens, sequences,  ws,       ws + kSums, ws + kSums + sequences + 1,
             0u,          0};
  // tokens of a list and page_size - 1 more below 2^31: M = ceil(2^(31 + s) / S) with s = ceil(log2 S) is below 2^32
  a.page_shift = (room + 1) * page_size <= INT32_MAX ? 0 : -1;
  if (a.page_shift == 0) {
    while ((1 << a.page_shift) < page_size) ++a.page_shift;
    a.page_magic = static_cast<uint32_t>(((uint64_t(1) << (31 + a.page_shift)) + page_size - 1) / static_cast<uint64_t>(page_size));
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool alone = sequences <= kAloneSequences && tokens <= kAloneTokens;
  paged_lists_kernel<<<1, kListThreads, 0, s>>>(a, alone);
  if (const int bad = check_launch("paged_cache_resize")) return bad;
  if (alone) return AS_OK;
  // a page that goes back is in a list, and one that is taken on the stack
  const auto blocks = [](int64_t items) {
    const int64_t n = (items + kBlock - 1) / kBlock;
    return static_cast<int>(n < 1 ? 1 : (n < kMostBlocks ? n : kMostBlocks));
  };
  const int64_t entries = sequences * room;
  paged_lists_back_kernel<<<static_cast<unsigned>(blocks(entries)), kBlock, 0, s>>>(a);
  if (const int bad = check_launch("paged_cache_resize (pages that go back)")) return bad;
  const int takers = blocks(entries < free_len ? entries : free_len);
  paged_lists_take_kernel<<<static_cast<unsigned>(takers + blocks(tokens)), kBlock, 0, s>>>(a, takers);
  return check_launch("paged_cache_resize (pages that are taken)");
}

}  // extern "C"
