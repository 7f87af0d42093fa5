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
// All of it is prefix sums and copies: bound by latency, and by memory for prompts.
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
  int64_t* base;  // [sequences] where in the stack its first page goes or comes from; -1: it is not served
};

struct Change {
  int64_t length, change;
  int64_t held;   // pages it has
  int64_t after;  // tokens, if it is served
  int64_t back;   // pages it gives up
  int64_t need;   // pages it needs more
  bool fits;      // its list has room
};
__device__ __forceinline__ int64_t pages_of(const ListArgs& a, int64_t tokens) {
  return static_cast<int64_t>((static_cast<uint64_t>(tokens) + a.page_size - 1) / a.page_size);
}
__device__ __forceinline__ Change change_of(const ListArgs& a, int64_t b) {
  Change c{};
  c.length = a.lengths[b];
  c.length = c.length < 0 ? 0 : (c.length > kMostTokens ? kMostTokens : c.length);
  c.change = a.change[b];
  c.change = c.change < -kMostTokens ? -kMostTokens : (c.change > kMostTokens ? kMostTokens : c.change);
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

// One workgroup: thread t sums over `each` sequences, then waves take turns with the
// sequences, first for the pages that go back, then for those that are taken.
__global__ __launch_bounds__(kListThreads) void paged_lists_kernel(ListArgs a) {
  __shared__ int64_t waves[kListWaves];
  __shared__ int64_t taken_of[kListWaves];
  const int64_t n = a.sequences;
  const int64_t each = (n + kListThreads - 1) / kListThreads;
  const int64_t from = threadIdx.x * each;
  const int64_t to = from + each < n ? from + each : n;
  int64_t count = *a.free_count;
  count = count < 0 ? 0 : (count > a.free_len ? a.free_len : count);
  int64_t back = 0;
  int64_t need = 0;
  int64_t tokens = 0;
  for (int64_t b = from; b < to; ++b) {
    const Change c = change_of(a, b);
    back += c.back;
    need += c.need;
    tokens += c.change > 0 ? c.change : 0;
  }
  int64_t all_back;
  int64_t all;
  back = block_before(back, waves, &all_back);
  need = block_before(need, waves, &all);
  tokens = block_before(tokens, waves, &all);
  if (threadIdx.x == 0) a.token_ptr[0] = 0;
  const int64_t top = count + all_back < a.free_len ? count + all_back : a.free_len;
  int64_t taken = 0;
  for (int64_t b = from; b < to; ++b) {
    const Change c = change_of(a, b);
    const bool served = c.change <= 0 || (c.fits && (c.need == 0 || need + c.need <= top));
    a.new_lengths[b] = served ? c.after : c.length;
    tokens += c.change > 0 ? c.change : 0;
    a.token_ptr[b + 1] = tokens;
    a.base[b] = c.change < 0 ? count + all_back - 1 - back : (!served ? -1 : (c.need > 0 ? top - 1 - need : 0));
    if (served && c.need > 0) taken = need + c.need;
    back += c.back;
    need += c.need;
  }
  // the last one that is served has the largest sum
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const int64_t t = __shfl_xor(taken, o, kWave);
    taken = taken > t ? taken : t;
  }
  if (lane_id() == 0) taken_of[wave_in_block()] = taken;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < kListWaves; ++w) taken = taken > taken_of[w] ? taken : taken_of[w];
    *a.free_count = top - taken;
  }
  for (int64_t b = wave_in_block(); b < n; b += kListWaves) {
    const Change c = change_of(a, b);
    const int64_t base = a.base[b];
    int64_t* const list = a.table + b * a.table_stride;
    for (int64_t k = lane_id(); k < c.back; k += kWave) {
      int64_t* const entry = list + c.held - c.back + k;
      if (base - k < a.free_len) a.free_pages[base - k] = *entry;
      *entry = -1;
    }
  }
  __syncthreads();
  for (int64_t b = wave_in_block(); b < n; b += kListWaves) {
    const Change c = change_of(a, b);
    if (c.change <= 0) continue;
    const int64_t base = a.base[b];
    int64_t* const list = a.table + b * a.table_stride;
    for (int64_t k = lane_id(); base >= 0 && k < c.need; k += kWave) list[c.held + k] = a.free_pages[base - k];
    const int64_t first = a.token_ptr[b];
    const int64_t last = first + c.change < a.tokens ? first + c.change : a.tokens;
    for (int64_t t = first + lane_id(); t < last; t += kWave) {
      const int64_t position = base >= 0 ? c.length + (t - first) : -1;
      int64_t slot = -1;
      if (base >= 0) {
        const int64_t k = position / a.page_size;
        const int64_t page = k < c.held ? list[k] : a.free_pages[base - (k - c.held)];
        slot = page < 0 ? -1 : page * a.page_size + (position - k * a.page_size);
      }
      a.positions[t] = position;
      a.slots[t] = slot;
    }
  }
  for (int64_t t = all + threadIdx.x; t < a.tokens; t += kListThreads) {
    a.positions[t] = -1;
    a.slots[t] = -1;
  }
}

}  // namespace

}  // namespace as

using namespace as;

extern "C" {

size_t as_paged_cache_resize_workspace_bytes(int64_t sequences) {
  return sequences < 0 ? 0 : static_cast<size_t>(sequences) * sizeof(int64_t);
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
  const ListArgs a{table,      table_stride, room,      lengths,   change, free_pages, free_len,  free_count,
                   page_size,  new_lengths,  token_ptr, positions, slots,  tokens,     sequences, static_cast<int64_t*>(workspace)};
  paged_lists_kernel<<<1, kListThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  return check_launch("paged_cache_resize");
}

}  // extern "C"
