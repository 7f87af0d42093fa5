// Attention of one new token of every sequence over the sequence's pages.
//
//   s[t] = scale * <q, k[t]> + table[bucket(length - 1 - t), h]   for the tokens t that are seen
//   out  = sum_t exp(s[t] - m) v[t] / sum_t exp(s[t] - m),   m = max_t s[t]
//   lse  = m + log(sum_t exp(s[t] - m))
//
// Every key and value is read once: bound by memory from a few thousand tokens
// on.  A sequence that sees no token, or only scores of -inf, gives zeros and
// an lse of -inf.  A length beyond the sequence's pages makes its results NaN,
// and so does a page id outside the cache, which is never read.
#include "paged_common.h"
#include "position_map.h"

namespace as {

namespace {

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
  float scale;
};

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

// One wave per (sequence, query head), the widths over its lanes.
template <typename T, typename C>
__global__ __launch_bounds__(kBlock) void paged_attention_kernel(AttentionArgs a, PositionMap map) {
  __shared__ int32_t border[kMaxBuckets];
  if (a.table != nullptr) {
    for (int i = threadIdx.x; i < map.side; i += blockDim.x) border[i] = map.border[i];
  }
  __syncthreads();
  const PagedCache& c = a.cache;
  const int heads_q = c.heads * a.group;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + wave_in_block();
  if (unit >= static_cast<int64_t>(c.sequences) * heads_q) return;
  const int b = static_cast<int>(unit / heads_q);
  const int hq = static_cast<int>(unit - static_cast<int64_t>(b) * heads_q);
  const int h = hq / a.group;
  const int lane = lane_id();
  const PageList list = page_list(c, b);
  const Seen seen = seen_tokens(a, b, list);
  const T* q = static_cast<const T*>(a.query) + b * a.query_stride[0] + hq * a.query_stride[1];
  constexpr int kParts = kMaxWidth / kWave;
  float qv[kParts], acc[kParts];
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const int d = lane + i * kWave;
    qv[i] = d < c.key.width ? Elem<T>::at(q, d) * a.scale : 0.0f;
    acc[i] = 0.0f;
  }
  float m = -INFINITY;
  float l = 0.0f;
  for (int t = seen.begin; t < seen.end; ++t) {
    const int k = t / c.page_size;
    const int slot = t - k * c.page_size;
    const int64_t id = c.page_idx[list.begin + k];
    const bool valid = id >= 0 && id < c.pages;
    const int64_t page = valid ? id : 0;
    const C* kr = static_cast<const C*>(c.key.data) + page * c.key.stride[0] + h * c.key.stride[1] +
                  slot * c.key.stride[2];
    const C* vr = static_cast<const C*>(c.value.data) + page * c.value.stride[0] + h * c.value.stride[1] +
                  slot * c.value.stride[2];
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int d = lane + i * kWave;
      if (d < c.key.width) s = fmaf(qv[i], Elem<C>::at(kr, d), s);
    }
    s = wave_sum_f32(s);
    int ev = 0;
    if constexpr (__is_same(C, E4m3)) {
      s = ldexpf(s, c.key.exponents[page * c.key.exponent_stride[0] + h * c.key.exponent_stride[1] +
                                    slot * c.key.exponent_stride[2]]);
      ev = c.value.exponents[page * c.value.exponent_stride[0] + h * c.value.exponent_stride[1] +
                             slot * c.value.exponent_stride[2]];
    }
    if (a.table != nullptr) {
      const int bucket = bucket_of_distance(border, map.side, seen.end - 1 - t);
      s += Elem<T>::at(static_cast<const T*>(a.table), static_cast<int64_t>(bucket) * heads_q + hq);
    }
    if (!valid) s = NAN;
    const float top = s > m ? s : m;
    const float base = top == -INFINITY ? 0.0f : top;
    const float keep = expf(m - base);
    const float p = expf(s - base);
    l = l * keep + p;
    m = top;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int d = lane + i * kWave;
      acc[i] *= keep;
      if (d < c.value.width) acc[i] = fmaf(p, ldexpf(Elem<C>::at(vr, d), ev), acc[i]);
    }
  }
  const bool empty = l == 0.0f && !seen.bad;
  T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(b) * heads_q + hq) * c.value.width;
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const int d = lane + i * kWave;
    if (d < c.value.width) out[d] = rounded<T>(empty ? 0.0f : acc[i] / l);
  }
  if (a.lse != nullptr && lane == 0) a.lse[unit] = seen.bad ? NAN : (empty ? -INFINITY : m + logf(l));
}

}  // namespace

}  // namespace as

using namespace as;

extern "C" {

size_t as_paged_attention_workspace_bytes(const as_paged_cache* cache, int64_t group, int64_t max_length) {
  (void)cache;
  (void)group;
  (void)max_length;
  return 8;
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
  const size_t need = as_paged_attention_workspace_bytes(cache, group, max_length);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(AS_ERR_WORKSPACE, "paged attention needs %zu workspace bytes", need);
  if (a.cache.sequences == 0) return AS_OK;
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
  a.scale = scale;
  const int64_t units = int64_t(a.cache.sequences) * a.cache.heads * group;
  const dim3 grid(static_cast<unsigned>((units + kWavesPerBlock - 1) / kWavesPerBlock));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_float_element(dtype, [&](auto e) {
    using T = decltype(e);
    if (cache->dtype == AS_DTYPE_E4M3) {
      paged_attention_kernel<T, E4m3><<<grid, kBlock, 0, s>>>(a, map);
    } else {
      paged_attention_kernel<T, T><<<grid, kBlock, 0, s>>>(a, map);
    }
    return check_launch("paged_attention");
  });
}

}  // extern "C"
