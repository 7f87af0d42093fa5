// Attention of one new token of every sequence over pages of 4-bit numbers.
//
// The same sums as over other pages (paged_attention.hip); keys and values are
// code * 2^(e - 127) with an exponent for each 32 numbers of a row.
//
// One workgroup has a query head of a sequence; its four waves take turns with 64
// tokens each.  A lane is a token for the scores, and two bytes of a row (four
// columns) for the weighted sum, so that nothing is read twice but the queries.

#include "paged_shares.h"

namespace as {

namespace {

__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

template <typename T>
__global__ __launch_bounds__(kBlock) void paged_attention_e2m1_kernel(AttentionArgs a, PositionMap map) {
  __shared__ int32_t border[kMaxBuckets + 1];
  __shared__ float q[kMaxWidth];
  __shared__ float wave_top[kWavesPerBlock];
  __shared__ float wave_sum[kWavesPerBlock];
  __shared__ float wave_out[kWavesPerBlock][kMaxWidth];

  const PagedCache& c = a.cache;
  const int heads_q = c.heads * a.group;
  const int b = static_cast<int>(blockIdx.x / static_cast<unsigned>(heads_q));
  const int hq = static_cast<int>(blockIdx.x) - b * heads_q;
  const int h = hq / a.group;
  const int lane = lane_id();
  const int wave = uniform_i32(wave_in_block());
  const int key_width = c.key.width;
  const int width = c.value.width;

  if (a.table != nullptr) stage_borders(border, map);
  const T* q_row = static_cast<const T*>(a.query) + b * a.query_stride[0] + hq * a.query_stride[1];
  for (int i = threadIdx.x; i < kMaxWidth; i += kBlock) q[i] = i < key_width ? Elem<T>::at(q_row, i) : 0.0f;
  __syncthreads();

  const PageList list = page_list(c, b);
  const Seen seen = seen_tokens(a, b, list);
  const int64_t* pages = c.page_idx + list.begin;
  const uint8_t* key_base = static_cast<const uint8_t*>(c.key.data) + h * c.key.stride[1];
  const uint8_t* value_base = static_cast<const uint8_t*>(c.value.data) + h * c.value.stride[1];
  const uint8_t* key_e = reinterpret_cast<const uint8_t*>(c.key.exponents) + h * c.key.exponent_stride[1];
  const uint8_t* value_e = reinterpret_cast<const uint8_t*>(c.value.exponents) + h * c.value.exponent_stride[1];

  float top = -INFINITY;
  float sum = 0.0f;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // columns 2 * lane, 2 * lane + 1, and those 128 further
  for (int t0 = seen.begin + wave * kWave; t0 < seen.end; t0 += kWavesPerBlock * kWave) {
    const int t = t0 + lane;
    const bool in_sight = t < seen.end;
    const int at = in_sight ? t : seen.end - 1;
    const int entry = page_of_token(a, at);
    const int64_t slot = at - entry * c.page_size;
    const int64_t id = pages[entry];
    const bool bad = id < 0 || id >= c.pages;
    const int64_t page = bad ? 0 : id;
    const uint8_t* row = key_base + page * c.key.stride[0] + slot * c.key.stride[2];
    const uint8_t* row_e = key_e + page * c.key.exponent_stride[0] + slot * c.key.exponent_stride[2];
    float score = 0.0f;
    for (int d0 = 0; d0 < key_width; d0 += kGroup) {
      const int d1 = d0 + kGroup < key_width ? d0 + kGroup : key_width;
      float part = 0.0f;
      for (int d = d0; d < d1; d += 2) {
        float x[8];
        pairs_to_floats(row[d / 2], x);
        part = fmaf(x[0], q[d], part);
        part = fmaf(x[1], q[d + 1], part);
      }
      score = fmaf(part, group_scale(row_e[d0 / kGroup]), score);
    }
    score *= a.scale;
    if (a.table != nullptr)
      score += Elem<T>::at(static_cast<const T*>(a.table),
                           static_cast<int64_t>(bucket_of_distance(border, map, seen.end - 1 - at)) * heads_q + hq);
    if (bad) score = NAN;
    if (!in_sight) score = -INFINITY;
    const float next = fmaxf(top, wave_max_f32(score));
    const float from = next == -INFINITY ? 0.0f : next;
    const float keep = top == -INFINITY ? 0.0f : exp_of(top - from);
    top = next;
    const float weight = exp_of(score - from);
    sum = sum * keep + weight;
#pragma unroll
    for (float& x : acc) x *= keep;
    const int count = seen.end - t0 < kWave ? seen.end - t0 : kWave;
    for (int i = 0; i < count; ++i) {
      const float w = bcast_f32(weight, i);
      const int64_t p = __shfl(page, i, kWave);
      const int64_t s = __shfl(slot, i, kWave);
      const uint8_t* from_row = value_base + p * c.value.stride[0] + s * c.value.stride[2];
      const uint8_t* from_e = value_e + p * c.value.exponent_stride[0] + s * c.value.exponent_stride[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int d = 2 * lane + 128 * k;
        if (d < width) {
          float x[8];
          pairs_to_floats(from_row[d / 2], x);
          const float scale = group_scale(from_e[d / kGroup]);
          acc[2 * k] = fmaf(w, x[0] * scale, acc[2 * k]);
          acc[2 * k + 1] = fmaf(w, x[1] * scale, acc[2 * k + 1]);
        }
      }
    }
  }
  sum = wave_sum_f32(sum);
  if (lane == 0) {
    wave_top[wave] = top;
    wave_sum[wave] = sum;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) wave_out[wave][2 * lane + 128 * (k / 2) + k % 2] = acc[k];
  __syncthreads();
  float most = wave_top[0];
#pragma unroll
  for (int w = 1; w < kWavesPerBlock; ++w) most = fmaxf(most, wave_top[w]);
  const int d = threadIdx.x;
  if (d >= width) return;
  float total = 0.0f;
  float x = 0.0f;
#pragma unroll
  for (int w = 0; w < kWavesPerBlock; ++w) {
    const float f = wave_top[w] == -INFINITY ? 0.0f : exp_of(wave_top[w] - most);
    total = fmaf(f, wave_sum[w], total);
    x = fmaf(f, wave_out[w][d], x);
  }
  const bool none = total == 0.0f;
  static_cast<T*>(a.out)[static_cast<int64_t>(blockIdx.x) * width + d] =
      rounded<T>(seen.bad ? NAN : (none ? 0.0f : x / total));
  if (a.lse != nullptr && d == 0)
    a.lse[blockIdx.x] = seen.bad ? NAN : (none ? -INFINITY : fmaf(__builtin_amdgcn_logf(total), kLn2, most));
}

}  // namespace

int launch_paged_attention_e2m1(const AttentionArgs& a, const PositionMap& map, int dtype, hipStream_t s) {
  return with_float_element(dtype, [&](auto e) {
    using T = decltype(e);
    const dim3 grid(static_cast<unsigned>(a.cache.sequences * a.cache.heads * a.group));
    paged_attention_e2m1_kernel<T><<<grid, kBlock, 0, s>>>(a, map);
    return check_launch("paged_attention");
  });
}

}  // namespace as
