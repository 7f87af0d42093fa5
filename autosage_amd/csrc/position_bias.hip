// Learned bias of the distance between the two nodes of every edge.
//
//   out[h, e] = table[bucket(pos[col[e]] - pos[row(e)]), h]
//   grad_table[b, h] = sum over the edges e of bucket b of grad[h, e]
//
// Both are bound by memory: 8 bytes of column and `heads` elements an edge.
#include "as_device.h"
#include "as_internal.h"
#include "elem16.h"
#include "position_map.h"

namespace as {

namespace {

// Edges of one wave: the row of the first is found once (64 probes a step),
// the rows of the others follow block by block.
constexpr int kEdgesPerWave = 1024;

struct EdgeWalk {
  const int64_t* crow;
  const int64_t* col;
  const int64_t* positions;  // null: node ids are positions
  int64_t n;
  int64_t nnz;
};

// The bucket of edge b + min(lane, cnt - 1); `row` is the row of edge b and
// becomes the row of the block's last edge.  Ids outside the positions are
// clamped to them, so that a bad graph reads nothing out of bounds.
__device__ __forceinline__ int block_buckets(const EdgeWalk& w, const int32_t* border, int side, int both_sides,
                                             int64_t b, int cnt, int64_t& row) {
  const int lane = lane_id();
  const int r = block_edge_rows(w.crow, w.n, b, cnt, row);
  row = uniform_i32(__builtin_amdgcn_readlane(r, 63));
  int64_t c = w.col[b + (lane < cnt ? lane : cnt - 1)];
  int64_t q = r;
  if (w.positions != nullptr) {
    c = c < 0 ? 0 : (c >= w.n ? w.n - 1 : c);
    c = w.positions[c];
    q = w.positions[r];
  }
  return bucket_of_relative(border, side, both_sides, c - q);
}

__device__ __forceinline__ void stage_borders(int32_t* lds, const PositionMap& map) {
  for (int i = threadIdx.x; i < map.side; i += blockDim.x) lds[i] = map.border[i];
}

template <typename T>
__global__ __launch_bounds__(kBlock) void position_bias_kernel(EdgeWalk w, PositionMap map,
                                                               const T* __restrict__ table, T* __restrict__ out,
                                                               int heads) {
  __shared__ int32_t border[kMaxBuckets];
  stage_borders(border, map);
  __syncthreads();
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + wave_in_block()) * kEdgesPerWave;
  if (first >= w.nnz) return;
  const int64_t end = first + kEdgesPerWave < w.nnz ? first + kEdgesPerWave : w.nnz;
  int64_t row = wave_row_of_edge(w.crow, w.n, first);
  for (int64_t b = first; b < end; b += kWave) {
    const int cnt = end - b < kWave ? static_cast<int>(end - b) : kWave;
    const int k = block_buckets(w, border, map.side, map.both_sides, b, cnt, row);
    if (lane_id() < cnt) {
      for (int h = 0; h < heads; ++h) out[h * w.nnz + b + lane_id()] = table[k * heads + h];
    }
  }
}

// ---- gradient -----------------------------------------------------------------
// Every thread keeps a sum of its own for each bucket, in a column of LDS
// (bucket-major: a wave's 64 columns lie in different banks), so nothing is
// added atomically and the order of every sum is fixed: the same inputs give
// the same bits.  A thread adds at most kEdgesPerThread numbers in fp32; all
// sums above that are fp64.
constexpr int kEdgesPerThread = 64;

inline int gradient_threads(int64_t buckets) { return buckets <= 64 ? 256 : (buckets <= 128 ? 128 : 64); }
inline int64_t gradient_chunks(int64_t nnz, int64_t buckets) {
  const int64_t edges = static_cast<int64_t>(gradient_threads(buckets)) * kEdgesPerThread;
  return (nnz + edges - 1) / edges;
}

template <typename T>
__global__ __launch_bounds__(kBlock) void position_bias_grad_kernel(EdgeWalk w, PositionMap map,
                                                                    const T* __restrict__ grad,
                                                                    double* __restrict__ partial, int heads,
                                                                    int buckets) {
  extern __shared__ float sums[];  // [buckets][blockDim.x]
  __shared__ int32_t border[kMaxBuckets];
  stage_borders(border, map);
  const int threads = blockDim.x;
  for (int k = 0; k < buckets; ++k) sums[k * threads + threadIdx.x] = 0.0f;
  __syncthreads();
  const int h = blockIdx.y;
  const int64_t first =
      (static_cast<int64_t>(blockIdx.x) * (threads / kWave) + wave_in_block()) * kWave * kEdgesPerThread;
  if (first < w.nnz) {
    const int64_t end = first + kWave * kEdgesPerThread < w.nnz ? first + kWave * kEdgesPerThread : w.nnz;
    int64_t row = wave_row_of_edge(w.crow, w.n, first);
    for (int64_t b = first; b < end; b += kWave) {
      const int cnt = end - b < kWave ? static_cast<int>(end - b) : kWave;
      const int k = block_buckets(w, border, map.side, map.both_sides, b, cnt, row);
      if (lane_id() < cnt) sums[k * threads + threadIdx.x] += Elem<T>::at(grad, h * w.nnz + b + lane_id());
    }
  }
  __syncthreads();
  for (int k = wave_in_block(); k < buckets; k += threads / kWave) {
    double s = 0.0;
    for (int t = lane_id(); t < threads; t += kWave) s += sums[k * threads + t];
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane_id() == 0) partial[(static_cast<int64_t>(blockIdx.x) * heads + h) * buckets + k] = s;
  }
}

// One wave per table entry sums the chunks, lane l those with index l mod 64.
template <typename T>
__global__ __launch_bounds__(kBlock) void position_bias_grad_join_kernel(const double* __restrict__ partial,
                                                                         T* __restrict__ grad_table, int64_t chunks,
                                                                         int heads, int buckets) {
  const int entry = blockIdx.x * kWavesPerBlock + wave_in_block();
  if (entry >= heads * buckets) return;
  const int h = entry / buckets;
  const int k = entry - h * buckets;
  double s = 0.0;
  for (int64_t c = lane_id(); c < chunks; c += kWave) s += partial[(c * heads + h) * buckets + k];
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane_id() == 0) Elem<T>::put(grad_table + static_cast<int64_t>(k) * heads + h, s);
}

int check_position_bias(const int64_t* crow, const int64_t* col, const void* table, const void* edges, int64_t n,
                        int64_t nnz, int64_t heads, int dtype) {
  if (dtype != AS_DTYPE_F32 && dtype != AS_DTYPE_BF16 && dtype != AS_DTYPE_F16)
    return fail(AS_ERR_INVALID_ARGUMENT, "dtype must be AS_DTYPE_F32, AS_DTYPE_BF16 or AS_DTYPE_F16");
  if (n < 0 || n > INT32_MAX) return fail(AS_ERR_INVALID_ARGUMENT, "N exceeds kernel index range");
  if (nnz < 0) return fail(AS_ERR_INVALID_ARGUMENT, "nnz must be non-negative");
  if (nnz > 0 && n == 0) return fail(AS_ERR_INVALID_ARGUMENT, "edges without rows");
  if (heads < 1 || heads > 65535) return fail(AS_ERR_INVALID_ARGUMENT, "heads must lie in [1, 65535]");
  if (table == nullptr) return fail(AS_ERR_INVALID_ARGUMENT, "null table pointer");
  if (nnz > 0 && (crow == nullptr || col == nullptr || edges == nullptr))
    return fail(AS_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (nnz > (int64_t(1) << 40)) return fail(AS_ERR_UNSUPPORTED, "at most 2^40 edges");
  return AS_OK;
}

template <typename F>
int with_element(int dtype, F&& f) {
  if (dtype == AS_DTYPE_BF16) return f(Bf16{});
  if (dtype == AS_DTYPE_F16) return f(Fp16{});
  return f(float{});
}

}  // namespace

}  // namespace as

using namespace as;

extern "C" {

int as_csr_position_bias(const int64_t* crow, const int64_t* col, const int64_t* positions, const void* table,
                         void* out, int64_t n, int64_t nnz, int64_t heads, int64_t buckets, const int32_t* borders,
                         int both_sides, int dtype, void* stream) {
  clear_error();
  if (const int bad = check_position_bias(crow, col, table, out, n, nnz, heads, dtype)) return bad;
  PositionMap map;
  if (const int bad = fill_position_map(&map, borders, buckets, both_sides)) return bad;
  if (nnz == 0) return AS_OK;
  const EdgeWalk walk{crow, col, positions, n, nnz};
  const int64_t per_block = int64_t(kEdgesPerWave) * kWavesPerBlock;
  const dim3 grid(static_cast<unsigned>((nnz + per_block - 1) / per_block));
  return with_element(dtype, [&](auto e) {
    using T = decltype(e);
    position_bias_kernel<T><<<grid, kBlock, 0, static_cast<hipStream_t>(stream)>>>(
        walk, map, static_cast<const T*>(table), static_cast<T*>(out), static_cast<int>(heads));
    return check_launch("csr_position_bias");
  });
}

size_t as_csr_position_bias_backward_workspace_bytes(int64_t nnz, int64_t heads, int64_t buckets) {
  if (nnz <= 0 || heads <= 0 || buckets <= 0) return 8;
  return static_cast<size_t>(gradient_chunks(nnz, buckets)) * heads * buckets * sizeof(double);
}

int as_csr_position_bias_backward(const int64_t* crow, const int64_t* col, const int64_t* positions, const void* grad,
                                  void* grad_table, int64_t n, int64_t nnz, int64_t heads, int64_t buckets,
                                  const int32_t* borders, int both_sides, int dtype, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  clear_error();
  if (const int bad = check_position_bias(crow, col, grad_table, grad, n, nnz, heads, dtype)) return bad;
  PositionMap map;
  if (const int bad = fill_position_map(&map, borders, buckets, both_sides)) return bad;
  const size_t need = as_csr_position_bias_backward_workspace_bytes(nnz, heads, buckets);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(AS_ERR_WORKSPACE, "the position bias gradient needs %zu workspace bytes", need);
  const EdgeWalk walk{crow, col, positions, n, nnz};
  const int threads = gradient_threads(buckets);
  const int64_t chunks = nnz > 0 ? gradient_chunks(nnz, buckets) : 0;
  double* partial = static_cast<double*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_element(dtype, [&](auto e) {
    using T = decltype(e);
    if (chunks > 0) {
      position_bias_grad_kernel<T>
          <<<dim3(static_cast<unsigned>(chunks), static_cast<unsigned>(heads)), threads,
             static_cast<size_t>(buckets) * threads * sizeof(float), s>>>(
              walk, map, static_cast<const T*>(grad), partial, static_cast<int>(heads), static_cast<int>(buckets));
      if (const int bad = check_launch("csr_position_bias (backward)")) return bad;
    }
    const int64_t entries = heads * buckets;
    position_bias_grad_join_kernel<T>
        <<<dim3(static_cast<unsigned>((entries + kWavesPerBlock - 1) / kWavesPerBlock)), kBlock, 0, s>>>(
            partial, static_cast<T*>(grad_table), chunks, static_cast<int>(heads), static_cast<int>(buckets));
    return check_launch("csr_position_bias (backward join)");
  });
}

}  // extern "C"
