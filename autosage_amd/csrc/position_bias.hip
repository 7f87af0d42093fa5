// Learned bias of the distance between the two nodes of every edge.
//
//   out[h, e] = table[bucket(pos[col[e]] - pos[row(e)]), h]
//   grad_table[b, h] = sum over the edges e of bucket b of grad[h, e]
//
// Both are bound by memory.  Forward, 8 bytes of column and `heads` elements an
// edge: a wave finds the buckets of 256 edges once, four neighbours a lane, and
// then goes through the heads with 16-byte accesses (8 bytes in 16 bits), stored
// past the caches (16M edges, 4 heads, float32: 68 us, 5.6 TB/s; 104 through
// them).  A forward pass that will be differentiated keeps the buckets, one byte
// an edge, so that the gradient reads neither the graph nor the positions.
#include "as_device.h"
#include "as_internal.h"
#include "elem16.h"
#include "position_map.h"

namespace as {

namespace {

constexpr int kRun = 4;                   // neighbouring edges of a lane
constexpr int kStep = kRun * kWave;       // edges of a wave's step

struct EdgeWalk {
  const int64_t* crow;
  const int64_t* col;
  const int64_t* positions;  // null: node ids are positions
  const int32_t* short_positions;  // null, or the positions in 32 bits
  const int32_t* fits;             // [kFitBlocks] whether they all have room there
  int64_t n;
  int64_t nnz;
};

// Edges gather positions of 8 bytes; from some 500,000 nodes on these outgrow
// what an XCD's 4 MB L2 keeps beside the streams, and a copy in 32 bits pays where
// each is gathered a few times (4 heads, with and without it: 1M nodes of 16 edges
// 136 and 192 us, of 4 edges 55 and 57, of 2 edges 36 and 32; 400,000 of 16 53 and
// 54, 250,000 of 16 40 and 34).  Positions that do not fit are read as they are.
constexpr int kFitBlocks = 4 * kBlock;
inline bool shorten(int64_t n, int64_t nnz) { return n > (int64_t(1) << 19) && nnz >= 4 * n; }

__global__ __launch_bounds__(kBlock) void short_positions_kernel(const int64_t* __restrict__ positions,
                                                                 int32_t* __restrict__ out,
                                                                 int32_t* __restrict__ fits, int64_t n) {
  bool ok = true;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < n; i += kFitBlocks * kBlock) {
    const int64_t p = positions[i];
    out[i] = static_cast<int32_t>(p);
    ok = ok && p == static_cast<int32_t>(p);
  }
  ok = __syncthreads_and(ok);
  if (threadIdx.x == 0) fits[blockIdx.x] = ok;
}

// The rows of edges b + 4 lane .. + 3 of a step of a wave, where `row` is the
// row of edge b or one before it, and becomes that of edge b + 255.  Every row
// that begins inside the step leaves its number at its first edge; the row of an
// edge is the largest number at or in front of it.  mark: kStep words of LDS of
// this wave.  Ends at row n - 1 whatever crow holds.
__device__ __forceinline__ void step_rows(const EdgeWalk& w, int32_t* mark, int64_t b, int64_t& row, int (&rows)[kRun]) {
  const int lane = lane_id();
  *reinterpret_cast<int4*>(mark + kRun * lane) = make_int4(0, 0, 0, 0);
  __builtin_amdgcn_wave_barrier();
  for (int64_t r = row;; r += kWave) {
    const int64_t mine = r + 1 + lane;
    const int64_t first = (mine < w.n ? w.crow[mine] : INT64_MAX) - b;
    // a row that begins in front of the step still counts from its first edge on
    if (mine < w.n && first < kStep)
      __hip_atomic_fetch_max(mark + (first < 0 ? 0 : first), static_cast<int32_t>(mine - row), __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_WAVEFRONT);
    if (__any(mine >= w.n || first >= kStep)) break;
  }
  __builtin_amdgcn_wave_barrier();
  const int4 m = *reinterpret_cast<const int4*>(mark + kRun * lane);
  int own = m.x > m.y ? m.x : m.y;
  own = own > m.z ? own : m.z;
  own = own > m.w ? own : m.w;
  int before = own;  // the largest of lanes 0 .. lane
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int t = __shfl_up(before, o, kWave);
    if (lane >= o) before = t > before ? t : before;
  }
  const int base = static_cast<int>(row);
  const int last = uniform_i32(__builtin_amdgcn_readlane(before, 63));
  before = __shfl_up(before, 1, kWave);
  before = lane == 0 ? 0 : before;
  rows[0] = before > m.x ? before : m.x;
  rows[1] = rows[0] > m.y ? rows[0] : m.y;
  rows[2] = rows[1] > m.z ? rows[1] : m.z;
  rows[3] = rows[2] > m.w ? rows[2] : m.w;
#pragma unroll
  for (int i = 0; i < kRun; ++i) rows[i] += base;
  row += last;
}

// The buckets of edges b + 4 lane .. + 3, a byte each; those behind the last
// edge have any.  Ids outside the positions are clamped to them, so that a bad
// graph reads nothing out of bounds.
__device__ __forceinline__ uint32_t step_buckets(const EdgeWalk& w, bool fits, const int32_t* border,
                                                 const PositionMap& map, int32_t* mark, int64_t b, int64_t& row) {
  const int64_t at = b + kRun * lane_id();
  int64_t c[kRun];
  if (b + kStep <= w.nnz) {
    __builtin_memcpy(c, w.col + at, sizeof(c));
  } else {
#pragma unroll
    for (int i = 0; i < kRun; ++i) c[i] = w.col[at + i < w.nnz ? at + i : w.nnz - 1];
  }
  int rows[kRun];
  step_rows(w, mark, b, row, rows);
  int64_t rel[kRun];
  if (w.positions == nullptr) {
#pragma unroll
    for (int i = 0; i < kRun; ++i) rel[i] = c[i] - rows[i];
  } else {
#pragma unroll
    for (int i = 0; i < kRun; ++i) c[i] = c[i] < 0 ? 0 : (c[i] >= w.n ? w.n - 1 : c[i]);
    if (fits) {
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        rel[i] = static_cast<int64_t>(w.short_positions[c[i]]) - w.short_positions[rows[i]];
    } else {
#pragma unroll
      for (int i = 0; i < kRun; ++i) rel[i] = w.positions[c[i]] - w.positions[rows[i]];
    }
  }
  uint32_t packed = 0;
#pragma unroll
  for (int i = 0; i < kRun; ++i)
    packed |= static_cast<uint32_t>(bucket_of_relative(border, map, rel[i])) << (8 * i);
  return packed;
}

// Table entries that a workgroup keeps in LDS; larger tables are read from the caches.
constexpr int kTableWords = 8192;

// Four neighbouring elements as words, stored past the caches: the output is read
// again only by another kernel, and would push the positions out of the L2s.
template <typename T>
struct Four {
  T v[kRun];
};
template <int WORDS>
struct Words;
template <>
struct Words<2> {
  typedef uint32_t type __attribute__((ext_vector_type(2), aligned(2)));
};
template <>
struct Words<4> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4)));
};
template <typename T>
__device__ __forceinline__ void stream_four(T* to, const Four<T>& four) {
  using W = typename Words<sizeof(Four<T>) / 4>::type;
  W w;
  __builtin_memcpy(&w, &four, sizeof(w));
  __builtin_nontemporal_store(w, reinterpret_cast<W*>(to));
}

template <typename T, bool IN_LDS>
__global__ __launch_bounds__(kBlock) void position_bias_kernel(EdgeWalk w, PositionMap map,
                                                               const T* __restrict__ table, T* __restrict__ out,
                                                               uint32_t* __restrict__ found, int heads, int steps) {
  __shared__ int32_t border[kMaxBuckets + 1];
  __shared__ int32_t marks[kWavesPerBlock][kStep];
  __shared__ T entries[IN_LDS ? kTableWords : 1];  // [head][bucket]
  stage_borders(border, map);
  const int buckets = map.both_sides ? 2 * map.side : map.side;
  if constexpr (IN_LDS) {
    for (int i = threadIdx.x; i < buckets * heads; i += kBlock) {
      const int k = i / heads;
      entries[(i - k * heads) * buckets + k] = table[i];
    }
  }
  bool fits = false;
  if (w.short_positions != nullptr) {
    const int4 four = reinterpret_cast<const int4*>(w.fits)[threadIdx.x];
    fits = __syncthreads_and(four.x & four.y & four.z & four.w);
  } else {
    __syncthreads();
  }
  const int wave = uniform_i32(wave_in_block());
  int64_t b = (static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + wave) * steps * kStep;
  if (b >= w.nnz) return;
  int64_t row = uniform_i64(wave_row_of_edge(w.crow, w.n, b));
  for (int s = 0; s < steps && b < w.nnz; ++s, b += kStep) {
    const uint32_t k = step_buckets(w, fits, border, map, marks[wave], b, row);
    const int64_t at = b + kRun * lane_id();
    T* to = out + at;
    // the last word may end behind the edges
    if (found != nullptr && at < w.nnz) __builtin_nontemporal_store(k, found + at / kRun);
    const int left = at + kRun <= w.nnz ? kRun : (at < w.nnz ? static_cast<int>(w.nnz - at) : 0);
    for (int h = 0; h < heads; ++h, to += w.nnz) {
      Four<T> four;
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        const int bucket = (k >> (8 * i)) & 0xffu;
        four.v[i] = IN_LDS ? entries[h * buckets + bucket] : table[static_cast<int64_t>(bucket) * heads + h];
      }
      if (left == kRun) {
        stream_four(to, four);  // rows of heads begin at any element
      } else {
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          if (i < left) to[i] = four.v[i];
        }
      }
    }
  }
}

// ---- gradient -----------------------------------------------------------------
// Every thread keeps a sum of its own for each bucket, in a column of LDS
// (bucket-major: a wave's columns lie in different banks), so nothing is added
// atomically and the order of every sum is fixed: the same inputs give the same
// bits.  (Adding with LDS atomics, which would not wait for the sum to come
// back, takes 190 cycles a wave here: 365 us where this takes 77, for 16M edges
// and 4 heads.)  A thread reads the sums of its four neighbouring edges at once
// and puts edges of one bucket together in registers.  It adds at most
// kMaxSteps * 4 = 64 numbers in fp32; all sums above that are fp64.
constexpr int kMaxSteps = 16;

// LDS of 32 KB up to 128 buckets: five workgroups a CU.
inline int gradient_threads(int64_t buckets) { return buckets <= 32 ? 256 : (buckets <= 64 ? 128 : 64); }

struct GradientGrid {
  int threads;
  int steps;  // of every wave
  int64_t chunks;
};
// A workgroup sums one head of one chunk.  2,048 waves fill the chip before a
// wave takes a second step (a chunk's end costs as much as 16 steps).
inline GradientGrid gradient_grid(int64_t nnz, int64_t heads, int64_t buckets) {
  GradientGrid g;
  g.threads = gradient_threads(buckets);
  const int64_t all = (nnz + kStep - 1) / kStep * heads;
  const int64_t steps = all / 2048;
  g.steps = static_cast<int>(steps < 1 ? 1 : (steps > kMaxSteps ? kMaxSteps : steps));
  const int64_t edges = int64_t(g.threads) * kRun * g.steps;
  g.chunks = (nnz + edges - 1) / edges;
  return g;
}

// Adds four numbers to a thread's column of sums, in their order.
template <int THREADS>
__device__ __forceinline__ void add_four(float* column, uint32_t four, const float (&x)[kRun], uint32_t buckets) {
  uint32_t k[kRun];
  float sum[kRun];
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    k[i] = (four >> (8 * i)) & 0xffu;
    k[i] = (k[i] < buckets ? k[i] : buckets - 1) * THREADS;  // a bad bucket adds to the last one
    sum[i] = column[k[i]];
  }
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
#pragma unroll
    for (int j = 0; j < i; ++j) sum[i] = k[j] == k[i] ? sum[j] : sum[i];
    sum[i] += x[i];
    column[k[i]] = sum[i];
  }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void position_bias_grad_kernel(const uint32_t* __restrict__ found,
                                                                     const T* __restrict__ grad,
                                                                     double* __restrict__ partial, int64_t nnz,
                                                                     int64_t chunks, int heads, int buckets,
                                                                     int steps) {
  extern __shared__ float sums[];  // [buckets][THREADS]
  const int64_t chunk = blockIdx.x / static_cast<unsigned>(heads);
  const int h = static_cast<int>(blockIdx.x - chunk * heads);
  for (int k = 0; k < buckets; ++k) sums[k * THREADS + threadIdx.x] = 0.0f;
  const int wave = uniform_i32(wave_in_block());
  const int64_t first = (chunk * (THREADS / kWave) + wave) * static_cast<int64_t>(steps) * kStep;
  float* const column = sums + threadIdx.x;
  constexpr int kAhead = 4;  // steps whose loads are under way at once
  for (int s0 = 0; s0 < steps; s0 += kAhead) {
    const int64_t b = first + static_cast<int64_t>(s0) * kStep;
    const int64_t at = b + kRun * lane_id();
    const T* from = grad + h * nnz + at;
    if (s0 + kAhead <= steps && b + kAhead * kStep <= nnz) {
      uint32_t four[kAhead];
      RawVec<kRun * sizeof(T)> raw[kAhead];
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        four[s] = found[at / kRun + s * kWave];
        __builtin_memcpy(&raw[s], from + s * kStep, sizeof(raw[s]));
      }
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        float x[kRun];
#pragma unroll
        for (int i = 0; i < kRun; ++i) x[i] = Elem<T>::get(raw[s].w, i);
        add_four<THREADS>(column, four[s], x, buckets);
      }
    } else {
      for (int s = 0; s < kAhead && s0 + s < steps; ++s) {
        const int64_t mine = at + s * kStep;
        if (mine >= nnz) break;
        float x[kRun];
#pragma unroll
        for (int i = 0; i < kRun; ++i) x[i] = mine + i < nnz ? Elem<T>::at(from, s * kStep + i) : 0.0f;
        add_four<THREADS>(column, found[mine / kRun], x, buckets);
      }
    }
  }
  __syncthreads();
  // four threads a bucket sum its columns; each begins at another column, so that
  // the reads of a wave lie in different banks
  constexpr int kQuarter = THREADS / 4;
  for (int k = threadIdx.x >> 2; k < buckets; k += kQuarter) {
    const int part = threadIdx.x & 3;
    const float* const of = sums + k * THREADS + part * kQuarter;
    double s = 0.0;
    for (int j = 0; j < kQuarter; j += 16) {
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = of[(j + i + threadIdx.x) & (kQuarter - 1)];
#pragma unroll
      for (int i = 0; i < 16; ++i) s += x[i];
    }
    s += __shfl_xor(s, 1, 64);
    s += __shfl_xor(s, 2, 64);
    if (part == 0) partial[(static_cast<int64_t>(h) * buckets + k) * chunks + chunk] = s;
  }
}

// A wave per table entry sums the chunks, lane l those with index l mod 64.
template <typename T>
__global__ __launch_bounds__(kBlock) void position_bias_grad_join_kernel(const double* __restrict__ partial,
                                                                         T* __restrict__ grad_table, int64_t chunks,
                                                                         int heads, int buckets) {
  const int entry = blockIdx.x * kWavesPerBlock + wave_in_block();
  if (entry >= heads * buckets) return;
  const int h = entry / buckets;
  const int k = entry - h * buckets;
  const double* const of = partial + entry * chunks;
  double s = 0.0;
  int64_t c = lane_id();
  for (; c + 7 * kWave < chunks; c += 8 * kWave) {
    double x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = of[c + i * kWave];
#pragma unroll
    for (int i = 0; i < 8; ++i) s += x[i];
  }
  for (; c < chunks; c += kWave) s += of[c];
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane_id() == 0) Elem<T>::put(grad_table + static_cast<int64_t>(k) * heads + h, s);
}

int check_position_bias(const void* table, const void* edges, int64_t nnz, int64_t heads, int64_t buckets, int dtype) {
  if (dtype != AS_DTYPE_F32 && dtype != AS_DTYPE_BF16 && dtype != AS_DTYPE_F16)
    return fail(AS_ERR_INVALID_ARGUMENT, "dtype must be AS_DTYPE_F32, AS_DTYPE_BF16 or AS_DTYPE_F16");
  if (nnz < 0) return fail(AS_ERR_INVALID_ARGUMENT, "nnz must be non-negative");
  if (heads < 1 || heads > 65535) return fail(AS_ERR_INVALID_ARGUMENT, "heads must lie in [1, 65535]");
  if (buckets < 1 || buckets > kMaxBuckets)
    return fail(AS_ERR_INVALID_ARGUMENT, "the number of buckets must lie in [1, %d]", kMaxBuckets);
  if (table == nullptr) return fail(AS_ERR_INVALID_ARGUMENT, "null table pointer");
  if (nnz > 0 && edges == nullptr) return fail(AS_ERR_INVALID_ARGUMENT, "null pointer argument");
  // one launch, of fewer than 2^32 work-items
  if (nnz > kMaxBlocksPerLaunch * kStep) return fail(AS_ERR_UNSUPPORTED, "at most 2^30 edges");
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

size_t as_csr_position_bias_workspace_bytes(int64_t n, int64_t nnz, int positions) {
  if (!positions || n <= 0 || !shorten(n, nnz)) return 0;
  return sizeof(int32_t) * (kFitBlocks + static_cast<size_t>(n));
}

int as_csr_position_bias(const int64_t* crow, const int64_t* col, const int64_t* positions, const void* table,
                         void* out, uint8_t* found, int64_t n, int64_t nnz, int64_t heads, int64_t buckets,
                         const int32_t* borders, int both_sides, int dtype, void* workspace, size_t workspace_bytes,
                         void* stream) {
  clear_error();
  if (const int bad = check_position_bias(table, out, nnz, heads, buckets, dtype)) return bad;
  if (n < 0 || n > INT32_MAX) return fail(AS_ERR_INVALID_ARGUMENT, "N exceeds kernel index range");
  if (nnz > 0 && n == 0) return fail(AS_ERR_INVALID_ARGUMENT, "edges without rows");
  if (nnz > 0 && (crow == nullptr || col == nullptr)) return fail(AS_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (!aligned(found, 4)) return fail(AS_ERR_INVALID_ARGUMENT, "found must be 4-byte aligned");
  PositionMap map;
  if (const int bad = fill_position_map(&map, borders, buckets, both_sides)) return bad;
  const size_t need = as_csr_position_bias_workspace_bytes(n, nnz, positions != nullptr);
  if (workspace_bytes < need || (need > 0 && workspace == nullptr))
    return fail(AS_ERR_WORKSPACE, "the position bias needs %zu workspace bytes", need);
  if (!aligned(workspace, 16)) return fail(AS_ERR_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
  if (nnz == 0) return AS_OK;
  EdgeWalk walk{crow, col, positions, nullptr, nullptr, n, nnz};
  // a wave takes further steps (which spare it the search for its first row) from 8,192 waves on
  const int64_t all = (nnz + kStep - 1) / kStep;
  const int steps = static_cast<int>(all / 8192 < 1 ? 1 : (all / 8192 > 8 ? 8 : all / 8192));
  const int64_t per_block = int64_t(kStep) * steps * kWavesPerBlock;
  const dim3 grid(static_cast<unsigned>((nnz + per_block - 1) / per_block));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (positions != nullptr && shorten(n, nnz)) {
    int32_t* const fits = static_cast<int32_t*>(workspace);
    short_positions_kernel<<<kFitBlocks, kBlock, 0, s>>>(positions, fits + kFitBlocks, fits, n);
    if (const int bad = check_launch("csr_position_bias (positions)")) return bad;
    walk.fits = fits;
    walk.short_positions = fits + kFitBlocks;
  }
  uint32_t* const words = reinterpret_cast<uint32_t*>(found);
  return with_element(dtype, [&](auto e) {
    using T = decltype(e);
    if (buckets * heads <= kTableWords) {
      position_bias_kernel<T, true><<<grid, kBlock, 0, s>>>(
          walk, map, static_cast<const T*>(table), static_cast<T*>(out), words, static_cast<int>(heads), steps);
    } else {
      position_bias_kernel<T, false><<<grid, kBlock, 0, s>>>(
          walk, map, static_cast<const T*>(table), static_cast<T*>(out), words, static_cast<int>(heads), steps);
    }
    return check_launch("csr_position_bias");
  });
}

size_t as_csr_position_bias_backward_workspace_bytes(int64_t nnz, int64_t heads, int64_t buckets) {
  if (nnz <= 0 || heads <= 0 || buckets <= 0) return 8;
  return static_cast<size_t>(gradient_grid(nnz, heads, buckets).chunks) * heads * buckets * sizeof(double);
}

int as_csr_position_bias_backward(const uint8_t* found, const void* grad, void* grad_table, int64_t nnz,
                                  int64_t heads, int64_t buckets, int dtype, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  clear_error();
  if (const int bad = check_position_bias(grad_table, grad, nnz, heads, buckets, dtype)) return bad;
  if (nnz > 0 && found == nullptr) return fail(AS_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (!aligned(found, 4)) return fail(AS_ERR_INVALID_ARGUMENT, "found must be 4-byte aligned");
  const size_t need = as_csr_position_bias_backward_workspace_bytes(nnz, heads, buckets);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(AS_ERR_WORKSPACE, "the position bias gradient needs %zu workspace bytes", need);
  if (!aligned(workspace, 16)) return fail(AS_ERR_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
  const GradientGrid g = gradient_grid(nnz, heads, buckets);
  if (g.chunks * heads * g.threads > UINT32_MAX)
    return fail(AS_ERR_UNSUPPORTED, "too many edges and heads for one launch");
  double* partial = static_cast<double*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_element(dtype, [&](auto e) {
    using T = decltype(e);
    if (g.chunks > 0) {
      const dim3 grid(static_cast<unsigned>(g.chunks * heads));
      const size_t lds = static_cast<size_t>(buckets) * g.threads * sizeof(float);
      const auto* words = reinterpret_cast<const uint32_t*>(found);
      const auto* from = static_cast<const T*>(grad);
      const int h = static_cast<int>(heads);
      const int k = static_cast<int>(buckets);
      if (g.threads == 256) {
        position_bias_grad_kernel<T, 256><<<grid, 256, lds, s>>>(words, from, partial, nnz, g.chunks, h, k, g.steps);
      } else if (g.threads == 128) {
        position_bias_grad_kernel<T, 128><<<grid, 128, lds, s>>>(words, from, partial, nnz, g.chunks, h, k, g.steps);
      } else {
        position_bias_grad_kernel<T, 64><<<grid, 64, lds, s>>>(words, from, partial, nnz, g.chunks, h, k, g.steps);
      }
      if (const int bad = check_launch("csr_position_bias (backward)")) return bad;
    }
    const int64_t entries = heads * buckets;
    position_bias_grad_join_kernel<T>
        <<<dim3(static_cast<unsigned>((entries + kWavesPerBlock - 1) / kWavesPerBlock)), kBlock, 0, s>>>(
            partial, static_cast<T*>(grad_table), g.chunks, static_cast<int>(heads), static_cast<int>(buckets));
    return check_launch("csr_position_bias (backward join)");
  });
}

}  // extern "C"
