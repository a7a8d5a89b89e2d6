// Rows on their way to their experts and back.
//
//   a pair is (row r, its j-th expert e); pairs are ordered by expert, and within one as they come: place[r, j]
//   rows[place[r, j]] = x[r],  offsets[e] = pairs of experts below e;   grad_x[r] = sum_j grad_rows[place[r, j]]
//   out[r] = sum_j w[r, j] y[place[r, j]];   grad_y[place[r, j]] = w[r, j] g[r],  grad_w[r, j] = sum_d g[r, d] y[place[r, j], d]
//
// A pair without an expert (-1) is behind all others and its place is the complement of where: its row is zeros and counts for nothing.
// So every row of the pairs' matrix has one pair, is written once, and nothing is cleared first. All of it is moving rows: what is read
// and written once bounds it.
//
// The order is a counting sort, stable: blocks count the experts of their pairs (k_expert_counts), an expert's counts are summed up block by
// block (k_expert_sums), and each block finds its pairs' places from those, its warps' counts and the lanes below with the same expert
// (k_expert_places). Few pairs are one block's, which needs no other's counts.
#include "dense.cuh"

namespace apt {

constexpr int kPairWarps = 8, kPairThreads = kPairWarps * 32;
constexpr int kPairsALane = 4, kPairsABlock = kPairThreads * kPairsALane;

struct PairCall {
  const int64_t* experts;
  int64_t pairs;
  int num_experts;
  int blocks;
  int* counts;              // [num_experts + 1][blocks]: pairs of a block; behind k_expert_sums those of the blocks before
  int* totals;              // [num_experts + 1]
  int64_t *offsets, *place;
  int32_t* status;
};

// A lane's pairs: a warp has kPairsALane runs of 32 neighbouring ones. The class of a pair: its expert, or num_experts.
__device__ __forceinline__ int64_t pair_of(int i) {
  return (int64_t)blockIdx.x * kPairsABlock + (threadIdx.x / 32) * (32 * kPairsALane) + i * 32 + threadIdx.x % 32;
}
__device__ __forceinline__ void load_classes(const PairCall& c, int (&cls)[kPairsALane]) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPairsALane; ++i) {
    const int64_t p = pair_of(i), e = p < c.pairs ? c.experts[p] : -1;
    bad |= e < -1 || e >= c.num_experts;
    cls[i] = p >= c.pairs ? -1 : e < 0 || e >= c.num_experts ? c.num_experts : (int)e;
  }
  if (bad) atomicOr(c.status, APT_FLAG_ID_OUT_OF_RANGE);
}

__global__ void __launch_bounds__(kPairThreads) k_expert_counts(const __grid_constant__ PairCall c) {
  wait_for_previous();
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e <= c.num_experts; e += kPairThreads) hist[e] = 0;
  int cls[kPairsALane];
  load_classes(c, cls);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPairsALane; ++i) {
    const unsigned same = __match_any_sync(0xffffffffu, cls[i]);
    if (cls[i] >= 0 && __ffs(same) - 1 == (int)(threadIdx.x % 32)) atomicAdd(hist + cls[i], __popc(same));
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= c.num_experts; e += kPairThreads) c.counts[(int64_t)e * c.blocks + blockIdx.x] = hist[e];
}

// An expert's counts, block by block, become sums of those before; a block an expert.
__global__ void __launch_bounds__(kPairThreads) k_expert_sums(const __grid_constant__ PairCall c) {
  wait_for_previous();
  __shared__ int scan[33];
  int* const mine = c.counts + (int64_t)blockIdx.x * c.blocks;
  int before = 0;
  for (int b0 = 0; b0 < c.blocks; b0 += kPairThreads) {
    const int b = b0 + threadIdx.x, n = b < c.blocks ? mine[b] : 0;
    int total;
    const int at = block_exclusive_scan(n, scan, &total);
    if (b < c.blocks) mine[b] = before + at;
    before += total;
  }
  if (threadIdx.x == 0) c.totals[blockIdx.x] = before;
}

// ONE: this block has all pairs.
template <bool ONE>
__global__ void __launch_bounds__(kPairThreads) k_expert_places(const __grid_constant__ PairCall c) {
  wait_for_previous();
  extern __shared__ int at[];      // [kPairWarps][num_experts + 1]: a warp's pairs of a class, then the place of its next one
  __shared__ int scan[33];
  const int classes = c.num_experts + 1, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int i = threadIdx.x; i < kPairWarps * classes; i += kPairThreads) at[i] = 0;
  int cls[kPairsALane];
  load_classes(c, cls);
  __syncthreads();
  int* const mine = at + warp * classes;
  unsigned same[kPairsALane];
#pragma unroll
  for (int i = 0; i < kPairsALane; ++i) {
    same[i] = __match_any_sync(0xffffffffu, cls[i]);
    if (cls[i] >= 0 && __ffs(same[i]) - 1 == lane) mine[cls[i]] += __popc(same[i]);
    __syncwarp();
  }
  __syncthreads();
  int before = 0;
  for (int e0 = 0; e0 < classes; e0 += kPairThreads) {
    const int e = e0 + threadIdx.x;
    int n = 0, total;
    if (e < classes) {
      if (ONE)
        for (int w = 0; w < kPairWarps; ++w) n += at[w * classes + e];
      else
        n = c.totals[e];
    }
    const int first = before + block_exclusive_scan(n, scan, &total);
    before += total;
    if (e < classes) {
      if (blockIdx.x == 0) c.offsets[e] = first;
      int next = first + (ONE ? 0 : c.counts[(int64_t)e * c.blocks + blockIdx.x]);
      for (int w = 0; w < kPairWarps; ++w) {
        const int m = at[w * classes + e];
        at[w * classes + e] = next;
        next += m;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPairsALane; ++i) {
    if (cls[i] >= 0) {
      const int64_t p = mine[cls[i]] + __popc(same[i] & ((1u << lane) - 1));
      c.place[pair_of(i)] = cls[i] < c.num_experts ? p : -1 - p;
    }
    __syncwarp();
    if (cls[i] >= 0 && __ffs(same[i]) - 1 == lane) mine[cls[i]] += __popc(same[i]);
    __syncwarp();
  }
}

// ---- rows ------------------------------------------------------------------------------
// Slices of W of every row; a team of lanes has a row.
template <typename W>
__device__ __forceinline__ W no_bits() {
  W w;
  memset(&w, 0, sizeof(W));
  return w;
}
template <typename W>
__global__ void __launch_bounds__(256) k_expert_spread(const W* __restrict__ x, int64_t rows, int slices, int k, const int64_t* __restrict__ place, W* __restrict__ out,
                                                       int lanes) {
  wait_for_previous();
  const int lane = threadIdx.x & ((1 << lanes) - 1);
  const int64_t by = (int64_t)gridDim.x * (256 >> lanes);
  for (int64_t r = (int64_t)blockIdx.x * (256 >> lanes) + (threadIdx.x >> lanes); r < rows; r += by)
    for (int s = lane; s < slices; s += 1 << lanes) {
      const W v = x[r * slices + s];
      for (int j = 0; j < k; ++j) {
        const int64_t p = place[r * k + j];
        out[(p < 0 ? -1 - p : p) * slices + s] = p < 0 ? no_bits<W>() : v;
      }
    }
}

struct SumCall {
  const void* y;
  int64_t rows, dim, pairs;
  int k, lanes;                 // logarithm of a team's lanes
  const float* weights;         // null: ones
  const int64_t* place;
  const void* grad;
  void *out, *grad_y;
  float* grad_weights;
  int32_t* status;
};
// Where the pair's row is; -1: nowhere. *to: the row that is its own all the same, -1 where there is none.
__device__ __forceinline__ int64_t checked_place(const SumCall& c, int64_t p, int64_t* to) {
  *to = p < 0 ? -1 - p : p;
  if (*to >= c.pairs) {
    atomicOr(c.status, APT_FLAG_ID_OUT_OF_RANGE);
    *to = -1;
    return -1;
  }
  return p;
}

template <typename T, int VE>
__global__ void __launch_bounds__(256) k_expert_sum(const __grid_constant__ SumCall c) {
  wait_for_previous();
  const int lane = threadIdx.x & ((1 << c.lanes) - 1);
  const int64_t by = (int64_t)gridDim.x * (256 >> c.lanes);
  for (int64_t r = (int64_t)blockIdx.x * (256 >> c.lanes) + (threadIdx.x >> c.lanes); r < c.rows; r += by)
    for (int64_t d = lane * VE; d < c.dim; d += VE << c.lanes) {
      float sum[VE];
#pragma unroll
      for (int q = 0; q < VE; ++q) sum[q] = 0.0f;
      for (int j = 0; j < c.k; ++j) {
        int64_t to;
        const int64_t p = checked_place(c, c.place[r * c.k + j], &to);
        if (p < 0) continue;
        const float w = c.weights ? c.weights[r * c.k + j] : 1.0f;
        const Raw<T, VE> v = load_raw<T, VE>((const T*)c.y + p * c.dim + d);
#pragma unroll
        for (int q = 0; q < VE; ++q) sum[q] = fmaf(w, v.get(q), sum[q]);
      }
      store_all<T, VE>((T*)c.out + r * c.dim + d, sum);
    }
}

template <typename T, int VE>
__global__ void __launch_bounds__(256) k_expert_sum_backward(const __grid_constant__ SumCall c) {
  wait_for_previous();
  const int lane = threadIdx.x & ((1 << c.lanes) - 1);
  const int64_t by = (int64_t)gridDim.x * (256 >> c.lanes);
  const int64_t first = (int64_t)blockIdx.x * (256 >> c.lanes) + (threadIdx.x >> c.lanes);
  // (a warp's teams go round together: they add up across lanes)
  for (int64_t r0 = first - first % (32 >> c.lanes), r = first; r0 < c.rows; r0 += by, r += by)
    for (int j = 0; j < c.k; ++j) {
      int64_t to = -1;
      const int64_t p = r < c.rows ? checked_place(c, c.place[r * c.k + j], &to) : -1;
      const float w = p >= 0 ? c.weights[r * c.k + j] : 0.0f;
      float dot = 0.0f;
      if (to >= 0)
        for (int64_t d = lane * VE; d < c.dim; d += VE << c.lanes) {
          const Raw<T, VE> g = load_raw<T, VE>((const T*)c.grad + r * c.dim + d);
          float out[VE];
#pragma unroll
          for (int q = 0; q < VE; ++q) out[q] = p >= 0 ? w * g.get(q) : 0.0f;
          if (c.grad_weights && p >= 0) {
            const Raw<T, VE> v = load_raw<T, VE>((const T*)c.y + p * c.dim + d);
#pragma unroll
            for (int q = 0; q < VE; ++q) dot = fmaf(g.get(q), v.get(q), dot);
          }
          if (c.grad_y) store_all<T, VE>((T*)c.grad_y + to * c.dim + d, out);
        }
      if (c.grad_weights) {
        for (int o = 0; o < c.lanes; ++o) dot += __shfl_xor_sync(0xffffffffu, dot, 1 << o);
        if (lane == 0 && r < c.rows) c.grad_weights[r * c.k + j] = dot;
      }
    }
}

// ---- host side -------------------------------------------------------------------------
static int log2_lanes(int64_t slices) {
  int l = 0;
  while (l < 5 && (1 << l) < slices) ++l;
  return l;
}

template <bool ONE>
static int launch_places(const PairCall& c, cudaStream_t s) {
  const size_t shared = (size_t)kPairWarps * (c.num_experts + 1) * 4;
  static bool sized[64] = {};
  int dev = 0;
  APT_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !sized[dev]) {
    APT_CUDA(cudaFuncSetAttribute(k_expert_places<ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairWarps * (APT_GROUPED_LINEAR_MAX_GROUPS + 1) * 4));
    if (dev < 64) sized[dev] = true;
  }
  APT_FOLLOW((k_expert_places<ONE>), c.blocks, kPairThreads, shared, s, c);
  return APT_OK;
}
static int expert_places(const PairCall& c, cudaStream_t s) {
  if (c.blocks == 1) return launch_places<true>(c, s);
  APT_FOLLOW(k_expert_counts, c.blocks, kPairThreads, (size_t)(c.num_experts + 1) * 4, s, c);
  APT_FOLLOW(k_expert_sums, c.num_experts + 1, kPairThreads, 0, s, c);
  return launch_places<false>(c, s);
}

template <typename W>
static int spread(const void* x, int64_t rows, int64_t row_bytes, int k, const int64_t* place, void* out, cudaStream_t s) {
  const int64_t slices = row_bytes / (int64_t)sizeof(W);
  const int lanes = log2_lanes(slices);
  APT_FOLLOW((k_expert_spread<W>), wave_grid(ceil_div(rows, 256 >> lanes), 8), 256, 0, s, (const W*)x, rows, (int)slices, k, place, (W*)out, lanes);
  return APT_OK;
}

template <typename T, int VE>
static int launch_sum(SumCall c, bool backward, cudaStream_t s) {
  c.lanes = log2_lanes(ceil_div(c.dim, VE));
  const int grid = wave_grid(ceil_div(c.rows, 256 >> c.lanes), 8);
  if (backward)
    APT_FOLLOW((k_expert_sum_backward<T, VE>), grid, 256, 0, s, c);
  else
    APT_FOLLOW((k_expert_sum<T, VE>), grid, 256, 0, s, c);
  return APT_OK;
}
template <typename T>
static int sum(const SumCall& c, bool backward, cudaStream_t s) {
  const uint64_t bits = (uint64_t)(c.dim * sizeof(T)) | (uintptr_t)c.y | (uintptr_t)c.out | (uintptr_t)c.grad | (uintptr_t)c.grad_y;
  switch (slice_elems(bits, sizeof(T))) {
    case 1: return launch_sum<T, 1>(c, backward, s);
    case 2: return launch_sum<T, 2>(c, backward, s);
    case 4: return launch_sum<T, 4>(c, backward, s);
  }
  if constexpr (sizeof(T) == 2) return launch_sum<T, 8>(c, backward, s);
  return APT_OK;
}
static int sum_of(int dtype, const SumCall& c, bool backward, cudaStream_t s) {
  if (dtype == APT_F32) return sum<float>(c, backward, s);
  if (dtype == APT_BF16) return sum<__nv_bfloat16>(c, backward, s);
  return sum<__half>(c, backward, s);
}
static int sum_check(const char* who, int dtype, int64_t rows, int64_t dim, int64_t k) {
  APT_CHECK_ARG(dtype == APT_F32 || dtype == APT_BF16 || dtype == APT_F16, "%s: unsupported dtype %d", who, dtype);
  APT_CHECK_ARG(rows >= 0 && dim >= 1 && k >= 1 && k < 1ll << 31 && rows <= ((1ll << 31) - 1) / k, "%s: %lld rows of %lld, %lld experts each", who, (long long)rows,
                (long long)dim, (long long)k);
  return APT_OK;
}

}  // namespace apt

extern "C" size_t apt_expert_rows_workspace_bytes(int64_t pairs, int64_t experts) {
  if (pairs <= apt::kPairsABlock || experts <= 0) return 0;
  return (size_t)(experts + 1) * (size_t)(apt::ceil_div(pairs, apt::kPairsABlock) + 1) * 4;
}

extern "C" int apt_expert_rows(const void* x, int64_t rows, int64_t row_bytes, const int64_t* experts, int64_t k, int64_t num_experts, void* out,
                               int64_t* offsets, int64_t* place, void* workspace, size_t workspace_bytes, int32_t* status_word, void* stream) {
  using namespace apt;
  APT_CHECK_ARG(rows >= 0 && k >= 1 && k < 1ll << 31 && rows <= ((1ll << 31) - 1 - kPairsABlock) / k, "apt_expert_rows: %lld rows, %lld experts each", (long long)rows,
                (long long)k);
  APT_CHECK_ARG(num_experts >= 1 && num_experts <= APT_GROUPED_LINEAR_MAX_GROUPS, "apt_expert_rows: %lld experts (1 to %d are possible)",
                (long long)num_experts, APT_GROUPED_LINEAR_MAX_GROUPS);
  APT_CHECK_ARG(row_bytes >= 2 && row_bytes % 2 == 0 && row_bytes < 1ll << 31, "apt_expert_rows: rows of %lld bytes", (long long)row_bytes);
  APT_CHECK_ARG(offsets && (rows == 0 || (x && experts && out && place && status_word)), "apt_expert_rows: null buffer");
  const int64_t pairs = rows * k;
  APT_CHECK_ARG(workspace_bytes >= apt_expert_rows_workspace_bytes(pairs, num_experts) && (uintptr_t)workspace % 4 == 0, "apt_expert_rows: workspace too small");
  const cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {
    APT_CUDA(cudaMemsetAsync(offsets, 0, (size_t)(num_experts + 1) * 8, s));
    return APT_OK;
  }
  PairCall c = {};
  c.experts = experts, c.pairs = pairs, c.num_experts = (int)num_experts, c.blocks = (int)ceil_div(pairs, kPairsABlock);
  c.counts = (int*)workspace, c.totals = c.counts + (num_experts + 1) * (int64_t)c.blocks;
  c.offsets = offsets, c.place = place, c.status = status_word;
  if (const int e = expert_places(c, s)) return e;
  const uint64_t bits = (uint64_t)row_bytes | (uintptr_t)x | (uintptr_t)out;
  if (bits % 16 == 0) return spread<uint4>(x, rows, row_bytes, (int)k, place, out, s);
  if (bits % 8 == 0) return spread<uint2>(x, rows, row_bytes, (int)k, place, out, s);
  if (bits % 4 == 0) return spread<uint32_t>(x, rows, row_bytes, (int)k, place, out, s);
  return spread<uint16_t>(x, rows, row_bytes, (int)k, place, out, s);
}

extern "C" int apt_expert_sum(int dtype, const void* y, int64_t rows, int64_t dim, int64_t k, const float* weights, const int64_t* place, void* out,
                              int32_t* status_word, void* stream) {
  using namespace apt;
  if (const int e = sum_check("apt_expert_sum", dtype, rows, dim, k)) return e;
  APT_CHECK_ARG(rows == 0 || (y && place && out && status_word), "apt_expert_sum: null buffer");
  if (rows == 0) return APT_OK;
  SumCall c = {};
  c.y = y, c.rows = rows, c.dim = dim, c.pairs = rows * k, c.k = (int)k, c.weights = weights, c.place = place, c.out = out, c.status = status_word;
  return sum_of(dtype, c, false, (cudaStream_t)stream);
}

extern "C" int apt_expert_sum_backward(int dtype, const void* y, int64_t rows, int64_t dim, int64_t k, const float* weights, const int64_t* place,
                                       const void* grad_out, void* grad_y, float* grad_weights, int32_t* status_word, void* stream) {
  using namespace apt;
  if (const int e = sum_check("apt_expert_sum_backward", dtype, rows, dim, k)) return e;
  APT_CHECK_ARG(rows == 0 || (weights && place && grad_out && status_word && (y || !grad_weights)), "apt_expert_sum_backward: null buffer");
  if (rows == 0 || (!grad_y && !grad_weights)) return APT_OK;
  SumCall c = {};
  c.y = y, c.rows = rows, c.dim = dim, c.pairs = rows * k, c.k = (int)k, c.weights = weights, c.place = place;
  c.grad = grad_out, c.grad_y = grad_y, c.grad_weights = grad_weights, c.status = status_word;
  return sum_of(dtype, c, true, (cudaStream_t)stream);
}
