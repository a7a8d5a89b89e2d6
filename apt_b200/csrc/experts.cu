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
#include <algorithm>

#include "dense.cuh"

namespace apt {

// One block that has all pairs is larger than one of many.
template <bool ONE>
struct PairBlock {
  static constexpr int kWarps = ONE ? 16 : 8, kThreads = 32 * kWarps, kALane = ONE ? 8 : 4, kPairs = kThreads * kALane;
};
constexpr int64_t kMostPairs = (1ll << 31) - 1 - PairBlock<false>::kPairs;      // counts, and the steps of loops beyond the last pair, are numbers of 32 bits
constexpr int kMostOfOne = 1024;      // experts that a larger block has counts for

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

// A lane's pairs: a warp has kALane runs of 32 neighbouring ones. The class of a pair: its expert, or num_experts.
template <bool ONE>
__device__ __forceinline__ int64_t pair_of(int i) {
  using B = PairBlock<ONE>;
  return (int64_t)blockIdx.x * B::kPairs + (threadIdx.x / 32) * (32 * B::kALane) + i * 32 + threadIdx.x % 32;
}
template <bool ONE>
__device__ __forceinline__ void load_classes(const PairCall& c, int (&cls)[PairBlock<ONE>::kALane]) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < PairBlock<ONE>::kALane; ++i) {
    const int64_t p = pair_of<ONE>(i), e = p < c.pairs ? c.experts[p] : -1;
    bad |= e < -1 || e >= c.num_experts;
    cls[i] = p >= c.pairs ? -1 : e < 0 || e >= c.num_experts ? c.num_experts : (int)e;
  }
  if (bad) atomicOr(c.status, APT_FLAG_ID_OUT_OF_RANGE);
}

__global__ void __launch_bounds__(PairBlock<false>::kThreads) k_expert_counts(const __grid_constant__ PairCall c) {
  wait_for_previous();
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e <= c.num_experts; e += PairBlock<false>::kThreads) hist[e] = 0;
  int cls[PairBlock<false>::kALane];
  load_classes<false>(c, cls);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PairBlock<false>::kALane; ++i) {
    const unsigned same = __match_any_sync(0xffffffffu, cls[i]);
    if (cls[i] >= 0 && __ffs(same) - 1 == (int)(threadIdx.x % 32)) atomicAdd(hist + cls[i], __popc(same));
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= c.num_experts; e += PairBlock<false>::kThreads) c.counts[(int64_t)e * c.blocks + blockIdx.x] = hist[e];
}

// An expert's counts, block by block, become sums of those before; a block an expert.
__global__ void __launch_bounds__(256) k_expert_sums(const __grid_constant__ PairCall c) {
  wait_for_previous();
  __shared__ int scan[33];
  int* const mine = c.counts + (int64_t)blockIdx.x * c.blocks;
  int before = 0;
  for (int b0 = 0; b0 < c.blocks; b0 += 256) {
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
__global__ void __launch_bounds__(PairBlock<ONE>::kThreads) k_expert_places(const __grid_constant__ PairCall c) {
  wait_for_previous();
  using B = PairBlock<ONE>;
  extern __shared__ int at[];      // [B::kWarps][num_experts + 1]: a warp's pairs of a class, then the place of its next one
  __shared__ int scan[33];
  const int classes = c.num_experts + 1, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int i = threadIdx.x; i < B::kWarps * classes; i += B::kThreads) at[i] = 0;
  int cls[B::kALane];
  load_classes<ONE>(c, cls);
  __syncthreads();
  int* const mine = at + warp * classes;
  unsigned same[B::kALane];
#pragma unroll
  for (int i = 0; i < B::kALane; ++i) {
    same[i] = __match_any_sync(0xffffffffu, cls[i]);
    if (cls[i] >= 0 && __ffs(same[i]) - 1 == lane) mine[cls[i]] += __popc(same[i]);
    __syncwarp();
  }
  __syncthreads();
  int before = 0;
  for (int e0 = 0; e0 < classes; e0 += B::kThreads) {
    const int e = e0 + threadIdx.x;
    int n = 0, total;
    if (e < classes) {
      if (ONE)
        for (int w = 0; w < B::kWarps; ++w) n += at[w * classes + e];
      else
        n = c.totals[e];
    }
    const int first = before + block_exclusive_scan(n, scan, &total);
    before += total;
    if (e < classes) {
      if (blockIdx.x == 0) c.offsets[e] = first;
      int next = first + (ONE ? 0 : c.counts[(int64_t)e * c.blocks + blockIdx.x]);
      for (int w = 0; w < B::kWarps; ++w) {
        const int m = at[w * classes + e];
        at[w * classes + e] = next;
        next += m;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < B::kALane; ++i) {
    if (cls[i] >= 0) {
      const int64_t p = mine[cls[i]] + __popc(same[i] & ((1u << lane) - 1));
      c.place[pair_of<ONE>(i)] = cls[i] < c.num_experts ? p : -1 - p;
    }
    __syncwarp();
    if (cls[i] >= 0 && __ffs(same[i]) - 1 == lane) mine[cls[i]] += __popc(same[i]);
    __syncwarp();
  }
}

// ---- rows ------------------------------------------------------------------------------
// A team of lanes has a row: at most a warp's, or a block's where few rows leave the GPU empty. A lane has 16 bytes of it at once: where rows are no whole 16-byte slices, as several narrower ones, each beside the other
// lanes' (100000 x 255 bf16, three experts each, with the gradient: one narrow slice at once 280 us, these 138; 256 wide: 96).
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
  constexpr int D = 16 / sizeof(W);
  const int lane = threadIdx.x & ((1 << lanes) - 1);
  const int64_t by = (int64_t)gridDim.x * (256 >> lanes);
  for (int64_t r = (int64_t)blockIdx.x * (256 >> lanes) + (threadIdx.x >> lanes); r < rows; r += by)
    for (int s0 = lane; s0 < slices; s0 += D << lanes) {
      W v[D];
#pragma unroll
      for (int i = 0; i < D; ++i)
        if (s0 + (i << lanes) < slices) v[i] = x[r * slices + s0 + (i << lanes)];
      for (int j = 0; j < k; ++j) {
        const int64_t p = place[r * k + j];
        W* const to = out + (p < 0 ? -1 - p : p) * slices + s0;
#pragma unroll
        for (int i = 0; i < D; ++i)
          if (s0 + (i << lanes) < slices) to[i << lanes] = p < 0 ? no_bits<W>() : v[i];
      }
    }
}

struct SumCall {
  const void* y;                // backward: null where the weights' gradient is not wanted
  int64_t rows, pairs;
  int dim, k, lanes;            // lanes: logarithm of a team's
  const float* weights;         // null: ones
  const int64_t* place;
  const void* grad;
  void *out, *grad_y;
  float* grad_weights;
  int32_t* status;
};
// U of a row's pairs, all of whose rows are on their way at once; more of them cost registers, and with them rows on their way. Places beyond the
// pairs are flagged and count for nothing.
constexpr int kNowhere = INT32_MIN;
template <int U>
struct Pairs {
  int at[U];      // the pair's row; -1 - that: the pair has no expert; kNowhere: there is none
  float weight[U];
};
template <int U>
__device__ __forceinline__ Pairs<U> load_pairs(const SumCall& c, int64_t r, int j0) {
  Pairs<U> p;
  bool bad = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool there = r < c.rows && j0 + u < c.k;
    const int64_t at = there ? c.place[r * c.k + j0 + u] : kNowhere;
    p.weight[u] = there && c.weights ? c.weights[r * c.k + j0 + u] : 1.0f;
    const bool known = at >= -c.pairs && at < c.pairs;
    bad |= there && !known;
    p.at[u] = known ? (int)at : kNowhere;
  }
  if (bad) atomicOr(c.status, APT_FLAG_ID_OUT_OF_RANGE);
  return p;
}

// A slice that is read once: not kept in L1.
template <typename T, int VE>
__device__ __forceinline__ Raw<T, VE> load_once(const T* p) {
  if constexpr (sizeof(T) * VE == 16) {
    const uint4 u = ld_stream_16(p);
    Raw<T, VE> r;
    r.w[0] = u.x, r.w[1] = u.y, r.w[2] = u.z, r.w[3] = u.w;
    return r;
  } else {
    return load_raw<T, VE>(p);
  }
}

// 151552 rows of 256 bf16, two of 16 experts: 47 us with weights or without (HBM: 36); four pairs at once of two rows 49 and 51, the next row's
// places asked for a row ahead, which spilled, 78.
template <typename T, int VE, int U>
__global__ void __launch_bounds__(256, U == 4 ? 5 : 6) k_expert_sum(const __grid_constant__ SumCall c) {
  wait_for_previous();
  constexpr int D = 16 / (int)sizeof(T) / VE;
  const T* __restrict__ const y = (const T*)c.y;
  T* __restrict__ const out = (T*)c.out;
  const int lane = threadIdx.x & ((1 << c.lanes) - 1), apart = VE << c.lanes;
  const int64_t by = (int64_t)gridDim.x * (256 >> c.lanes);
  for (int64_t r = (int64_t)blockIdx.x * (256 >> c.lanes) + (threadIdx.x >> c.lanes); r < c.rows; r += by)
    for (int d0 = lane * VE; d0 < c.dim; d0 += D * apart) {
      float sum[D][VE];
#pragma unroll
      for (int i = 0; i < D; ++i)
#pragma unroll
        for (int q = 0; q < VE; ++q) sum[i][q] = 0.0f;
      for (int j0 = 0; j0 < c.k; j0 += U) {
        const Pairs<U> p = load_pairs<U>(c, r, j0);
        Raw<T, VE> v[U][D];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < D; ++i)
            if (p.at[u] >= 0 && d0 + i * apart < c.dim) v[u][i] = load_once<T, VE>(y + (int64_t)p.at[u] * c.dim + d0 + i * apart);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (p.at[u] >= 0)
#pragma unroll
            for (int i = 0; i < D; ++i)
#pragma unroll
              for (int q = 0; q < VE; ++q) sum[i][q] = fmaf(p.weight[u], v[u][i].get(q), sum[i][q]);
      }
#pragma unroll
      for (int i = 0; i < D; ++i)
        if (d0 + i * apart < c.dim) store_all<T, VE>(out + r * c.dim + d0 + i * apart, sum[i]);
    }
}

// The same rows: 80 us (HBM: 59). A team has at most a warp, or all of a block.
template <typename T, int VE, int U>
__global__ void __launch_bounds__(256, U == 4 || VE == 1 ? 4 : 5) k_expert_sum_backward(const __grid_constant__ SumCall c) {
  wait_for_previous();
  constexpr int D = 16 / (int)sizeof(T) / VE;
  __shared__ float parts[8][U];
  const T *__restrict__ const y = (const T*)c.y, *__restrict__ const grad = (const T*)c.grad;
  T* __restrict__ const grad_y = (T*)c.grad_y;
  const int lane = threadIdx.x & ((1 << c.lanes) - 1), apart = VE << c.lanes;
  const int64_t by = (int64_t)gridDim.x * (256 >> c.lanes);
  int64_t r = (int64_t)blockIdx.x * (256 >> c.lanes) + (threadIdx.x >> c.lanes);
  // (a warp's teams go round together: they add up across lanes)
  for (int64_t first = r - (threadIdx.x % 32 >> c.lanes); first < c.rows; first += by, r += by)
    for (int j0 = 0; j0 < c.k; j0 += U) {
      const Pairs<U> p = load_pairs<U>(c, r, j0);
      float dot[U] = {};
      if (r < c.rows)
        for (int d0 = lane * VE; d0 < c.dim; d0 += D * apart) {
          Raw<T, VE> g[D], v[U][D];
#pragma unroll
          for (int i = 0; i < D; ++i)
            if (d0 + i * apart < c.dim) g[i] = load_raw<T, VE>(grad + r * c.dim + d0 + i * apart);
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < D; ++i)
              if (p.at[u] >= 0 && y && d0 + i * apart < c.dim) v[u][i] = load_once<T, VE>(y + (int64_t)p.at[u] * c.dim + d0 + i * apart);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (p.at[u] == kNowhere) continue;
            if (grad_y) {
              T* const to = grad_y + (int64_t)(p.at[u] >= 0 ? p.at[u] : -1 - p.at[u]) * c.dim + d0;
#pragma unroll
              for (int i = 0; i < D; ++i) {
                float out[VE];
#pragma unroll
                for (int q = 0; q < VE; ++q) out[q] = p.at[u] >= 0 ? p.weight[u] * g[i].get(q) : 0.0f;
                if (d0 + i * apart < c.dim) store_all<T, VE>(to + i * apart, out);
              }
            }
            if (p.at[u] >= 0 && y)
#pragma unroll
              for (int i = 0; i < D; ++i)
                if (d0 + i * apart < c.dim)
#pragma unroll
                  for (int q = 0; q < VE; ++q) dot[u] = fmaf(g[i].get(q), v[u][i].get(q), dot[u]);
          }
        }
      if (y) {
        for (int o = 0; o < min(c.lanes, 5); ++o)
#pragma unroll
          for (int u = 0; u < U; ++u) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], 1 << o);
        if (c.lanes > 5) {
          __syncthreads();
          if (lane % 32 == 0)
#pragma unroll
            for (int u = 0; u < U; ++u) parts[lane / 32][u] = dot[u];
          __syncthreads();
          if (lane == 0)
            for (int w = 1; w < 8; ++w)
#pragma unroll
              for (int u = 0; u < U; ++u) dot[u] += parts[w][u];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (lane == 0 && r < c.rows && j0 + u < c.k) c.grad_weights[r * c.k + j0 + u] = dot[u];
      }
    }
}

// ---- host side -------------------------------------------------------------------------
// Lanes for a row of so many slices: a warp's, and up to a block's while all rows' would be a quarter of what the SMs hold. One row of 8192 bf16, eight
// experts: rows 30 -> 13 us, sums 72 -> 15, their gradients 72 -> 16.
static int log2_lanes(int64_t slices, int64_t rows) {
  int l = 0;
  while (l < 8 && (1 << l) < slices && (l < 5 || rows << l < kNumSMs * 512)) ++l;
  return l;
}

static bool one_block(int64_t pairs, int64_t experts) { return pairs <= (experts <= kMostOfOne ? PairBlock<true>::kPairs : 0); }
template <bool ONE>
static int launch_places(const PairCall& c, cudaStream_t s) {
  using B = PairBlock<ONE>;
  const int most = B::kWarps * ((ONE ? kMostOfOne : APT_GROUPED_LINEAR_MAX_GROUPS) + 1) * 4;
  static bool sized[64] = {};
  int dev = 0;
  APT_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !sized[dev]) {
    APT_CUDA(cudaFuncSetAttribute(k_expert_places<ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    if (dev < 64) sized[dev] = true;
  }
  APT_FOLLOW((k_expert_places<ONE>), c.blocks, B::kThreads, (size_t)B::kWarps * (c.num_experts + 1) * 4, s, c);
  return APT_OK;
}
static int expert_places(PairCall c, cudaStream_t s) {
  c.blocks = one_block(c.pairs, c.num_experts) ? 1 : (int)ceil_div(c.pairs, PairBlock<false>::kPairs);
  c.totals = c.counts + (c.num_experts + 1) * (int64_t)c.blocks;
  if (one_block(c.pairs, c.num_experts)) return launch_places<true>(c, s);
  APT_FOLLOW(k_expert_counts, c.blocks, PairBlock<false>::kThreads, (size_t)(c.num_experts + 1) * 4, s, c);
  APT_FOLLOW(k_expert_sums, c.num_experts + 1, 256, 0, s, c);
  return launch_places<false>(c, s);
}

template <typename W>
static int spread(const void* x, int64_t rows, int64_t row_bytes, int k, const int64_t* place, void* out, cudaStream_t s) {
  const int64_t slices = row_bytes / (int64_t)sizeof(W);
  const int lanes = log2_lanes(ceil_div(row_bytes, 16), rows);
  APT_FOLLOW((k_expert_spread<W>), wave_grid(ceil_div(rows, 256 >> lanes), 8), 256, 0, s, (const W*)x, rows, (int)slices, k, place, (W*)out, lanes);
  return APT_OK;
}

template <typename T, int VE, int U>
static int launch_pairs(const SumCall& c, bool backward, cudaStream_t s) {
  const int grid = wave_grid(ceil_div(c.rows, 256 >> c.lanes), 8);
  if (backward)
    APT_FOLLOW((k_expert_sum_backward<T, VE, U>), grid, 256, 0, s, c);
  else
    APT_FOLLOW((k_expert_sum<T, VE, U>), grid, 256, 0, s, c);
  return APT_OK;
}
template <typename T, int VE>
static int launch_sum(SumCall c, bool backward, cudaStream_t s) {
  c.lanes = log2_lanes(ceil_div(c.dim, 16 / (int)sizeof(T)), c.rows);
  if (backward) c.lanes = c.lanes > 6 ? 8 : std::min(c.lanes, 5);
  // pairs at once: eight slices of a lane are on their way at the most (narrow ones take as many registers as wide ones)
  constexpr int kMost = VE * (int)sizeof(T) / 2 < 4 ? VE * (int)sizeof(T) / 2 : 4;
  if constexpr (kMost >= 4)
    if (c.k > 2) return launch_pairs<T, VE, 4>(c, backward, s);
  if constexpr (kMost >= 2)
    if (c.k > 1) return launch_pairs<T, VE, 2>(c, backward, s);
  return launch_pairs<T, VE, 1>(c, backward, s);
}
template <typename T>
static int sum(const SumCall& c, bool backward, cudaStream_t s) {
  const uint64_t bits = (uint64_t)c.dim * sizeof(T) | (uintptr_t)c.y | (uintptr_t)c.out | (uintptr_t)c.grad | (uintptr_t)c.grad_y;
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
  APT_CHECK_ARG(rows >= 0 && dim >= 1 && dim < 1ll << 30 && k >= 1 && k < 1ll << 31 && rows <= kMostPairs / k, "%s: %lld rows of %lld, %lld experts each", who, (long long)rows,
                (long long)dim, (long long)k);
  return APT_OK;
}

}  // namespace apt

extern "C" size_t apt_expert_rows_workspace_bytes(int64_t pairs, int64_t experts) {
  if (pairs <= 0 || experts <= 0 || apt::one_block(pairs, experts)) return 0;
  return (size_t)(experts + 1) * (size_t)(apt::ceil_div(pairs, apt::PairBlock<false>::kPairs) + 1) * 4;
}

extern "C" int apt_expert_rows(const void* x, int64_t rows, int64_t row_bytes, const int64_t* experts, int64_t k, int64_t num_experts, void* out,
                               int64_t* offsets, int64_t* place, void* workspace, size_t workspace_bytes, int32_t* status_word, void* stream) {
  using namespace apt;
  APT_CHECK_ARG(rows >= 0 && k >= 1 && k < 1ll << 31 && rows <= kMostPairs / k, "apt_expert_rows: %lld rows, %lld experts each", (long long)rows,
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
  c.experts = experts, c.pairs = pairs, c.num_experts = (int)num_experts, c.counts = (int*)workspace;
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
  c.y = y, c.rows = rows, c.dim = (int)dim, c.pairs = rows * k, c.k = (int)k, c.weights = weights, c.place = place, c.out = out, c.status = status_word;
  return sum_of(dtype, c, false, (cudaStream_t)stream);
}

extern "C" int apt_expert_sum_backward(int dtype, const void* y, int64_t rows, int64_t dim, int64_t k, const float* weights, const int64_t* place,
                                       const void* grad_out, void* grad_y, float* grad_weights, int32_t* status_word, void* stream) {
  using namespace apt;
  if (const int e = sum_check("apt_expert_sum_backward", dtype, rows, dim, k)) return e;
  APT_CHECK_ARG(rows == 0 || (weights && place && grad_out && status_word && (y || !grad_weights)), "apt_expert_sum_backward: null buffer");
  if (rows == 0 || (!grad_y && !grad_weights)) return APT_OK;
  SumCall c = {};
  c.y = grad_weights ? y : nullptr, c.rows = rows, c.dim = (int)dim, c.pairs = rows * k, c.k = (int)k, c.weights = weights, c.place = place;
  c.grad = grad_out, c.grad_y = grad_y, c.grad_weights = grad_weights, c.status = status_word;
  return sum_of(dtype, c, true, (cudaStream_t)stream);
}
