// Products of rows in ragged groups with the weights of their group.
//
//   out[r, n] = sum_k x[r, k] w[g, n, k] + b[g, n]      rows r of group g
//   dx[r, k]  = sum_n dy[r, n] w[g, n, k]
//   dw[g, n, k] = sum_{r in g} dy[r, n] x[r, k],   db[g, n] = sum_{r in g} dy[r, n]
//
// Where the groups end is on the device only: the grid is for the most tiles there can be, and a block finds its tile from the ends.
#include "dense.cuh"

namespace apt {

constexpr int kTile = 64, kStep = 16;

// The group and the first row of row tile `tile`, counted group by group; tiles behind the last group's are those of the rows that
// belong to none (group == groups). False: there is no such tile.
__device__ __forceinline__ bool find_tile(const int64_t* offsets, int groups, int64_t rows, int64_t tile, int* group, RowRange* range) {
  for (int g = 0; g <= groups; ++g) {
    RowRange r = {0, rows};
    if (g < groups) r = group_rows(offsets, g, rows);
    else r.begin = min(max(offsets[groups], (int64_t)0), rows);
    const int64_t n = (r.end - r.begin + kTile - 1) / kTile;
    if (tile < n) {
      *group = g;
      *range = {r.begin + tile * kTile, min(r.begin + (tile + 1) * kTile, r.end)};
      return true;
    }
    tile -= n;
  }
  return false;
}

// acc += A[m, k] B[n, k] over one tile; a thread has 4 x 4 of 64 x 64.
template <typename T>
__device__ __forceinline__ void tile_product(const T* a, int64_t am, int64_t ak, int64_t num_m, const T* b, int64_t bn, int64_t bk, int64_t num_n,
                                             int64_t num_k, float (&acc)[4][4]) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const int tm = threadIdx.x / 16, tn = threadIdx.x % 16;
  for (int64_t k0 = 0; k0 < num_k; k0 += kStep) {
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
      // the contiguous one of the two indices moves fastest
      const int m = ak == 1 ? i / kStep : i % kTile, k = ak == 1 ? i % kStep : i / kTile;
      sa[k][m] = m < num_m && k0 + k < num_k ? Elem<T>::to_f(a[m * am + (k0 + k) * ak]) : 0.0f;
      const int n = bk == 1 ? i / kStep : i % kTile, l = bk == 1 ? i % kStep : i / kTile;
      sb[l][n] = n < num_n && k0 + l < num_k ? Elem<T>::to_f(b[n * bn + (k0 + l) * bk]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k) {
      float u[4], v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = sa[k][tm + 16 * i], v[i] = sb[k][tn + 16 * i];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(u[i], v[j], acc[i][j]);
    }
  }
}

// Rows against weights: out (w by its rows) or dx (w by its columns).
template <typename T>
__global__ void __launch_bounds__(256)
k_rows_product(const T* __restrict__ in, int64_t rows, int64_t num_k, const T* __restrict__ w, int64_t wn, int64_t wk, int64_t num_n, const T* bias,
               const int64_t* __restrict__ offsets, int groups, T* __restrict__ out, int32_t* status) {
  wait_for_previous();
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int g = threadIdx.x; g < groups; g += 256)
      if (bad_group(offsets, g, rows)) atomicOr(status, APT_FLAG_BAD_OFFSETS);
  int g;
  RowRange r;
  if (!find_tile(offsets, groups, rows, blockIdx.x, &g, &r)) return;
  const int64_t n0 = (int64_t)blockIdx.y * kTile, here = min((int64_t)kTile, num_n - n0);
  float acc[4][4] = {};
  if (g < groups)
    tile_product(in + r.begin * num_k, num_k, (int64_t)1, r.end - r.begin, w + (int64_t)g * num_n * num_k + n0 * wn, wn, wk, here, num_k, acc);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = r.begin + threadIdx.x / 16 + 16 * i, n = n0 + threadIdx.x % 16 + 16 * j;
      if (m < r.end && n < num_n) out[m * num_n + n] = Elem<T>::from_f(acc[i][j] + (bias && g < groups ? Elem<T>::to_f(bias[g * num_n + n]) : 0.0f));
    }
}

// dw of one group and tile.
template <typename T>
__global__ void __launch_bounds__(256)
k_weight_product(const T* __restrict__ x, int64_t rows, int64_t dim, const T* __restrict__ grad, int64_t out_dim, const int64_t* __restrict__ offsets,
                 T* __restrict__ grad_weight) {
  wait_for_previous();
  const int g = blockIdx.z;
  const RowRange r = group_rows(offsets, g, rows);
  const int64_t n0 = (int64_t)blockIdx.x * kTile, k0 = (int64_t)blockIdx.y * kTile;
  float acc[4][4] = {};
  tile_product(grad + r.begin * out_dim + n0, (int64_t)1, out_dim, min((int64_t)kTile, out_dim - n0), x + r.begin * dim + k0, (int64_t)1, dim,
               min((int64_t)kTile, dim - k0), r.end - r.begin, acc);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + threadIdx.x / 16 + 16 * i, k = k0 + threadIdx.x % 16 + 16 * j;
      if (n < out_dim && k < dim) grad_weight[((int64_t)g * out_dim + n) * dim + k] = Elem<T>::from_f(acc[i][j]);
    }
}

template <typename T>
__global__ void __launch_bounds__(256)
k_bias_sums(const T* __restrict__ grad, int64_t rows, int64_t out_dim, const int64_t* __restrict__ offsets, int groups, T* __restrict__ grad_bias,
            int32_t* status) {
  wait_for_previous();
  __shared__ float part[8][33];
  const int g = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (threadIdx.x == 0 && blockIdx.x == 0 && bad_group(offsets, g, rows)) atomicOr(status, APT_FLAG_BAD_OFFSETS);
  const RowRange r = group_rows(offsets, g, rows);
  const int64_t n = (int64_t)blockIdx.x * 32 + lane;
  float sum = 0.0f;
  if (n < out_dim)
    for (int64_t row = r.begin + warp; row < r.end; row += 8) sum += Elem<T>::to_f(grad[row * out_dim + n]);
  part[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && n < out_dim) {
    for (int k = 1; k < 8; ++k) sum += part[k][lane];
    grad_bias[g * out_dim + n] = Elem<T>::from_f(sum);
  }
}

template <typename T>
static int linear_forward(const void* x, int64_t rows, int64_t dim, const void* weight, const void* bias, int64_t out_dim, const int64_t* offsets, int groups,
                          void* out, int32_t* status, cudaStream_t s) {
  const dim3 grid((unsigned)(ceil_div(rows, kTile) + groups + 1), (unsigned)ceil_div(out_dim, kTile));
  APT_FOLLOW((k_rows_product<T>), grid, 256, 0, s, (const T*)x, rows, dim, (const T*)weight, dim, (int64_t)1, out_dim, (const T*)bias, offsets, groups,
             (T*)out, status);
  return APT_OK;
}
template <typename T>
static int linear_backward(const void* x, int64_t rows, int64_t dim, const void* weight, int64_t out_dim, const int64_t* offsets, int groups,
                           const void* grad, void* grad_x, void* grad_weight, void* grad_bias, int32_t* status, cudaStream_t s) {
  if (grad_x && rows) {
    const dim3 grid((unsigned)(ceil_div(rows, kTile) + groups + 1), (unsigned)ceil_div(dim, kTile));
    APT_FOLLOW((k_rows_product<T>), grid, 256, 0, s, (const T*)grad, rows, out_dim, (const T*)weight, (int64_t)1, dim, dim, (const T*)nullptr, offsets, groups,
               (T*)grad_x, status);
  }
  if (grad_weight) {
    const dim3 grid((unsigned)ceil_div(out_dim, kTile), (unsigned)ceil_div(dim, kTile), (unsigned)groups);
    APT_FOLLOW((k_weight_product<T>), grid, 256, 0, s, (const T*)x, rows, dim, (const T*)grad, out_dim, offsets, (T*)grad_weight);
  }
  if (grad_bias) {
    const dim3 grid((unsigned)ceil_div(out_dim, 32), (unsigned)groups);
    APT_FOLLOW((k_bias_sums<T>), grid, 256, 0, s, (const T*)grad, rows, out_dim, offsets, groups, (T*)grad_bias, status);
  }
  return APT_OK;
}

static int linear_check(const char* who, int dtype, int64_t rows, int64_t dim, int64_t out_dim, int64_t groups) {
  APT_CHECK_ARG(dtype == APT_F32 || dtype == APT_BF16 || dtype == APT_F16, "%s: unsupported dtype %d", who, dtype);
  APT_CHECK_ARG(rows >= 0 && rows < (1ll << 31) - (1 << 20) && dim > 0 && out_dim > 0 && dim <= APT_GROUPED_LINEAR_MAX_DIM && out_dim <= APT_GROUPED_LINEAR_MAX_DIM,
                "%s: %lld rows of %lld by %lld", who, (long long)rows, (long long)dim, (long long)out_dim);
  APT_CHECK_ARG(groups > 0 && groups <= APT_GROUPED_LINEAR_MAX_GROUPS, "%s: %lld groups (1 to %d are possible)", who, (long long)groups,
                APT_GROUPED_LINEAR_MAX_GROUPS);
  return APT_OK;
}

}  // namespace apt

extern "C" size_t apt_grouped_linear_workspace_bytes(int dtype, int64_t rows, int64_t dim, int64_t out_dim, int64_t groups, int backward) {
  return 0;
}

extern "C" int apt_grouped_linear_forward(int dtype, const void* x, int64_t rows, int64_t dim, const void* weight, const void* bias, int64_t out_dim,
                                          const int64_t* offsets, int64_t groups, void* out, void* workspace, size_t workspace_bytes,
                                          int32_t* status_word, void* stream) {
  using namespace apt;
  if (const int e = linear_check("apt_grouped_linear_forward", dtype, rows, dim, out_dim, groups)) return e;
  if (rows == 0) return APT_OK;
  APT_CHECK_ARG(x && weight && offsets && out && status_word, "apt_grouped_linear_forward: null buffer");
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == APT_F32) return linear_forward<float>(x, rows, dim, weight, bias, out_dim, offsets, (int)groups, out, status_word, s);
  if (dtype == APT_BF16) return linear_forward<__nv_bfloat16>(x, rows, dim, weight, bias, out_dim, offsets, (int)groups, out, status_word, s);
  return linear_forward<__half>(x, rows, dim, weight, bias, out_dim, offsets, (int)groups, out, status_word, s);
}

extern "C" int apt_grouped_linear_backward(int dtype, const void* x, int64_t rows, int64_t dim, const void* weight, int64_t out_dim,
                                           const int64_t* offsets, int64_t groups, const void* grad_out, void* grad_x, void* grad_weight,
                                           void* grad_bias, void* workspace, size_t workspace_bytes, int32_t* status_word, void* stream) {
  using namespace apt;
  if (const int e = linear_check("apt_grouped_linear_backward", dtype, rows, dim, out_dim, groups)) return e;
  APT_CHECK_ARG(offsets && status_word && (rows == 0 || grad_out) && (!grad_x || rows == 0 || weight) && (!grad_weight || rows == 0 || x),
                "apt_grouped_linear_backward: null buffer");
  const cudaStream_t s = (cudaStream_t)stream;
  const int g = (int)groups;
  if (dtype == APT_F32) return linear_backward<float>(x, rows, dim, weight, out_dim, offsets, g, grad_out, grad_x, grad_weight, grad_bias, status_word, s);
  if (dtype == APT_BF16)
    return linear_backward<__nv_bfloat16>(x, rows, dim, weight, out_dim, offsets, g, grad_out, grad_x, grad_weight, grad_bias, status_word, s);
  return linear_backward<__half>(x, rows, dim, weight, out_dim, offsets, g, grad_out, grad_x, grad_weight, grad_bias, status_word, s);
}
