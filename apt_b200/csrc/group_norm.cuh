// Group norm with an activation and dropout behind it, channels last.
//
// A segment of rows (each row, equal blocks of rows, or ragged groups) and a group of neighbouring channels have one mean and one
// variance. xh = (x - mean) rstd, z = xh gamma + beta, y = drop(act(z)); backwards dz = drop(dy) act'(z), dgamma = sum dz xh,
// dbeta = sum dz, and with dxh = dz gamma: dx = rstd (dxh - mean(dxh) - xh mean(dxh xh)).
// Everything is held in 32 bits. A variance is taken around its mean, over numbers that are in registers, or by running means that are
// joined by their counts, so that a mean far from zero costs nothing.
//
// Rows by themselves (k_norm_rows): a group of a row is a run of numbers that a few lanes hold; read once, written once, forwards and
// backwards (statistics are made again rather than kept).
// Segments: one whose rows a block's registers can hold is done by one block in one go (k_norm_first); of longer ones that kernel
// makes the sums of tiles of rows, and k_norm_second joins them and does the rest. Which segments are which only the device knows, so
// both kernels run always and look.
// Groups too wide for either: k_norm_wide_*, a block a segment and group, by walks over memory.
#pragma once

#include <algorithm>

#include "dense.cuh"

namespace apt {

struct NormShape {
  int64_t rows, dim, segments, per_segment;      // per_segment: rows of each where there are no offsets
  const int64_t* offsets;
  int groups, per;                               // channels of a group
};
struct NormCall {
  const void *x, *grad, *weight, *bias;          // grad: null in the forward
  void *out, *grad_weight, *grad_bias;           // out: y, or the gradient of x
  float2* stats;
  float eps;
  int act, wide_params;                          // wide_params: weight and bias are fp32 whatever x is
  bool drop;
  Drop d;
  int32_t* status;
  float* columns;                                // [blocks][2][dim] sums for dgamma and dbeta
  float2* parts;                                 // of the pieces of segments
};

__device__ __forceinline__ RowRange segment_rows(const NormShape& s, int64_t k) {
  if (s.offsets) return group_rows(s.offsets, (int)k, s.rows);
  return {k * s.per_segment, (k + 1) * s.per_segment};
}
// The first segment that ends behind the row.
__device__ __forceinline__ int64_t segment_at(const NormShape& s, int64_t row) {
  if (!s.offsets) return row / s.per_segment;
  int64_t lo = 0, hi = s.segments;
  while (lo < hi) {
    const int64_t m = (lo + hi) / 2;
    if (s.offsets[m + 1] <= row) lo = m + 1; else hi = m;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ float param(const void* p, int wide, int64_t c, float otherwise) {
  if (!p) return otherwise;
  return wide ? ((const float*)p)[c] : Elem<T>::to_f(((const T*)p)[c]);
}
template <typename T>
__device__ __forceinline__ void put_param(void* p, int wide, int64_t c, float v) {
  if (!p) return;
  if (wide) ((float*)p)[c] = v; else ((T*)p)[c] = Elem<T>::from_f(v);
}

template <int N>
__device__ __forceinline__ void act_all(int act, float (&z)[N]) {
  switch (act) {
    case APT_ACT_RELU:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = act_of<APT_ACT_RELU>(z[k]);
      break;
    case APT_ACT_SILU:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = act_of<APT_ACT_SILU>(z[k]);
      break;
    case APT_ACT_GELU:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = act_of<APT_ACT_GELU>(z[k]);
      break;
  }
}
template <int N>
__device__ __forceinline__ void slope_all(int act, float (&z)[N]) {
  switch (act) {
    case APT_ACT_RELU:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = act_slope<APT_ACT_RELU>(z[k]);
      break;
    case APT_ACT_SILU:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = act_slope<APT_ACT_SILU>(z[k]);
      break;
    case APT_ACT_GELU:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = act_slope<APT_ACT_GELU>(z[k]);
      break;
    default:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = 1.0f;
  }
}
// The elements from e on, dropout behind them.
template <int N>
__device__ __forceinline__ void drop_all(const Drop& d, int64_t e, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
      const Philox4 w = drop_words(d, (e >> 2) + q);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[4 * q + k] = dropped(d, w.w[k], v[4 * q + k]);
    }
  } else {      // one or two elements of a quad
    const Philox4 w = drop_words(d, e >> 2);
    const int at = (int)(e & 3);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = dropped(d, at + k == 0 ? w.w[0] : at + k == 1 ? w.w[1] : at + k == 2 ? w.w[2] : w.w[3], v[k]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_all(T* p, const float (&v)[N]) {
  Pack<T, N> r;
#pragma unroll
  for (int k = 0; k < N; ++k) r.v[k] = Elem<T>::from_f(v[k]);
  store_pack<T, N>(p, r);
}

// y of normalised elements, in place.
template <int N>
__device__ __forceinline__ void finish_forward(const NormCall& c, int64_t e, float (&v)[N], const float (&gamma)[N], const float (&beta)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = fmaf(v[k], gamma[k], beta[k]);
  act_all(c.act, v);
  if (c.drop) drop_all(c.d, e, v);
}
// dz of normalised elements and gradients, into the gradients.
template <int N>
__device__ __forceinline__ void begin_backward(const NormCall& c, int64_t e, const float (&xh)[N], float (&grad)[N], const float (&gamma)[N], const float (&beta)[N]) {
  float z[N];
#pragma unroll
  for (int k = 0; k < N; ++k) z[k] = fmaf(xh[k], gamma[k], beta[k]);
  slope_all(c.act, z);
  if (c.drop) drop_all(c.d, e, grad);
#pragma unroll
  for (int k = 0; k < N; ++k) grad[k] *= z[k];
}

// ------------------------------------------------------------------------------------------ rows by themselves
struct NormLanes {
  int width;              // lanes of a row's group: a power of two up to 32, or 256
  int groups, rows;       // a block has side by side
};

// A sum over the lanes of each group, of U rows at once.
template <bool BLOCK, int U>
__device__ __forceinline__ void sum_lanes(float (&v)[U], int width, float (*shared)[U]) {
#pragma unroll
  for (int u = 0; u < U; ++u)
    for (int o = (BLOCK ? 32 : width) / 2; o; o >>= 1) v[u] += __shfl_xor_sync(0xffffffffu, v[u], o);
  if constexpr (BLOCK) {
    __syncthreads();
    if (threadIdx.x % 32 == 0)
#pragma unroll
      for (int u = 0; u < U; ++u) shared[threadIdx.x / 32][u] = v[u];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) v[u] += shared[k][u];
    }
  }
}

// NV slices of VE elements a lane, U rows on their way.
template <typename T, int VE, int NV, int U, bool BLOCK, bool BACK>
__global__ void __launch_bounds__(256)
k_norm_rows(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c, const __grid_constant__ NormLanes l) {
  wait_for_previous();
  __shared__ float shared[8][U];
  __shared__ float sums[BACK ? 256 * VE : 1];
  const int width = BLOCK ? 256 : l.width;
  const int lane = threadIdx.x % width, slot = threadIdx.x / width % l.groups, line = threadIdx.x / (width * l.groups), g = blockIdx.y * l.groups + slot;
  const bool mine = line < l.rows && g < s.groups;
  const T* const x = (const T*)c.x;
  const T* const grad = (const T*)c.grad;
  T* const out = (T*)c.out;
  int at[NV];
  bool in[NV];
  float gamma[NV][VE], beta[NV][VE], dgamma[NV][VE], dbeta[NV][VE];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int k0 = (lane + j * width) * VE;
    in[j] = mine && k0 < s.per;
    at[j] = g * s.per + k0;
#pragma unroll
    for (int k = 0; k < VE; ++k) {
      gamma[j][k] = in[j] ? param<T>(c.weight, c.wide_params, at[j] + k, 1.0f) : 0.0f;
      beta[j][k] = in[j] ? param<T>(c.bias, c.wide_params, at[j] + k, 0.0f) : 0.0f;
      dgamma[j][k] = dbeta[j][k] = 0.0f;
    }
  }
  const float inv = 1.0f / (float)s.per;
  const int64_t step = (int64_t)l.rows * U;
  for (int64_t base = blockIdx.x * step; base < s.rows; base += gridDim.x * step) {
    Raw<T, VE> rx[U][NV], rg[BACK ? U : 1][NV];
    int64_t row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      row[u] = base + u * l.rows + line;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (in[j] && row[u] < s.rows) {
          rx[u][j] = load_raw<T, VE>(x + row[u] * s.dim + at[j]);
          if constexpr (BACK) rg[u][j] = load_raw<T, VE>(grad + row[u] * s.dim + at[j]);
        } else {
          rx[u][j] = Raw<T, VE>{};
          if constexpr (BACK) rg[u][j] = Raw<T, VE>{};
        }
      }
    }
    float mean[U], rstd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mean[u] = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VE; ++k) mean[u] += rx[u][j].get(k);
    }
    sum_lanes<BLOCK, U>(mean, width, shared);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mean[u] *= inv;
      rstd[u] = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          const float d = rx[u][j].get(k) - mean[u];
          rstd[u] += in[j] ? d * d : 0.0f;
        }
    }
    sum_lanes<BLOCK, U>(rstd, width, shared);
#pragma unroll
    for (int u = 0; u < U; ++u) rstd[u] = rsqrtf(rstd[u] * inv + c.eps);
    if constexpr (!BACK) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (row[u] >= s.rows) continue;
        if (c.stats && mine && lane == 0) c.stats[row[u] * s.groups + g] = make_float2(mean[u], rstd[u]);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (!in[j]) continue;
          float v[VE];
#pragma unroll
          for (int k = 0; k < VE; ++k) v[k] = (rx[u][j].get(k) - mean[u]) * rstd[u];
          const int64_t e = row[u] * s.dim + at[j];
          finish_forward(c, e, v, gamma[j], beta[j]);
          store_all<T, VE>(out + e, v);
        }
      }
    } else {
      float a[U], b[U], dz[U][NV][VE];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        a[u] = b[u] = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float xh[VE];
#pragma unroll
          for (int k = 0; k < VE; ++k) xh[k] = (rx[u][j].get(k) - mean[u]) * rstd[u], dz[u][j][k] = rg[u][j].get(k);
          begin_backward(c, row[u] * s.dim + at[j], xh, dz[u][j], gamma[j], beta[j]);
          if (!in[j] || row[u] >= s.rows) continue;
#pragma unroll
          for (int k = 0; k < VE; ++k) {
            const float v = dz[u][j][k], dxh = __fmul_rn(v, gamma[j][k]);
            dgamma[j][k] = fmaf(v, xh[k], dgamma[j][k]);
            dbeta[j][k] += v;
            dz[u][j][k] = dxh;
            a[u] += dxh;
            b[u] = fmaf(dxh, xh[k], b[u]);
          }
        }
      }
      sum_lanes<BLOCK, U>(a, width, shared);
      sum_lanes<BLOCK, U>(b, width, shared);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (row[u] >= s.rows) continue;
        a[u] *= inv, b[u] *= inv;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (!in[j]) continue;
          float v[VE];
#pragma unroll
          for (int k = 0; k < VE; ++k) v[k] = rstd[u] * (dz[u][j][k] - a[u] - (rx[u][j].get(k) - mean[u]) * rstd[u] * b[u]);
          store_all<T, VE>(out + row[u] * s.dim + at[j], v);
        }
      }
    }
  }
  if constexpr (BACK) {
    if (!c.columns) return;
    // the block's rows of each channel added up
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < VE; ++k) sums[threadIdx.x * VE + k] = which ? dbeta[j][k] : dgamma[j][k];
        __syncthreads();
        if (line == 0 && in[j]) {
#pragma unroll
          for (int k = 0; k < VE; ++k) {
            float v = 0.0f;
            for (int r = 0; r < l.rows; ++r) v += sums[(threadIdx.x + r * width * l.groups) * VE + k];
            c.columns[((int64_t)blockIdx.x * 2 + which) * s.dim + at[j] + k] = v;
          }
        }
      }
  }
}

// dgamma and dbeta of 32 channels from the blocks' sums, in the blocks' order.
template <typename T>
__device__ __forceinline__ void join_columns(const NormShape& s, const NormCall& c, int64_t block, int64_t blocks) {
  __shared__ float part[8][33];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t col = block * 32 + lane, all = 2 * s.dim;
  float v = 0.0f;
  if (col < all) {
    int64_t r = warp;
    for (; r + 56 < blocks; r += 64) {
      float u[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = c.columns[(r + 8 * k) * all + col];
#pragma unroll
      for (int k = 0; k < 8; ++k) v += u[k];
    }
    for (; r < blocks; r += 8) v += c.columns[r * all + col];
  }
  part[warp][lane] = v;
  __syncthreads();
  if (warp || col >= all) return;
  v = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) v += part[k][lane];
  put_param<T>(col < s.dim ? c.grad_weight : c.grad_bias, c.wide_params, col < s.dim ? col : col - s.dim, v);
}
template <typename T>
__global__ void __launch_bounds__(256) k_norm_columns(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c, int64_t blocks) {
  wait_for_previous();
  join_columns<T>(s, c, blockIdx.x, blocks);
}

// ------------------------------------------------------------------------------------------------- segments
constexpr int kMostColumns = 2048;      // of a block: 8 a thread
constexpr int kMostGroups = 512;        // of a block

// A thread has NC slices of VE neighbouring channels of every `lines`-th row. Up to 32 threads side by side are lanes of one warp.
struct NormTiles {
  int64_t tile, tiles;      // rows of a tile, how many
  int short_blocks;         // behind the tiles' blocks: whole segments
  int chunk;                // groups of a block
  int slots, lines;         // threads side by side in a row, rows side by side
  int cap;                  // rows of the segments that are done whole
};

// GN: groups that a slice may have channels of (1 where a group is whole slices).
template <int VE, int NC, int GN>
struct NormThread {
  int slot, line, group0, groups, per, col0;
  bool mine;
  bool in[NC];
  int col[NC];
  uint16_t group[NC][GN];        // within the block's
  __device__ __forceinline__ NormThread(const NormShape& s, const NormTiles& t) {
    if (t.slots <= 32) {
      const int lane = threadIdx.x % 32, per_warp = 32 / t.slots;
      slot = lane % t.slots, line = threadIdx.x / 32 * per_warp + lane / t.slots;
      mine = lane < per_warp * t.slots;
    } else {
      slot = threadIdx.x % t.slots, line = threadIdx.x / t.slots;
      mine = line < t.lines;
    }
    group0 = blockIdx.y * t.chunk, groups = min(t.chunk, s.groups - group0), per = s.per, col0 = group0 * s.per;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int k = (slot + j * t.slots) * VE;
      in[j] = mine && k < groups * per;
      col[j] = col0 + k;
#pragma unroll
      for (int i = 0; i < GN; ++i) group[j][i] = in[j] ? (uint16_t)((k + i) / per) : 0;
    }
  }
};

// Sums of K numbers over the rows and each group from per-thread sums a channel, into result[group][k]; by all threads of a block, or of
// a warp with shared memory of its own.
template <int VE, int NC, int GN, int K, bool WARP>
__device__ __forceinline__ void sum_groups(const float (&v)[K][NC][VE], float* room, float* result, const NormThread<VE, NC, GN>& me, int slots, int lines, int line) {
  // a slice of one group is one number
  constexpr int kOwn = GN == 1 ? 1 : VE;
  const int columns = slots * NC * kOwn, pitch = columns + 1, per = GN == 1 ? me.per / VE : me.per, lane = threadIdx.x % 32;
  const auto sync = [] {
    if (WARP) __syncwarp(); else __syncthreads();
  };
#pragma unroll
  for (int k = 0; k < K; ++k) {
    sync();
    if (me.mine)
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        if constexpr (kOwn == 1) {
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < VE; ++i) sum += v[k][j][i];
          room[line * pitch + me.slot + j * slots] = sum;
        } else {
#pragma unroll
          for (int i = 0; i < VE; ++i) room[line * pitch + (me.slot + j * slots) * VE + i] = v[k][j][i];
        }
      }
    sync();
    if (WARP && me.groups > 8) {
      for (int g = lane; g < me.groups; g += 32) {
        float sum = 0.0f;
        for (int r = 0; r < lines; ++r)
          for (int i = 0; i < per; ++i) sum += room[r * pitch + g * per + i];
        result[g * K + k] = sum;
      }
    } else {
      for (int g = WARP ? 0 : threadIdx.x / 32; g < me.groups; g += WARP ? 1 : 8) {
        float sum = 0.0f;
        if (per >= 32)
          for (int r = 0; r < lines; ++r)
            for (int i = lane; i < per; i += 32) sum += room[r * pitch + g * per + i];
        else if (per == 1 || lines >= 32)
          for (int r = lane; r < lines; r += 32)
            for (int i = 0; i < per; ++i) sum += room[r * pitch + g * per + i];
        else
          for (int i = lane; i < lines * per; i += 32) sum += room[i / per * pitch + g * per + i % per];
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) result[g * K + k] = sum;
      }
    }
  }
  sync();
}

// (v - mean) / deviation of a slice.
template <int VE, int GN>
__device__ __forceinline__ void normalise(float (&v)[VE], const float2 (&st)[GN]) {
#pragma unroll
  for (int i = 0; i < VE; ++i) v[i] = (v[i] - st[i % GN].x) * st[i % GN].y;
}
// dx of a slice: v is xh and becomes dx.
template <int VE, int GN>
__device__ __forceinline__ void finish_backward(float (&v)[VE], const float (&dxh)[VE], const float2 (&st)[GN], const float2 (&means)[GN]) {
#pragma unroll
  for (int i = 0; i < VE; ++i) v[i] = st[i % GN].y * (dxh[i] - means[i % GN].x - v[i] * means[i % GN].y);
}

template <typename T, int VE, int NC, int GN>
__device__ __forceinline__ void load_params(const NormCall& c, const NormThread<VE, NC, GN>& me, float (&gamma)[NC][VE], float (&beta)[NC][VE]) {
#pragma unroll
  for (int j = 0; j < NC; ++j)
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      gamma[j][i] = me.in[j] ? param<T>(c.weight, c.wide_params, me.col[j] + i, 1.0f) : 0.0f;
      beta[j][i] = me.in[j] ? param<T>(c.bias, c.wide_params, me.col[j] + i, 0.0f) : 0.0f;
    }
}
template <int VE, int NC, int GN>
__device__ __forceinline__ void load_stats(const NormShape& s, const NormCall& c, const NormThread<VE, NC, GN>& me, int64_t seg, float2 (&st)[NC][GN]) {
#pragma unroll
  for (int j = 0; j < NC; ++j)
#pragma unroll
    for (int i = 0; i < GN; ++i) st[j][i] = c.stats[seg * s.groups + me.group0 + me.group[j][i]];
}

// A block's sums of dgamma and dbeta to its line of c.columns.
template <int VE, int NC, int GN>
__device__ __forceinline__ void put_columns(const NormShape& s, const NormCall& c, const NormTiles& t, const NormThread<VE, NC, GN>& me, float* room,
                                            const float (&dgamma)[NC][VE], const float (&dbeta)[NC][VE]) {
  const int pitch = t.slots * NC * VE;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
    if (me.mine)
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) room[me.line * pitch + (me.slot + j * t.slots) * VE + i] = which ? dbeta[j][i] : dgamma[j][i];
    __syncthreads();
    for (int k = threadIdx.x; k < me.groups * me.per; k += 256) {
      float v = 0.0f;
      for (int l = 0; l < t.lines; ++l) v += room[l * pitch + k];
      c.columns[((int64_t)blockIdx.x * 2 + which) * s.dim + me.col0 + k] = v;
    }
  }
}

// Sums of a tile's rows of long segments, piece by piece: piece number tile + segment, which no other has. Forwards mean and squares around
// it, backwards the sums of dxh and dxh xh. Bound by HBM: 151552 x 256 bf16 in 8 segments, 8 groups of channels a slice.
template <typename T, int VE, int NC, int GN, bool BACK>
__device__ __forceinline__ void tile_sums(const NormShape& s, const NormCall& c, const NormTiles& t, float* room, float* result) {
  const NormThread<VE, NC, GN> me(s, t);
  const T* const x = (const T*)c.x;
  const T* const grad = (const T*)c.grad;
  float gamma[BACK ? NC : 1][VE], beta[BACK ? NC : 1][VE], dgamma[BACK ? NC : 1][VE], dbeta[BACK ? NC : 1][VE];
  if constexpr (BACK) {
    load_params<T>(c, me, gamma, beta);
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < VE; ++i) dgamma[j][i] = dbeta[j][i] = 0.0f;
  }
  const int64_t row0 = blockIdx.x * t.tile, row1 = min(row0 + t.tile, s.rows);
  for (int64_t seg = segment_at(s, row0); seg < s.segments; ++seg) {
    const RowRange whole = segment_rows(s, seg);
    if (whole.begin >= row1) break;
    const int64_t b = max(whole.begin, row0), e = min(whole.end, row1);
    if (whole.end - whole.begin <= t.cap || e <= b) continue;
    float2* const parts = c.parts + (blockIdx.x + seg) * s.groups + me.group0;
    if constexpr (!BACK) {
      float v[1][NC][VE], q[NC][VE];
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) v[0][j][i] = q[j][i] = 0.0f;
      float n = 0.0f;
      for (int64_t r0 = b + me.line; r0 < e; r0 += 4 * t.lines) {
        Raw<T, VE> raw[4][NC];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && r0 + u * t.lines < e) raw[u][j] = load_raw<T, VE>(x + (r0 + u * t.lines) * s.dim + me.col[j]);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (!me.mine || r0 + u * t.lines >= e) break;
          n += 1.0f;
          const float share = __fdividef(1.0f, n);
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j])
#pragma unroll
              for (int i = 0; i < VE; ++i) {
                const float y = raw[u][j].get(i), d = y - v[0][j][i];
                v[0][j][i] = fmaf(d, share, v[0][j][i]);
                q[j][i] = fmaf(d, y - v[0][j][i], q[j][i]);
              }
        }
      }
      // the piece's mean, then the squares around it
      float own[1][NC][VE];
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) own[0][j][i] = me.in[j] ? v[0][j][i] * n : 0.0f;
      sum_groups<VE, NC, GN, 1, false>(own, room, result, me, t.slots, t.lines, me.line);
      const float count = (float)(e - b) * (float)me.per;
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float d = v[0][j][i] - result[me.group[j][i % GN]] / count;
          own[0][j][i] = me.in[j] ? fmaf(n * d, d, q[j][i]) : 0.0f;
        }
      sum_groups<VE, NC, GN, 1, false>(own, room, result + kMostGroups, me, t.slots, t.lines, me.line);
      for (int g = threadIdx.x; g < me.groups; g += 256) parts[g] = make_float2(result[g] / count, result[kMostGroups + g]);
    } else {
      float2 st[NC][GN];
      load_stats(s, c, me, seg, st);
      float ab[2][NC][VE];
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) ab[0][j][i] = ab[1][j][i] = 0.0f;
      for (int64_t r0 = b + me.line; r0 < e; r0 += 2 * t.lines) {
        Raw<T, VE> rx[2][NC], rg[2][NC];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && r0 + u * t.lines < e) {
              rx[u][j] = load_raw<T, VE>(x + (r0 + u * t.lines) * s.dim + me.col[j]);
              rg[u][j] = load_raw<T, VE>(grad + (r0 + u * t.lines) * s.dim + me.col[j]);
            }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (r0 + u * t.lines >= e) break;
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            if (!me.in[j]) continue;
            float xh[VE], dz[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) xh[i] = rx[u][j].get(i), dz[i] = rg[u][j].get(i);
            normalise(xh, st[j]);
            begin_backward(c, (r0 + u * t.lines) * s.dim + me.col[j], xh, dz, gamma[j], beta[j]);
#pragma unroll
            for (int i = 0; i < VE; ++i) ab[0][j][i] += dz[i], ab[1][j][i] = fmaf(dz[i], xh[i], ab[1][j][i]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          dbeta[j][i] += ab[0][j][i], dgamma[j][i] += ab[1][j][i];
          ab[0][j][i] *= gamma[j][i], ab[1][j][i] *= gamma[j][i];
        }
      sum_groups<VE, NC, GN, 2, false>(ab, room, result, me, t.slots, t.lines, me.line);
      for (int g = threadIdx.x; g < me.groups; g += 256) parts[g] = make_float2(result[2 * g], result[2 * g + 1]);
    }
    __syncthreads();      // `result` is the next piece's
  }
  if constexpr (BACK)
    if (c.columns) put_columns(s, c, t, me, room, dgamma, dbeta);
}

// Whole segments, each by a block or a warp: rows in registers, in chunks where they are more (which are read again then, from L1).
// A warp has eight chunks at most: 55001 x 64 f16 in 2048 segments, whose blocks of 256 threads were 86 us of latency backwards.
constexpr int kWarpChunks = 8;
constexpr int held_rows(bool back, int nc) { return (back ? 2 : 8) / nc > 0 ? (back ? 2 : 8) / nc : 1; }
template <typename T, int VE, int NC, int GN, bool BACK, bool WARP>
__device__ __forceinline__ void short_segments(const NormShape& s, const NormCall& c, const NormTiles& t, float* room, float* result) {
  constexpr int kHeld = held_rows(BACK, NC), kTeams = WARP ? 8 : 1;
  const NormThread<VE, NC, GN> me(s, t);
  const int lines = t.lines / kTeams, line = me.line % lines, warp = threadIdx.x / 32, tid = WARP ? threadIdx.x % 32 : threadIdx.x, team = WARP ? 32 : 256;
  float* const my_room = WARP ? room + warp * (32 * NC * VE + 32) : room;
  float* const sums = WARP ? result + warp * 512 : result;      // 256 columns are 256 groups at most
  float* const squares = WARP ? sums + 256 : sums + kMostGroups;
  const T* const x = (const T*)c.x;
  const T* const grad = (const T*)c.grad;
  T* const out = (T*)c.out;
  float gamma[NC][VE], beta[NC][VE], dgamma[NC][VE], dbeta[NC][VE];
  load_params<T>(c, me, gamma, beta);
#pragma unroll
  for (int j = 0; j < NC; ++j)
#pragma unroll
    for (int i = 0; i < VE; ++i) dgamma[j][i] = dbeta[j][i] = 0.0f;
  const int64_t first = (int64_t)(blockIdx.x - t.tiles) * kTeams + (WARP ? warp : 0);
  for (int64_t seg = first; seg < s.segments; seg += (int64_t)t.short_blocks * kTeams) {
    const RowRange r = segment_rows(s, seg);
    const int rows = (int)min(r.end - r.begin, (int64_t)t.cap + 1);
    if (rows > t.cap || rows == 0) continue;
    const int chunks = (rows + kHeld * lines - 1) / (kHeld * lines);
    const float inv = 1.0f / ((float)rows * (float)me.per);
    Raw<T, VE> rx[kHeld][NC], rg[BACK ? kHeld : 1][NC];
    const auto row_of = [&](int chunk, int u) { return (chunk * kHeld + u) * lines + line; };
    const auto load = [&](int chunk, bool both) {
#pragma unroll
      for (int u = 0; u < kHeld; ++u)
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (me.in[j] && row_of(chunk, u) < rows) {
            rx[u][j] = load_raw<T, VE>(x + (r.begin + row_of(chunk, u)) * s.dim + me.col[j]);
            if constexpr (BACK) rg[u][j] = load_raw<T, VE>(grad + (r.begin + row_of(chunk, u)) * s.dim + me.col[j]);
          }
    };
    load(0, BACK);
    float2 st[NC][GN];
    if constexpr (!BACK) {
      float own[1][NC][VE];
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) own[0][j][i] = 0.0f;
      for (int k = 0; k < chunks; ++k) {
        if (k) load(k, false);
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && row_of(k, u) < rows)
#pragma unroll
              for (int i = 0; i < VE; ++i) own[0][j][i] += rx[u][j].get(i);
      }
      sum_groups<VE, NC, GN, 1, WARP>(own, my_room, sums, me, t.slots, lines, line);
#pragma unroll
      for (int j = 0; j < NC; ++j) {
#pragma unroll
        for (int i = 0; i < GN; ++i) st[j][i].x = sums[me.group[j][i]] * inv;
#pragma unroll
        for (int i = 0; i < VE; ++i) own[0][j][i] = 0.0f;
      }
      for (int k = 0; k < chunks; ++k) {
        if (chunks > 1) load(k, false);
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && row_of(k, u) < rows)
#pragma unroll
              for (int i = 0; i < VE; ++i) {
                const float d = rx[u][j].get(i) - st[j][i % GN].x;
                own[0][j][i] = fmaf(d, d, own[0][j][i]);
              }
      }
      sum_groups<VE, NC, GN, 1, WARP>(own, my_room, squares, me, t.slots, lines, line);
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < GN; ++i) st[j][i].y = rsqrtf(squares[me.group[j][i]] * inv + c.eps);
      for (int g = tid; g < me.groups; g += team) c.stats[seg * s.groups + me.group0 + g] = make_float2(sums[g] * inv, rsqrtf(squares[g] * inv + c.eps));
      for (int k = 0; k < chunks; ++k) {
        if (chunks > 1) load(k, false);
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && row_of(k, u) < rows) {
              float v[VE];
#pragma unroll
              for (int i = 0; i < VE; ++i) v[i] = rx[u][j].get(i);
              normalise(v, st[j]);
              const int64_t e = (r.begin + row_of(k, u)) * s.dim + me.col[j];
              finish_forward(c, e, v, gamma[j], beta[j]);
              store_all<T, VE>(out + e, v);
            }
      }
    } else {
      load_stats(s, c, me, seg, st);
      float ab[2][NC][VE], dz[kHeld][NC][VE];
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) ab[0][j][i] = ab[1][j][i] = 0.0f;
      const auto begin = [&](int k) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && row_of(k, u) < rows) {
              float xh[VE];
#pragma unroll
              for (int i = 0; i < VE; ++i) xh[i] = rx[u][j].get(i), dz[u][j][i] = rg[u][j].get(i);
              normalise(xh, st[j]);
              begin_backward(c, (r.begin + row_of(k, u)) * s.dim + me.col[j], xh, dz[u][j], gamma[j], beta[j]);
            }
      };
      for (int k = 0; k < chunks; ++k) {
        if (k) load(k, true);
        begin(k);
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && row_of(k, u) < rows)
#pragma unroll
              for (int i = 0; i < VE; ++i) {
                const float v = dz[u][j][i], xh = (rx[u][j].get(i) - st[j][i % GN].x) * st[j][i % GN].y, dxh = __fmul_rn(v, gamma[j][i]);
                dbeta[j][i] += v, dgamma[j][i] = fmaf(v, xh, dgamma[j][i]);
                ab[0][j][i] += dxh, ab[1][j][i] = fmaf(dxh, xh, ab[1][j][i]);
              }
      }
      sum_groups<VE, NC, GN, 2, WARP>(ab, my_room, sums, me, t.slots, lines, line);
      float2 means[NC][GN];
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < GN; ++i) means[j][i] = make_float2(sums[2 * me.group[j][i]] * inv, sums[2 * me.group[j][i] + 1] * inv);
      for (int k = 0; k < chunks; ++k) {
        if (chunks > 1) {
          load(k, true);
          begin(k);
        }
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && row_of(k, u) < rows) {
              float v[VE], dxh[VE];
#pragma unroll
              for (int i = 0; i < VE; ++i) v[i] = rx[u][j].get(i), dxh[i] = __fmul_rn(dz[u][j][i], gamma[j][i]);
              normalise(v, st[j]);
              finish_backward(v, dxh, st[j], means[j]);
              store_all<T, VE>(out + (r.begin + row_of(k, u)) * s.dim + me.col[j], v);
            }
      }
    }
    if (WARP) __syncwarp(); else __syncthreads();      // `sums` are the next segment's
  }
  if constexpr (BACK)
    if (c.columns) put_columns(s, c, t, me, room, dgamma, dbeta);
}

// Offsets that are none are flagged, and segments without rows have statistics of zero.
__device__ __forceinline__ void look_at_segments(const NormShape& s, const NormCall& c) {
  for (int64_t seg = threadIdx.x; seg < s.segments; seg += blockDim.x) {
    const RowRange r = group_rows(s.offsets, (int)seg, s.rows);
    if (bad_group(s.offsets, (int)seg, s.rows)) atomicOr(c.status, APT_FLAG_BAD_OFFSETS);
    if (r.end <= r.begin)
      for (int g = 0; g < s.groups; ++g) c.stats[seg * s.groups + g] = make_float2(0.0f, 0.0f);
  }
}

// Sums alone, where segments are long.
template <typename T, int VE, int NC, int GN, bool BACK>
__global__ void __launch_bounds__(256, BACK ? 2 : 4)
k_norm_sums(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c, const __grid_constant__ NormTiles t) {
  wait_for_previous();
  __shared__ float room[256 * NC * VE + 256], result[2 * kMostGroups];
  if (!BACK && s.offsets && blockIdx.x == 0 && blockIdx.y == 0) look_at_segments(s, c);
  tile_sums<T, VE, NC, GN, BACK>(s, c, t, room, result);
}
// Sums of long segments and all of short ones.
template <typename T, int VE, int NC, int GN, bool BACK, bool WARP>
__global__ void __launch_bounds__(256, 2)
k_norm_first(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c, const __grid_constant__ NormTiles t) {
  wait_for_previous();
  __shared__ float room[256 * NC * VE + 256], result[WARP ? 8 * 512 : 2 * kMostGroups];
  if (!BACK && s.offsets && blockIdx.x == 0 && blockIdx.y == 0) look_at_segments(s, c);
  if (blockIdx.x < t.tiles) tile_sums<T, VE, NC, GN, BACK>(s, c, t, room, result);
  else short_segments<T, VE, NC, GN, BACK, WARP>(s, c, t, room, result);
}

// Rows of long segments, and rows of none. Tiles from the last to the first: what was read last is still in L2.
template <typename T, int VE, int NC, int GN, bool BACK>
__global__ void __launch_bounds__(256, GN > 1 || NC > 1 ? 2 : BACK ? 3 : 4)
k_norm_second(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c, const __grid_constant__ NormTiles t, int joins) {
  wait_for_previous();
  if (BACK && (int)blockIdx.x < joins) {
    if (blockIdx.y == 0) join_columns<T>(s, c, blockIdx.x, t.tiles + t.short_blocks);
    return;
  }
  __shared__ float2 table[kMostGroups];
  const NormThread<VE, NC, GN> me(s, t);
  const T* const x = (const T*)c.x;
  const T* const grad = (const T*)c.grad;
  T* const out = (T*)c.out;
  const int64_t tile = t.tiles - 1 - (blockIdx.x - joins), row0 = tile * t.tile, row1 = min(row0 + t.tile, s.rows);
  float gamma[NC][VE], beta[NC][VE];
  bool loaded = false;
  int64_t done = row0;      // rows up to here are of segments
  for (int64_t seg = segment_at(s, row0); seg < s.segments; ++seg) {
    const RowRange whole = segment_rows(s, seg);
    if (whole.begin >= row1) break;
    const int64_t b = max(whole.begin, row0), e = min(whole.end, row1);
    if (e > done) done = e;
    if (whole.end - whole.begin <= t.cap || e <= b) continue;
    if (!loaded) load_params<T>(c, me, gamma, beta);
    loaded = true;
    // the segment's pieces, a warp a group
    const int64_t first = whole.begin / t.tile, last = (whole.end - 1) / t.tile;
    const float inv = 1.0f / ((float)(whole.end - whole.begin) * (float)me.per);
    __syncthreads();
    for (int g = threadIdx.x / 32; g < me.groups; g += 8) {
      const float2* const parts = c.parts + me.group0 + g;
      const auto rows_of = [&](int64_t i) { return (float)(min((i + 1) * t.tile, whole.end) - max(i * t.tile, whole.begin)); };
      float a = 0.0f, q = 0.0f;
      for (int64_t i = first + threadIdx.x % 32; i <= last; i += 32) {
        const float2 p = parts[(i + seg) * s.groups];
        if constexpr (BACK) a += p.x, q += p.y;
        else a = fmaf(p.x, rows_of(i) * (float)me.per, a);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        if constexpr (BACK) q += __shfl_xor_sync(0xffffffffu, q, o);
      }
      a *= inv;
      if constexpr (!BACK) {
        for (int64_t i = first + threadIdx.x % 32; i <= last; i += 32) {
          const float2 p = parts[(i + seg) * s.groups];
          q += fmaf(rows_of(i) * (float)me.per * (p.x - a), p.x - a, p.y);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) q += __shfl_xor_sync(0xffffffffu, q, o);
      }
      if (threadIdx.x % 32 == 0) {
        const float2 r = make_float2(a, BACK ? q * inv : rsqrtf(q * inv + c.eps));
        table[g] = r;
        if (!BACK && tile == first) c.stats[seg * s.groups + me.group0 + g] = r;
      }
    }
    __syncthreads();
    float2 st[NC][GN], ab[BACK ? NC : 1][GN];
    if constexpr (BACK) load_stats(s, c, me, seg, st);
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < GN; ++i) (BACK ? ab : st)[j][i] = table[me.group[j][i]];
    constexpr int U = BACK ? 2 : 4;
    for (int64_t r0 = b + me.line; r0 < e; r0 += U * t.lines) {
      Raw<T, VE> rx[U][NC], rg[BACK ? U : 1][NC];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (me.in[j] && r0 + u * t.lines < e) {
            rx[u][j] = load_raw<T, VE>(x + (r0 + u * t.lines) * s.dim + me.col[j]);
            if constexpr (BACK) rg[u][j] = load_raw<T, VE>(grad + (r0 + u * t.lines) * s.dim + me.col[j]);
          }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r0 + u * t.lines >= e) break;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          if (!me.in[j]) continue;
          const int64_t at = (r0 + u * t.lines) * s.dim + me.col[j];
          float v[VE];
#pragma unroll
          for (int i = 0; i < VE; ++i) v[i] = rx[u][j].get(i);
          normalise(v, st[j]);
          if constexpr (BACK) {
            float dz[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) dz[i] = rg[u][j].get(i);
            begin_backward(c, at, v, dz, gamma[j], beta[j]);
#pragma unroll
            for (int i = 0; i < VE; ++i) dz[i] = __fmul_rn(dz[i], gamma[j][i]);
            finish_backward(v, dz, st[j], ab[j]);
          } else {
            finish_forward(c, at, v, gamma[j], beta[j]);
          }
          store_all<T, VE>(out + at, v);
        }
      }
    }
  }
  // rows of no segment
  const float zeros[VE] = {};
  for (int64_t r = done + me.line; r < row1; r += t.lines)
#pragma unroll
    for (int j = 0; j < NC; ++j)
      if (me.in[j]) store_all<T, VE>(out + r * s.dim + me.col[j], zeros);
}

// --------------------------------------------------------------------------------------- groups of very many channels
__device__ __forceinline__ float block_sum(float v, float* shared) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.0f;
  for (int k = 0; k < 8; ++k) v += shared[k];
  return v;
}
template <typename T>
__device__ __forceinline__ float2 wide_xh_dz(const NormCall& c, int64_t e, int64_t col, float2 st, float* gamma) {
  const float g = *gamma = param<T>(c.weight, c.wide_params, col, 1.0f);
  float xh[1] = {(Elem<T>::to_f(((const T*)c.x)[e]) - st.x) * st.y}, dz[1] = {Elem<T>::to_f(((const T*)c.grad)[e])};
  const float gs[1] = {g}, bs[1] = {param<T>(c.bias, c.wide_params, col, 0.0f)};
  begin_backward(c, e, xh, dz, gs, bs);
  return make_float2(xh[0], dz[0]);
}
template <typename T, bool BACK>
__global__ void __launch_bounds__(256) k_norm_wide(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c) {
  wait_for_previous();
  __shared__ float shared[8];
  const T* const x = (const T*)c.x;
  T* const out = (T*)c.out;
  for (int64_t item = blockIdx.x; item < s.segments * s.groups; item += gridDim.x) {
    const int64_t seg = item / s.groups, c0 = item % s.groups * s.per;
    const RowRange r = segment_rows(s, seg);
    if (!BACK && s.offsets && c0 == 0 && threadIdx.x == 0 && bad_group(s.offsets, (int)seg, s.rows)) atomicOr(c.status, APT_FLAG_BAD_OFFSETS);
    const float inv = 1.0f / ((float)(r.end - r.begin) * (float)s.per);
    const auto walk = [&](auto&& f) {
      for (int64_t row = r.begin; row < r.end; ++row)
        for (int k = threadIdx.x; k < s.per; k += 256) f(row * s.dim + c0 + k, c0 + k);
    };
    if constexpr (!BACK) {
      float sum = 0.0f;
      walk([&](int64_t e, int64_t) { sum += Elem<T>::to_f(x[e]); });
      const float mean = block_sum(sum, shared) * inv;
      sum = 0.0f;
      walk([&](int64_t e, int64_t) {
        const float d = Elem<T>::to_f(x[e]) - mean;
        sum = fmaf(d, d, sum);
      });
      const float rstd = rsqrtf(block_sum(sum, shared) * inv + c.eps);
      if (threadIdx.x == 0) c.stats[item] = r.end > r.begin ? make_float2(mean, rstd) : make_float2(0.0f, 0.0f);
      walk([&](int64_t e, int64_t col) {
        float v[1] = {(Elem<T>::to_f(x[e]) - mean) * rstd};
        const float g[1] = {param<T>(c.weight, c.wide_params, col, 1.0f)}, b[1] = {param<T>(c.bias, c.wide_params, col, 0.0f)};
        finish_forward(c, e, v, g, b);
        out[e] = Elem<T>::from_f(v[0]);
      });
    } else {
      const float2 st = c.stats[item];
      float a = 0.0f, b = 0.0f, gamma;
      walk([&](int64_t e, int64_t col) {
        const float2 v = wide_xh_dz<T>(c, e, col, st, &gamma);
        const float dxh = __fmul_rn(v.y, gamma);
        a += dxh, b = fmaf(dxh, v.x, b);
      });
      a = block_sum(a, shared) * inv, b = block_sum(b, shared) * inv;
      walk([&](int64_t e, int64_t col) {
        const float2 v = wide_xh_dz<T>(c, e, col, st, &gamma);
        out[e] = Elem<T>::from_f(st.y * (__fmul_rn(v.y, gamma) - a - v.x * b));
      });
    }
  }
  if (s.offsets)      // rows of no segment
    for (int64_t row = min(max(s.offsets[s.segments], (int64_t)0), s.rows) + blockIdx.x; row < s.rows; row += gridDim.x)
      for (int64_t k = threadIdx.x; k < s.dim; k += 256) out[row * s.dim + k] = Elem<T>::from_f(0.0f);
}
// dgamma and dbeta, a channel a thread.
template <typename T>
__global__ void __launch_bounds__(256) k_norm_wide_params(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c) {
  wait_for_previous();
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= s.dim) return;
  float dgamma = 0.0f, dbeta = 0.0f, gamma;
  for (int64_t seg = 0; seg < s.segments; ++seg) {
    const RowRange r = segment_rows(s, seg);
    float a = 0.0f, b = 0.0f;
    for (int64_t row = r.begin; row < r.end; ++row) {
      const float2 v = wide_xh_dz<T>(c, row * s.dim + col, col, c.stats[seg * s.groups + col / s.per], &gamma);
      a = fmaf(v.x, v.y, a), b += v.y;
    }
    dgamma += a, dbeta += b;
  }
  put_param<T>(c.grad_weight, c.wide_params, col, dgamma);
  put_param<T>(c.grad_bias, c.wide_params, col, dbeta);
}

// ------------------------------------------------------------------------------------------------- host side
enum NormKind { kNormRows, kNormTiles, kNormWide };
struct NormPlan {
  NormKind kind;
  int slice;              // elements of an access
  NormLanes lanes;
  int held;               // slices a lane (thread) has of a row
  int64_t blocks, chunks; // grid of the first kernel
  NormTiles tiles;
  bool warps;             // short segments by warps
};

template <typename T, int VE, bool BACK>
static int norm_rows(const NormShape& s, const NormCall& c, const NormPlan& p, cudaStream_t st) {
  const dim3 grid((unsigned)p.blocks, (unsigned)p.chunks);
  if (p.lanes.width == 256) {
    if (p.held == 1) APT_FOLLOW((k_norm_rows<T, VE, 1, BACK ? 1 : 2, true, BACK>), grid, 256, 0, st, s, c, p.lanes);
    else if (p.held == 2) APT_FOLLOW((k_norm_rows<T, VE, 2, 1, true, BACK>), grid, 256, 0, st, s, c, p.lanes);
    else APT_FOLLOW((k_norm_rows<T, VE, 4, 1, true, BACK>), grid, 256, 0, st, s, c, p.lanes);
  } else {
    if (p.held == 1) APT_FOLLOW((k_norm_rows<T, VE, 1, BACK ? 2 : 4, false, BACK>), grid, 256, 0, st, s, c, p.lanes);
    else APT_FOLLOW((k_norm_rows<T, VE, 2, BACK ? 1 : 2, false, BACK>), grid, 256, 0, st, s, c, p.lanes);
  }
  if (BACK && c.columns) APT_FOLLOW((k_norm_columns<T>), ceil_div(2 * s.dim, 32), 256, 0, st, s, c, p.blocks);
  return APT_OK;
}
template <typename T, int VE, int NC, int GN, bool BACK>
static int norm_tiles(const NormShape& s, const NormCall& c, const NormPlan& p, cudaStream_t st) {
  const dim3 first((unsigned)p.blocks, (unsigned)p.chunks);
  if (!p.tiles.short_blocks) APT_FOLLOW((k_norm_sums<T, VE, NC, GN, BACK>), first, 256, 0, st, s, c, p.tiles);
  else if (p.warps) APT_FOLLOW((k_norm_first<T, VE, NC, GN, BACK, true>), first, 256, 0, st, s, c, p.tiles);
  else APT_FOLLOW((k_norm_first<T, VE, NC, GN, BACK, false>), first, 256, 0, st, s, c, p.tiles);
  const int joins = BACK && c.columns ? (int)ceil_div(2 * s.dim, 32) : 0;
  const dim3 second((unsigned)(p.tiles.tiles + joins), (unsigned)p.chunks);
  APT_FOLLOW((k_norm_second<T, VE, NC, GN, BACK>), second, 256, 0, st, s, c, p.tiles, joins);
  return APT_OK;
}
template <typename T, int VE, int NC, bool BACK>
static int norm_held(const NormShape& s, const NormCall& c, const NormPlan& p, cudaStream_t st) {
  if constexpr (VE > 1)
    if (s.per % VE) return norm_tiles<T, VE, NC, VE, BACK>(s, c, p, st);
  return norm_tiles<T, VE, NC, 1, BACK>(s, c, p, st);
}
template <typename T, int VE, bool BACK>
static int norm_slices(const NormShape& s, const NormCall& c, const NormPlan& p, cudaStream_t st) {
  if (p.kind == kNormRows) return norm_rows<T, VE, BACK>(s, c, p, st);
  if constexpr (VE < 8)
    if (p.held > 1) return norm_held<T, VE, 8 / VE, BACK>(s, c, p, st);
  return norm_held<T, VE, 1, BACK>(s, c, p, st);
}
template <typename T, bool BACK>
int norm(const NormShape& s, const NormCall& c, const NormPlan& p, cudaStream_t st) {
  if (p.kind == kNormWide) {
    if (s.rows) APT_FOLLOW((k_norm_wide<T, BACK>), wave_grid(s.segments * s.groups, 8), 256, 0, st, s, c);
    if (BACK && (c.grad_weight || c.grad_bias)) APT_FOLLOW((k_norm_wide_params<T>), ceil_div(s.dim, 256), 256, 0, st, s, c);
    return APT_OK;
  }
  if (p.slice == 16 / (int)sizeof(T)) return norm_slices<T, 16 / (int)sizeof(T), BACK>(s, c, p, st);
  if constexpr (sizeof(T) == 2)
    if (p.slice == 2) return norm_slices<T, 2, BACK>(s, c, p, st);
  return norm_slices<T, 1, BACK>(s, c, p, st);
}

}  // namespace apt
