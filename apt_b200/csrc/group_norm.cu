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

// A thread has NC slices of VE neighbouring channels of every `lines`-th row.
struct NormTiles {
  int64_t tile, tiles;      // rows of a tile, how many
  int small_blocks;
  int chunk;                // groups of a block
  int slots, lines;         // threads side by side in a row, rows side by side
  int cap;                  // rows of the segments that a block does by itself
};

// Sums of K numbers over a segment's piece and each group, from per-thread sums a channel: result[k][group] in shared memory.
template <int VE, int NC, int K>
__device__ __forceinline__ void sum_groups(const float (&v)[K][NC][VE], float* room, float (*result)[K], int slots, int lines, int per, int groups, int slot, int line,
                                           bool mine) {
  const int columns = slots * NC * VE, pitch = columns + 1;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    __syncthreads();
    if (mine)
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) room[line * pitch + (slot + j * slots) * VE + i] = v[k][j][i];
    __syncthreads();
    const int lane = threadIdx.x % 32;
    for (int g = threadIdx.x / 32; g < groups; g += 8) {
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
      if (lane == 0) result[g][k] = sum;
    }
  }
  __syncthreads();
}

template <typename T, int VE, int NC, bool BACK>
struct NormThread {
  int slot, line, group0, groups, per, col0;
  bool mine;
  bool in[NC];
  int col[NC];
  uint16_t group[NC][VE];        // within the block's
  __device__ __forceinline__ NormThread(const NormShape& s, const NormTiles& t) {
    slot = threadIdx.x % t.slots, line = threadIdx.x / t.slots;
    mine = line < t.lines;
    group0 = blockIdx.y * t.chunk, groups = min(t.chunk, s.groups - group0), per = s.per, col0 = group0 * s.per;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int k = (slot + j * t.slots) * VE;
      in[j] = mine && k < groups * per;
      col[j] = col0 + k;
#pragma unroll
      for (int i = 0; i < VE; ++i) group[j][i] = in[j] ? (uint16_t)((k + i) / per) : 0;
    }
  }
};

// Means and 1 / deviations of the groups in `table`, or the two means of the backward in `table2`, applied to a slice.
template <int VE>
__device__ __forceinline__ void normalise(float (&v)[VE], const float2 (&st)[VE]) {
#pragma unroll
  for (int i = 0; i < VE; ++i) v[i] = (v[i] - st[i].x) * st[i].y;
}

template <typename T, int VE, int NC, bool BACK>
__global__ void __launch_bounds__(256, 2)
k_norm_first(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c, const __grid_constant__ NormTiles t) {
  wait_for_previous();
  constexpr int kHeld = (BACK ? 4 : 8) / NC > 0 ? (BACK ? 4 : 8) / NC : 1;      // rows of a thread in registers
  __shared__ float room[256 * NC * VE + 256];
  __shared__ float result[2][kMostColumns / 4][2];      // few groups are wide, many are narrow: a block's chunk is at most 512 groups
  const NormThread<T, VE, NC, BACK> me(s, t);
  const T* const x = (const T*)c.x;
  const T* const grad = (const T*)c.grad;
  T* const out = (T*)c.out;
  float gamma[NC][VE], beta[NC][VE], dgamma[NC][VE], dbeta[NC][VE];
#pragma unroll
  for (int j = 0; j < NC; ++j)
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      gamma[j][i] = me.in[j] ? param<T>(c.weight, c.wide_params, me.col[j] + i, 1.0f) : 0.0f;
      beta[j][i] = me.in[j] ? param<T>(c.bias, c.wide_params, me.col[j] + i, 0.0f) : 0.0f;
      dgamma[j][i] = dbeta[j][i] = 0.0f;
    }
  if (blockIdx.x < t.tiles) {
    // ---- sums of a tile's rows of long segments
    const int64_t row0 = blockIdx.x * t.tile, row1 = min(row0 + t.tile, s.rows);
    for (int64_t seg = segment_at(s, row0); seg < s.segments; ++seg) {
      const RowRange whole = segment_rows(s, seg);
      if (whole.begin >= row1) break;
      const int64_t b = max(whole.begin, row0), e = min(whole.end, row1);
      if (whole.end - whole.begin <= t.cap || e <= b) continue;
      float2* const parts = c.parts + (blockIdx.x + seg) * s.groups + me.group0;
      if constexpr (!BACK) {
        float v[1][NC][VE], q[1][NC][VE];
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int i = 0; i < VE; ++i) v[0][j][i] = q[0][j][i] = 0.0f;
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
            const float share = 1.0f / n;
#pragma unroll
            for (int j = 0; j < NC; ++j)
              if (me.in[j])
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                  const float y = raw[u][j].get(i), d = y - v[0][j][i];
                  v[0][j][i] = fmaf(d, share, v[0][j][i]);
                  q[0][j][i] = fmaf(d, y - v[0][j][i], q[0][j][i]);
                }
          }
        }
        // the piece's mean, then the squares around it
        float own[1][NC][VE];
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int i = 0; i < VE; ++i) own[0][j][i] = me.in[j] ? v[0][j][i] * n : 0.0f;
        float(*const sums)[1] = (float(*)[1])result[0];
        sum_groups<VE, NC, 1>(own, room, sums, t.slots, t.lines, me.per, me.groups, me.slot, me.line, me.mine);
        const float count = (float)(e - b) * (float)me.per;
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            const float d = v[0][j][i] - sums[me.group[j][i]][0] / count;
            own[0][j][i] = me.in[j] ? fmaf(n * d, d, q[0][j][i]) : 0.0f;
          }
        float(*const squares)[1] = (float(*)[1])result[1];
        sum_groups<VE, NC, 1>(own, room, squares, t.slots, t.lines, me.per, me.groups, me.slot, me.line, me.mine);
        for (int g = threadIdx.x; g < me.groups; g += 256) parts[g] = make_float2(sums[g][0] / count, squares[g][0]);
      } else {
        float2 st[NC][VE];
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int i = 0; i < VE; ++i) st[j][i] = c.stats[seg * s.groups + me.group0 + me.group[j][i]];
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
        sum_groups<VE, NC, 2>(ab, room, result[0], t.slots, t.lines, me.per, me.groups, me.slot, me.line, me.mine);
        for (int g = threadIdx.x; g < me.groups; g += 256) parts[g] = make_float2(result[0][g][0], result[0][g][1]);
      }
    }
  } else {
    // ---- short segments, whole
    for (int64_t seg = blockIdx.x - t.tiles; seg < s.segments; seg += t.small_blocks) {
      const RowRange r = segment_rows(s, seg);
      if (!BACK && s.offsets && blockIdx.y == 0 && threadIdx.x == 0 && bad_group(s.offsets, (int)seg, s.rows)) atomicOr(c.status, APT_FLAG_BAD_OFFSETS);
      const int rows = (int)min(r.end - r.begin, (int64_t)t.cap + 1);
      if (!BACK && rows == 0)
        for (int g = threadIdx.x; g < me.groups; g += 256) c.stats[seg * s.groups + me.group0 + g] = make_float2(0.0f, 0.0f);
      if (rows > t.cap || rows == 0) continue;
      const float inv = 1.0f / ((float)rows * (float)me.per);
      Raw<T, VE> rx[kHeld][NC], rg[BACK ? kHeld : 1][NC];
#pragma unroll
      for (int u = 0; u < kHeld; ++u)
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (me.in[j] && me.line + u * t.lines < rows) {
            rx[u][j] = load_raw<T, VE>(x + (r.begin + me.line + u * t.lines) * s.dim + me.col[j]);
            if constexpr (BACK) rg[u][j] = load_raw<T, VE>(grad + (r.begin + me.line + u * t.lines) * s.dim + me.col[j]);
          }
      float2 st[NC][VE];
      if constexpr (!BACK) {
        float own[1][NC][VE];
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            own[0][j][i] = 0.0f;
#pragma unroll
            for (int u = 0; u < kHeld; ++u)
              if (me.in[j] && me.line + u * t.lines < rows) own[0][j][i] += rx[u][j].get(i);
          }
        float(*const sums)[1] = (float(*)[1])result[0];
        sum_groups<VE, NC, 1>(own, room, sums, t.slots, t.lines, me.per, me.groups, me.slot, me.line, me.mine);
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            st[j][i].x = sums[me.group[j][i]][0] * inv;
            own[0][j][i] = 0.0f;
#pragma unroll
            for (int u = 0; u < kHeld; ++u)
              if (me.in[j] && me.line + u * t.lines < rows) {
                const float d = rx[u][j].get(i) - st[j][i].x;
                own[0][j][i] = fmaf(d, d, own[0][j][i]);
              }
          }
        float(*const squares)[1] = (float(*)[1])result[1];
        sum_groups<VE, NC, 1>(own, room, squares, t.slots, t.lines, me.per, me.groups, me.slot, me.line, me.mine);
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int i = 0; i < VE; ++i) st[j][i].y = rsqrtf(squares[me.group[j][i]][0] * inv + c.eps);
        for (int g = threadIdx.x; g < me.groups; g += 256)
          c.stats[seg * s.groups + me.group0 + g] = make_float2(sums[g][0] * inv, rsqrtf(squares[g][0] * inv + c.eps));
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && me.line + u * t.lines < rows) {
              float v[VE];
#pragma unroll
              for (int i = 0; i < VE; ++i) v[i] = rx[u][j].get(i);
              normalise(v, st[j]);
              const int64_t e = (r.begin + me.line + u * t.lines) * s.dim + me.col[j];
              finish_forward(c, e, v, gamma[j], beta[j]);
              store_all<T, VE>(out + e, v);
            }
      } else {
        float ab[2][NC][VE];
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            st[j][i] = c.stats[seg * s.groups + me.group0 + me.group[j][i]];
            ab[0][j][i] = ab[1][j][i] = 0.0f;
          }
        float dz[kHeld][NC][VE];
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && me.line + u * t.lines < rows) {
              float xh[VE];
#pragma unroll
              for (int i = 0; i < VE; ++i) xh[i] = rx[u][j].get(i), dz[u][j][i] = rg[u][j].get(i);
              normalise(xh, st[j]);
              begin_backward(c, (r.begin + me.line + u * t.lines) * s.dim + me.col[j], xh, dz[u][j], gamma[j], beta[j]);
#pragma unroll
              for (int i = 0; i < VE; ++i) {
                const float v = dz[u][j][i];
                dbeta[j][i] += v, dgamma[j][i] = fmaf(v, xh[i], dgamma[j][i]);
                dz[u][j][i] = __fmul_rn(v, gamma[j][i]);
                ab[0][j][i] += dz[u][j][i], ab[1][j][i] = fmaf(dz[u][j][i], xh[i], ab[1][j][i]);
              }
            }
        sum_groups<VE, NC, 2>(ab, room, result[0], t.slots, t.lines, me.per, me.groups, me.slot, me.line, me.mine);
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && me.line + u * t.lines < rows) {
              float v[VE];
#pragma unroll
              for (int i = 0; i < VE; ++i) {
                const float xh = (rx[u][j].get(i) - st[j][i].x) * st[j][i].y;
                v[i] = st[j][i].y * (dz[u][j][i] - result[0][me.group[j][i]][0] * inv - xh * (result[0][me.group[j][i]][1] * inv));
              }
              store_all<T, VE>(out + (r.begin + me.line + u * t.lines) * s.dim + me.col[j], v);
            }
      }
      __syncthreads();      // `result` is the next segment's
    }
  }
  if constexpr (BACK) {
    if (!c.columns) return;
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
}

// Rows of long segments, and rows of none. Tiles from the last to the first: what k_norm_first read last is still in L2.
template <typename T, int VE, int NC, bool BACK>
__global__ void __launch_bounds__(256, 2)
k_norm_second(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c, const __grid_constant__ NormTiles t, int joins) {
  wait_for_previous();
  if (BACK && (int)blockIdx.x < joins) {
    if (blockIdx.y == 0) join_columns<T>(s, c, blockIdx.x, t.tiles + t.small_blocks);
    return;
  }
  __shared__ float2 table[kMostColumns / 4];
  const NormThread<T, VE, NC, BACK> me(s, t);
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
    if (!loaded) {
      loaded = true;
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          gamma[j][i] = me.in[j] ? param<T>(c.weight, c.wide_params, me.col[j] + i, 1.0f) : 0.0f;
          beta[j][i] = me.in[j] ? param<T>(c.bias, c.wide_params, me.col[j] + i, 0.0f) : 0.0f;
        }
    }
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
    float2 st[NC][VE], ab[BACK ? NC : 1][VE];
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        if constexpr (BACK) {
          ab[j][i] = table[me.group[j][i]];
          st[j][i] = c.stats[seg * s.groups + me.group0 + me.group[j][i]];
        } else {
          st[j][i] = table[me.group[j][i]];
        }
      }
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
            for (int i = 0; i < VE; ++i) v[i] = st[j][i].y * (__fmul_rn(dz[i], gamma[j][i]) - ab[j][i].x - v[i] * ab[j][i].y);
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
};

// Elements of an access that `run` elements from any of the addresses on are a whole number of: 16 or 4 bytes, or one.
static int slice_of(int64_t run, size_t size, uintptr_t addresses) {
  for (const int bytes : {16, 4})
    if (bytes > (int)size && (run * (int64_t)size) % bytes == 0 && addresses % bytes == 0) return bytes / (int)size;
  return 1;
}

static NormPlan norm_plan(const NormShape& s, size_t size, uintptr_t addresses, bool back) {
  NormPlan p = {};
  if (!s.offsets && s.per_segment == 1) {
    p.slice = slice_of(s.per, size, addresses);
    const int64_t slices = ceil_div(s.per, p.slice);
    if (slices <= 1024) {
      p.kind = kNormRows;
      int w = 1;
      while (w < 32 && w < slices) w *= 2;
      if (slices > 64) w = 256;
      p.held = (int)ceil_div(slices, w);
      if (p.held == 3) p.held = 4;
      p.lanes.width = w;
      p.lanes.groups = (int)std::min<int64_t>(s.groups, 256 / w);
      p.lanes.rows = 256 / (w * p.lanes.groups);
      p.chunks = ceil_div(s.groups, p.lanes.groups);
      p.blocks = std::max<int64_t>(1, std::min<int64_t>(ceil_div(s.rows, p.lanes.rows * (back ? 2 : 4)), ceil_div(kNumSMs * (back ? 4 : 8), p.chunks)));
      return p;
    }
  }
  p.slice = slice_of(s.dim, size, addresses);
  // a block has whole groups, a chunk of them that begins on an access
  int chunk = s.groups;
  if (s.dim > kMostColumns || s.groups > kMostColumns / 4) {
    chunk = std::min<int>(kMostColumns / s.per, kMostColumns / 4);
    while (chunk > 0 && (int64_t)chunk * s.per % p.slice) --chunk;
  }
  const int64_t slices = chunk > 0 ? ceil_div((int64_t)std::min(chunk, s.groups) * s.per, p.slice) : 0;
  if (chunk <= 0 || slices > 256 * (8 / p.slice) || s.segments == 0) {
    p.kind = kNormWide;
    return p;
  }
  p.kind = kNormTiles;
  NormTiles& t = p.tiles;
  p.held = slices <= 256 ? 1 : 8 / p.slice;
  t.chunk = chunk;
  p.chunks = ceil_div(s.groups, chunk);
  t.slots = (int)ceil_div(slices, p.held);
  t.lines = 256 / t.slots;
  t.cap = std::max((back ? 4 : 8) / p.held, 1) * t.lines;
  // tiles for four blocks an SM, of eight rounds of rows at least
  t.tile = std::max<int64_t>(8 * t.lines, ceil_div(ceil_div(s.rows, ceil_div(kNumSMs * 4, p.chunks)), t.lines) * t.lines);
  t.tiles = ceil_div(s.rows, t.tile);
  t.small_blocks = (int)std::min<int64_t>(s.segments, kNumSMs * 4);
  p.blocks = t.tiles + t.small_blocks;
  return p;
}

static size_t norm_room(const NormShape& s, const NormPlan& p, bool back) {
  const size_t columns = back && p.kind != kNormWide ? align_up((size_t)p.blocks * 2 * s.dim * 4, 256) : 0;
  return columns + (p.kind == kNormTiles ? (size_t)(p.tiles.tiles + s.segments) * s.groups * 8 : 0);
}

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
template <typename T, int VE, int NC, bool BACK>
static int norm_tiles(const NormShape& s, const NormCall& c, const NormPlan& p, cudaStream_t st) {
  const dim3 first((unsigned)p.blocks, (unsigned)p.chunks);
  APT_FOLLOW((k_norm_first<T, VE, NC, BACK>), first, 256, 0, st, s, c, p.tiles);
  const int joins = BACK && c.columns ? (int)ceil_div(2 * s.dim, 32) : 0;
  const dim3 second((unsigned)(p.tiles.tiles + joins), (unsigned)p.chunks);
  APT_FOLLOW((k_norm_second<T, VE, NC, BACK>), second, 256, 0, st, s, c, p.tiles, joins);
  return APT_OK;
}
template <typename T, int VE, bool BACK>
static int norm_slices(const NormShape& s, const NormCall& c, const NormPlan& p, cudaStream_t st) {
  if (p.kind == kNormRows) return norm_rows<T, VE, BACK>(s, c, p, st);
  if constexpr (VE < 8)
    if (p.held > 1) return norm_tiles<T, VE, 8 / VE, BACK>(s, c, p, st);
  return norm_tiles<T, VE, 1, BACK>(s, c, p, st);
}
template <typename T, bool BACK>
static int norm(const NormShape& s, const NormCall& c, const NormPlan& p, cudaStream_t st) {
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
template <bool BACK>
static int norm_typed(int dtype, const NormShape& s, const NormCall& c, const NormPlan& p, cudaStream_t st) {
  if (dtype == APT_F32) return norm<float, BACK>(s, c, p, st);
  if (dtype == APT_BF16) return norm<__nv_bfloat16, BACK>(s, c, p, st);
  return norm<__half, BACK>(s, c, p, st);
}

static int norm_check(const char* who, int dtype, int param_dtype, int64_t rows, int64_t dim, int groups, const int64_t* offsets, int64_t segments,
                      double eps, int act, double p) {
  APT_CHECK_ARG(dtype == APT_F32 || dtype == APT_BF16 || dtype == APT_F16, "%s: unsupported dtype %d", who, dtype);
  APT_CHECK_ARG(param_dtype == dtype || param_dtype == APT_F32, "%s: parameters of type %d beside type %d", who, param_dtype, dtype);
  APT_CHECK_ARG(rows >= 0 && dim > 0 && dim < (1 << 24) && groups > 0 && dim % groups == 0, "%s: %lld channels in %d groups", who, (long long)dim, groups);
  APT_CHECK_ARG(segments >= 0 && segments < (1 << 30) && (rows == 0 || segments > 0) && (offsets || segments == 0 || rows % segments == 0),
                "%s: %lld rows in %lld segments", who, (long long)rows, (long long)segments);
  APT_CHECK_ARG(eps >= 0.0, "%s: eps = %g", who, eps);
  APT_CHECK_ARG(act >= APT_ACT_NONE && act <= APT_ACT_GELU, "%s: unknown activation %d", who, act);
  APT_CHECK_ARG(p >= 0.0 && p <= 1.0, "%s: p = %g is no probability", who, p);
  return APT_OK;
}
static NormShape norm_shape(int64_t rows, int64_t dim, int groups, const int64_t* offsets, int64_t segments) {
  return {rows, dim, segments, segments ? rows / segments : 0, offsets, groups, (int)(dim / groups)};
}

}  // namespace apt

extern "C" size_t apt_group_norm_workspace_bytes(int dtype, int64_t rows, int64_t dim, int groups, const int64_t* offsets, int64_t segments, int backward) {
  using namespace apt;
  if (rows <= 0 || dim <= 0 || groups <= 0 || segments <= 0) return 0;
  // buffers that begin anywhere may take narrower accesses
  const NormShape s = norm_shape(rows, dim, groups, offsets, segments);
  size_t most = 0;
  for (const uintptr_t addresses : {0, 4, 2}) most = std::max(most, norm_room(s, norm_plan(s, dtype == APT_F32 ? 4 : 2, addresses, backward), backward));
  return most;
}

extern "C" int apt_group_norm_forward(int dtype, int param_dtype, const void* x, int64_t rows, int64_t dim, int groups, const int64_t* offsets,
                                      int64_t segments, double eps, int act, const void* weight, const void* bias, double p, uint64_t key,
                                      uint32_t call_id, void* out, float* stats, void* workspace, size_t workspace_bytes, int32_t* status_word,
                                      void* stream) {
  using namespace apt;
  if (const int e = norm_check("apt_group_norm_forward", dtype, param_dtype, rows, dim, groups, offsets, segments, eps, act, p)) return e;
  if (rows == 0) return APT_OK;
  const NormShape s = norm_shape(rows, dim, groups, offsets, segments);
  APT_CHECK_ARG(x && out && status_word && (stats || (!offsets && segments == rows && dim / groups <= APT_GROUP_NORM_ROW_CHANNELS)), "apt_group_norm_forward: null buffer");
  APT_CHECK_ARG(workspace_bytes >= apt_group_norm_workspace_bytes(dtype, rows, dim, groups, offsets, segments, 0), "apt_group_norm_forward: workspace too small");
  const NormPlan plan = norm_plan(s, dtype == APT_F32 ? 4 : 2, (uintptr_t)x | (uintptr_t)out, false);
  const NormCall c{x, nullptr, weight, bias, out, nullptr, nullptr, (float2*)stats, (float)eps, act, param_dtype == APT_F32, p > 0.0,
                   make_drop(p, key, call_id), status_word, nullptr, (float2*)workspace};
  return norm_typed<false>(dtype, s, c, plan, (cudaStream_t)stream);
}

extern "C" int apt_group_norm_backward(int dtype, int param_dtype, const void* x, const void* grad_out, int64_t rows, int64_t dim, int groups,
                                       const int64_t* offsets, int64_t segments, double eps, int act, const void* weight, const void* bias, double p,
                                       uint64_t key, uint32_t call_id, const float* stats, void* grad_x, void* grad_weight, void* grad_bias,
                                       void* workspace, size_t workspace_bytes, int32_t* status_word, void* stream) {
  using namespace apt;
  if (const int e = norm_check("apt_group_norm_backward", dtype, param_dtype, rows, dim, groups, offsets, segments, eps, act, p)) return e;
  const cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    const size_t bytes = (size_t)dim * (param_dtype == APT_F32 ? 4 : 2);
    if (grad_weight) APT_CUDA(cudaMemsetAsync(grad_weight, 0, bytes, st));
    if (grad_bias) APT_CUDA(cudaMemsetAsync(grad_bias, 0, bytes, st));
    return APT_OK;
  }
  APT_CHECK_ARG(x && grad_out && grad_x && status_word && (stats || (!offsets && segments == rows && dim / groups <= APT_GROUP_NORM_ROW_CHANNELS)), "apt_group_norm_backward: null buffer");
  APT_CHECK_ARG(workspace_bytes >= apt_group_norm_workspace_bytes(dtype, rows, dim, groups, offsets, segments, 1), "apt_group_norm_backward: workspace too small");
  const NormShape s = norm_shape(rows, dim, groups, offsets, segments);
  const NormPlan plan = norm_plan(s, dtype == APT_F32 ? 4 : 2, (uintptr_t)x | (uintptr_t)grad_out | (uintptr_t)grad_x, true);
  const bool params = grad_weight || grad_bias;
  const size_t columns = plan.kind != kNormWide ? align_up((size_t)plan.blocks * 2 * dim * 4, 256) : 0;
  const NormCall c{x, grad_out, weight, bias, grad_x, grad_weight, grad_bias, (float2*)stats, (float)eps, act, param_dtype == APT_F32, p > 0.0,
                   make_drop(p, key, call_id), status_word, params ? (float*)workspace : nullptr, (float2*)((char*)workspace + columns)};
  return norm_typed<true>(dtype, s, c, plan, st);
}
