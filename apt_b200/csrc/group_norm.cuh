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
// Segments: tiles of rows are summed up, piece by piece of the segments they have rows of (k_norm_sums), the pieces are joined
// (k_norm_join) and the rows walked again (k_norm_apply), so that a segment's length matters to nobody: a batch of small graphs and a few
// long node types are the same work. The second walk finds in L2 what fits there.
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
  float2 *parts, *means;                         // sums of the pieces of segments, the backward's two means of each
  uint8_t* mask;                                 // backward of long segments, slices of whole quads: what stays
};

__device__ __forceinline__ RowRange segment_rows(const NormShape& s, int64_t k) {
  if (s.offsets) return group_rows(s.offsets, (int)k, s.rows);
  return {k * s.per_segment, (k + 1) * s.per_segment};
}
// The first segment that ends behind the row, by all lanes of a warp: 32 ends are looked at in a round.
__device__ __forceinline__ int64_t segment_at(const NormShape& s, int64_t row) {
  if (!s.offsets) return row / s.per_segment;
  int64_t lo = 0, hi = s.segments;
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32, at = lo + (threadIdx.x % 32) * step;
    const uint32_t behind = __ballot_sync(0xffffffffu, at < hi && s.offsets[at + 1] > row);
    if (behind) {
      const int first = __ffs(behind) - 1;
      hi = lo + first * step;
      if (first) lo = hi - step + 1;
    } else {
      lo += (hi - 1 - lo) / step * step + 1;
    }
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

template <typename T, int N>
__device__ __forceinline__ void act_all(int act, float (&z)[N]) {
  switch (act) {
    case APT_ACT_RELU:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = act_of<T, APT_ACT_RELU>(z[k]);
      break;
    case APT_ACT_SILU:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = act_of<T, APT_ACT_SILU>(z[k]);
      break;
    case APT_ACT_GELU:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = act_of<T, APT_ACT_GELU>(z[k]);
      break;
  }
}
template <typename T, int N>
__device__ __forceinline__ void slope_all(int act, float (&z)[N]) {
  switch (act) {
    case APT_ACT_RELU:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = act_slope<T, APT_ACT_RELU>(z[k]);
      break;
    case APT_ACT_SILU:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = act_slope<T, APT_ACT_SILU>(z[k]);
      break;
    case APT_ACT_GELU:
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = act_slope<T, APT_ACT_GELU>(z[k]);
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
// Which of the elements from e on stay, a bit each.
template <int N>
__device__ __forceinline__ uint32_t kept(const Drop& d, int64_t e) {
  static_assert(N % 4 == 0, "whole quads");
  uint32_t bits = 0;
#pragma unroll
  for (int q = 0; q < N / 4; ++q) {
    const Philox4 w = drop_words(d, (e >> 2) + q);
#pragma unroll
    for (int k = 0; k < 4; ++k) bits |= w.w[k] >= d.threshold && d.scale != 0.0f ? 1u << (4 * q + k) : 0u;
  }
  return bits;
}
template <int N>
__device__ __forceinline__ void drop_by(const Drop& d, uint32_t bits, float (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = bits >> k & 1 ? v[k] * d.scale : 0.0f;
}

// y of normalised elements, in place.
template <typename T, int N>
__device__ __forceinline__ void finish_forward(const NormCall& c, int64_t e, float (&v)[N], const float (&gamma)[N], const float (&beta)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = fmaf(v[k], gamma[k], beta[k]);
  act_all<T>(c.act, v);
  if (c.drop) drop_all(c.d, e, v);
}
// dz of normalised elements and gradients, into the gradients. Where a call meets its elements twice, the first time leaves what stays in
// c.mask, a byte a slice of whole quads, and the second takes it from there: making it anew is half of such a pass.
enum MaskUse { kMaskMade, kMaskLeft, kMaskTaken };
template <typename T, int USE, int N>
__device__ __forceinline__ void begin_backward(const NormCall& c, int64_t e, const float (&xh)[N], float (&grad)[N], const float (&gamma)[N], const float (&beta)[N]) {
  float z[N];
#pragma unroll
  for (int k = 0; k < N; ++k) z[k] = fmaf(xh[k], gamma[k], beta[k]);
  slope_all<T>(c.act, z);
  if (c.drop) {
    if constexpr (USE == kMaskMade || N % 4) {
      drop_all(c.d, e, grad);
    } else {
      uint8_t* const at = c.mask + e / N;
      const uint32_t bits = USE == kMaskTaken ? *at : kept<N>(c.d, e);
      if (USE == kMaskLeft) *at = (uint8_t)bits;
      drop_by(c.d, bits, grad);
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) grad[k] *= z[k];
}

// ------------------------------------------------------------------------------------------ rows by themselves
struct NormLanes {
  int width;              // lanes of a row's group: a power of two up to 256; BLOCK: above 32
  int groups, rows;       // a block has side by side
  int blocks;             // for the rows of each such chunk of groups (all in one dimension of the grid: of chunks there may be over 65535)
};

// A sum over the lanes of each group, of U rows at once. `shared`: not that of the sum before, whose readers this one's barrier waits for.
template <bool BLOCK, int U>
__device__ __forceinline__ void sum_lanes(float (&v)[U], int width, float* shared) {
#pragma unroll
  for (int u = 0; u < U; ++u)
    for (int o = (BLOCK ? 32 : width) / 2; o; o >>= 1) v[u] += __shfl_xor_sync(0xffffffffu, v[u], o);
  if constexpr (BLOCK) {
    if (threadIdx.x % 32 == 0)
#pragma unroll
      for (int u = 0; u < U; ++u) shared[threadIdx.x / 32 * U + u] = v[u];
    __syncthreads();
    const int warps = width / 32, first = threadIdx.x / width * warps;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < 2; ++k) sum += shared[(first + k) * U + u];
      if (warps > 2)
#pragma unroll
        for (int k = 2; k < 4; ++k) sum += shared[(first + k) * U + u];
      if (warps > 4)
#pragma unroll
        for (int k = 4; k < 8; ++k) sum += shared[(first + k) * U + u];
      v[u] = sum;
    }
  }
}

// NV slices of VE elements a lane, U rows on their way. 67584 x 256 fp32 in 8 groups, silu and dropout: forwards 42 us (HBM: 21), backwards 65 (32),
// of which no pipe is full: issue slots 60 per cent, integer 52 and 45, DRAM 25 and 33. 65536 x 1024 bf16, gelu: 85 (41) and 161 (62), where a row's sums follow one another (three
// barriers backwards) and registers leave room for few rows at a time.
template <typename T, int VE, int NV, int U, bool BLOCK, bool BACK>
__global__ void __launch_bounds__(256)
k_norm_rows(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c, const __grid_constant__ NormLanes l) {
  wait_for_previous();
  __shared__ float shared[3][16 * U];
  __shared__ float sums[BACK ? 256 * VE : 1];
  const int width = l.width;
  const int lane = threadIdx.x % width, slot = threadIdx.x / width % l.groups, line = threadIdx.x / (width * l.groups);
  const int block = blockIdx.x % l.blocks, g = blockIdx.x / l.blocks * l.groups + slot;
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
  constexpr bool kAhead = BLOCK && NV <= 2;      // the next rows are loaded in front of the sums of these
  Raw<T, VE> rx[U][NV], rg[BACK ? U : 1][NV], next_x[kAhead ? U : 1][NV], next_g[kAhead && BACK ? U : 1][NV];
  const auto load = [&](int64_t base, auto& to_x, auto& to_g) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = base + u * l.rows + line;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (in[j] && row < s.rows) {
          to_x[u][j] = load_raw<T, VE>(x + row * s.dim + at[j]);
          if constexpr (BACK) to_g[u][j] = load_raw<T, VE>(grad + row * s.dim + at[j]);
        } else {
          to_x[u][j] = Raw<T, VE>{};
          if constexpr (BACK) to_g[u][j] = Raw<T, VE>{};
        }
      }
    }
  };
  if constexpr (kAhead) load(block * step, next_x, next_g);
  for (int64_t base = block * step; base < s.rows; base += l.blocks * step) {
    if constexpr (kAhead) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          rx[u][j] = next_x[u][j];
          if constexpr (BACK) rg[u][j] = next_g[u][j];
        }
      }
      load(base + l.blocks * step, next_x, next_g);
    } else {
      load(base, rx, rg);
    }
    int64_t row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) row[u] = base + u * l.rows + line;
    float mean[U], rstd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mean[u] = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VE; ++k) mean[u] += rx[u][j].get(k);
    }
    sum_lanes<BLOCK, U>(mean, width, shared[0]);
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
    sum_lanes<BLOCK, U>(rstd, width, shared[1]);
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
          finish_forward<T>(c, e, v, gamma[j], beta[j]);
          store_all<T, VE>(out + e, v);
        }
      }
    } else {
      float ab[2 * U], dz[U][NV][VE];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ab[u] = ab[U + u] = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          float xh[VE];
#pragma unroll
          for (int k = 0; k < VE; ++k) xh[k] = (rx[u][j].get(k) - mean[u]) * rstd[u], dz[u][j][k] = rg[u][j].get(k);
          begin_backward<T, kMaskMade>(c, row[u] * s.dim + at[j], xh, dz[u][j], gamma[j], beta[j]);
          if (!in[j] || row[u] >= s.rows) continue;
#pragma unroll
          for (int k = 0; k < VE; ++k) {
            const float v = dz[u][j][k], dxh = __fmul_rn(v, gamma[j][k]);
            dgamma[j][k] = fmaf(v, xh[k], dgamma[j][k]);
            dbeta[j][k] += v;
            dz[u][j][k] = dxh;
            ab[u] += dxh;
            ab[U + u] = fmaf(dxh, xh[k], ab[U + u]);
          }
        }
      }
      sum_lanes<BLOCK, 2 * U>(ab, width, shared[2]);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (row[u] >= s.rows) continue;
        const float a = ab[u] * inv, b = ab[U + u] * inv;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (!in[j]) continue;
          float v[VE];
#pragma unroll
          for (int k = 0; k < VE; ++k) v[k] = rstd[u] * (dz[u][j][k] - a - (rx[u][j].get(k) - mean[u]) * rstd[u] * b);
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
            c.columns[((int64_t)block * 2 + which) * s.dim + at[j] + k] = v;
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

// The rows are cut into tiles for teams of threads, a warp each where its lanes hold a row, else a block. A thread has NC slices of VE
// neighbouring channels of every `lines`-th row of its tile.
struct NormTiles {
  int64_t sum_rows, sum_tiles;        // of k_norm_sums, whose tiles the pieces are of
  int64_t apply_rows, apply_tiles;    // of k_norm_apply
  int fold;                           // parts of a group that the kernels take for groups (those that are wider than a block's columns)
  int chunk;                          // groups of a team
  int slots, lines;                   // threads side by side in a row, rows side by side
  int join_groups, join_segments;     // of a block of k_norm_join
};

// GN: groups that a slice may have channels of (1 where a group is whole slices).
template <int VE, int NC, int GN>
struct NormThread {
  int slot, line, group0, groups, per, col0;
  bool mine, even;      // even: sum_groups
  bool in[NC];
  int col[NC];
  uint16_t group[NC][GN];        // within the team's
  uint32_t heads;                // channels that are their group's first
  __device__ __forceinline__ NormThread(const NormShape& s, const NormTiles& t, int thread) {
    slot = thread % t.slots, line = thread / t.slots;
    mine = line < t.lines;
    group0 = blockIdx.y * t.chunk, groups = min(t.chunk, s.groups - group0), per = s.per, col0 = group0 * s.per;
    const int slices = per / VE;
    heads = 0;
    even = 32 % t.slots == 0 && (GN == 1 ? (slices & (slices - 1)) == 0 && slices <= t.slots : per == 1);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int k = (slot + j * t.slots) * VE;
      in[j] = mine && k < groups * per;
      col[j] = col0 + k;
#pragma unroll
      for (int i = 0; i < GN; ++i) {
        group[j][i] = in[j] ? (uint16_t)((k + i) / per) : 0;
        if (in[j] && (k + i) % per == 0) heads |= 1u << (j * GN + i);
      }
    }
  }
};

// Sums of K numbers over the rows and each group from per-thread sums a channel, by all threads of a block, or of a warp: got[k] of the groups that
// a thread has channels of. Between lanes directly where a warp's rows and a group's slices are powers of two (`even`) or a team has one group (18305 x 319
// bf16 in 1651 segments, us: backwards 106 -> 55, forwards 82 -> 37); else through shared memory (`room`, `result`: a team's own).
template <int VE, int NC, int GN, int K, bool WARP>
__device__ __forceinline__ void sum_groups(const float (&v)[K][NC][VE], float (&got)[K][NC][GN], float* room, float* result, const NormThread<VE, NC, GN>& me, int slots,
                                           int lines) {
  // a slice of one group is one number
  constexpr int kOwn = GN == 1 ? 1 : VE;
  const int columns = slots * NC * kOwn, pitch = columns + 1, per = GN == 1 ? me.per / VE : me.per, lane = threadIdx.x % 32;
  float own[K][NC][kOwn];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      if constexpr (kOwn == 1) {
        own[k][j][0] = 0.0f;
#pragma unroll
        for (int i = 0; i < VE; ++i) own[k][j][0] += v[k][j][i];
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) own[k][j][i] = v[k][j][i];
      }
    }
  if (WARP && me.even) {
    for (int o = 16; o; o >>= 1) {
      if (o < slots && (GN > 1 || o >= per)) continue;      // between rows, or within a group
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
          for (int i = 0; i < kOwn; ++i) own[k][j][i] += __shfl_xor_sync(0xffffffffu, own[k][j][i], o);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < GN; ++i) got[k][j][i] = own[k][j][i];
    return;
  }
  const auto sync = [] {
    if (WARP) __syncwarp(); else __syncthreads();
  };
  if (me.groups == 1) {      // all of the team's numbers
    float all[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      all[k] = 0.0f;
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < kOwn; ++i) all[k] += own[k][j][i];
#pragma unroll
      for (int o = 16; o; o >>= 1) all[k] += __shfl_xor_sync(0xffffffffu, all[k], o);
    }
    if constexpr (!WARP) {
      sync();
      if (lane == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) room[threadIdx.x / 32 * K + k] = all[k];
      sync();
#pragma unroll
      for (int k = 0; k < K; ++k) {
        all[k] = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) all[k] += room[w * K + k];
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < GN; ++i) got[k][j][i] = all[k];
    return;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    sync();
    if (me.mine)
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < kOwn; ++i) room[me.line * pitch + (me.slot + j * slots) * kOwn + i] = own[k][j][i];
    sync();
    if (WARP && me.groups > 8) {
      for (int g = lane; g < me.groups; g += 32) {
        float sum = 0.0f;
        for (int r = 0; r < lines; ++r)
          for (int i = 0; i < per; ++i) sum += room[r * pitch + g * per + i];
        result[g] = sum;
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
        if (lane == 0) result[g] = sum;
      }
    }
    sync();
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < GN; ++i) got[k][j][i] = result[me.group[j][i]];
  }
}
// Two numbers of each group to `to`, by the thread that has a group's first channel in the first row.
template <int VE, int NC, int GN>
__device__ __forceinline__ void put_groups(float2* to, const float (&a)[NC][GN], const float (&b)[NC][GN], const NormThread<VE, NC, GN>& me) {
  if (me.line) return;
#pragma unroll
  for (int j = 0; j < NC; ++j)
#pragma unroll
    for (int i = 0; i < GN; ++i)
      if (me.heads >> (j * GN + i) & 1) to[me.group[j][i]] = make_float2(a[j][i], b[j][i]);
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
__device__ __forceinline__ void load_stats(const NormShape& s, const NormTiles& t, const float2* stats, const NormThread<VE, NC, GN>& me, int64_t seg,
                                           float2 (&st)[NC][GN]) {
  if (t.fold > 1) {
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < GN; ++i) st[j][i] = stats[seg * (s.groups / t.fold) + (me.group0 + me.group[j][i]) / t.fold];
    return;
  }
#pragma unroll
  for (int j = 0; j < NC; ++j)
#pragma unroll
    for (int i = 0; i < GN; ++i) st[j][i] = stats[seg * s.groups + me.group0 + me.group[j][i]];
}

// A block's sums of dgamma and dbeta to its line of c.columns.
template <bool WARP, int VE, int NC, int GN>
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
        for (int i = 0; i < VE; ++i) room[(WARP ? threadIdx.x / 32 * t.lines + me.line : me.line) * pitch + (me.slot + j * t.slots) * VE + i] = which ? dbeta[j][i] : dgamma[j][i];
    __syncthreads();
    for (int k = threadIdx.x; k < me.groups * me.per; k += 256) {
      float v = 0.0f;
      for (int l = 0; l < (WARP ? 8 : 1) * t.lines; ++l) v += room[l * pitch + k];
      c.columns[((int64_t)blockIdx.x * 2 + which) * s.dim + me.col0 + k] = v;
    }
  }
}

// Sums of each tile's rows, piece by piece (the rows a tile has of a segment): piece number tile + segment, which no other has. Forwards the mean
// and the squares around it, backwards the sums of dxh and dxh xh.
// 151552 x 256 bf16 in 8 segments, us: forwards 23 (HBM: 12), backwards 84 (24) with silu and the dropout's generator.
template <typename T, int VE, int NC, int GN, bool BACK, bool WARP>
__global__ void __launch_bounds__(256, BACK ? 2 : 3)
k_norm_sums(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c, const __grid_constant__ NormTiles t) {
  wait_for_previous();
  constexpr int kRoom = (WARP ? 32 : 256) * (NC * VE + 1), kGroups = WARP ? 256 : kMostGroups;
  __shared__ float rooms[(WARP ? 8 : 1) * kRoom], results[(WARP ? 8 : 1) * kGroups];
  const int team = WARP ? threadIdx.x / 32 : 0, thread = WARP ? threadIdx.x % 32 : threadIdx.x;
  float *const room = rooms + team * kRoom, *const result = results + team * kGroups;
  const NormThread<VE, NC, GN> me(s, t, thread);
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
  const int64_t tile = (int64_t)blockIdx.x * (WARP ? 8 : 1) + team, row0 = tile * t.sum_rows, row1 = min(row0 + t.sum_rows, s.rows), step = t.lines * s.dim;
  for (int64_t seg = row0 < row1 ? segment_at(s, row0) : s.segments; seg < s.segments; ++seg) {
    const RowRange whole = segment_rows(s, seg);
    if (whole.begin >= row1) break;
    const int64_t b = max(whole.begin, row0), e = min(whole.end, row1);
    if (e <= b) continue;
    float2* const parts = c.parts + (tile + seg) * s.groups + me.group0;
    int left = (int)(e - b) - me.line;      // rows from the thread's next one on
    int64_t at = (b + me.line) * s.dim;
    constexpr int U = BACK || NC > 4 ? 2 : 4;
    if constexpr (!BACK) {
      float v[1][NC][VE], q[NC][VE];
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) v[0][j][i] = q[j][i] = 0.0f;
      float n = 0.0f;
      for (; left > 0; left -= U * t.lines, at += U * step) {
        Raw<T, VE> raw[U][NC];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && left > u * t.lines) raw[u][j] = load_raw<T, VE>(x + at + u * step + me.col[j]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (!me.mine || left <= u * t.lines) break;
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
      float sums[1][NC][GN], squares[1][NC][GN];
      sum_groups<VE, NC, GN, 1, WARP>(own, sums, room, result, me, t.slots, t.lines);
      const float share = __fdividef(1.0f, (float)(e - b) * (float)me.per);
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < GN; ++i) sums[0][j][i] *= share;
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float d = v[0][j][i] - sums[0][j][i % GN];
          own[0][j][i] = me.in[j] ? fmaf(n * d, d, q[j][i]) : 0.0f;
        }
      sum_groups<VE, NC, GN, 1, WARP>(own, squares, room, result, me, t.slots, t.lines);
      put_groups(parts, sums[0], squares[0], me);
    } else {
      float2 st[NC][GN];
      load_stats(s, t, c.stats, me, seg, st);
      float ab[2][NC][VE];
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) ab[0][j][i] = ab[1][j][i] = 0.0f;
      for (; left > 0; left -= U * t.lines, at += U * step) {
        Raw<T, VE> rx[U][NC], rg[U][NC];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j)
            if (me.in[j] && left > u * t.lines) {
              rx[u][j] = load_raw<T, VE>(x + at + u * step + me.col[j]);
              rg[u][j] = load_raw<T, VE>(grad + at + u * step + me.col[j]);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (left <= u * t.lines) break;
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            if (!me.in[j]) continue;
            float xh[VE], dz[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) xh[i] = rx[u][j].get(i), dz[i] = rg[u][j].get(i);
            normalise(xh, st[j]);
            begin_backward<T, kMaskLeft>(c, at + u * step + me.col[j], xh, dz, gamma[j], beta[j]);
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
          // one rounding, as of a single row's
          ab[0][j][i] = __fmul_rn(ab[0][j][i], gamma[j][i]), ab[1][j][i] *= gamma[j][i];
        }
      float sums[2][NC][GN];
      sum_groups<VE, NC, GN, 2, WARP>(ab, sums, room, result, me, t.slots, t.lines);
      put_groups(parts, sums[0], sums[1], me);
    }
  }
  if constexpr (BACK) {
    if (!c.columns) return;
    __syncthreads();
    put_columns<WARP>(s, c, t, me, rooms, dgamma, dbeta);
  }
}

// The pieces of each segment joined: forwards mean and 1 / deviation (zeros for a segment without rows), backwards the two means. A block has
// some groups of a segment; or, where there are many segments, eight of them, a warp each, and all of its threads those that turn out to
// be long. The first `joins` blocks join the columns' sums for dgamma and dbeta. Offsets that are none are flagged here. 5 to 9 us whatever the
// shape: a launch and a chain of four loads out of L2.
struct NormPieces {
  const float2* parts;
  int64_t first, last, tile, pitch;
  int fold;
  RowRange rows;
  float per, inv;
  __device__ __forceinline__ NormPieces(const NormShape& s, const NormCall& c, const NormTiles& t, int64_t seg, const RowRange& r)
      : parts(c.parts + seg * s.groups), first(r.begin / t.sum_rows), last((r.end - 1) / t.sum_rows), tile(t.sum_rows), pitch(s.groups), fold(t.fold), rows(r),
        per((float)s.per), inv(1.0f / ((float)(r.end - r.begin) * (float)s.per * (float)t.fold)) {}
  __device__ __forceinline__ float count(int64_t i) const { return (float)(min((i + 1) * tile, rows.end) - max(i * tile, rows.begin)) * per; }
  // of every step-th piece: the backward's sums, or the sum of the means
  template <bool BACK>
  __device__ __forceinline__ float2 sums(int g, int64_t from, int64_t step) const {
    float2 v = make_float2(0.0f, 0.0f);
    for (int f = g * fold; f < (g + 1) * fold; ++f)
#pragma unroll 4
      for (int64_t i = from; i <= last; i += step) {
        const float2 p = parts[i * pitch + f];
        if constexpr (BACK) v.x += p.x, v.y += p.y;
        else v.x = fmaf(p.x, count(i), v.x);
      }
    return v;
  }
  __device__ __forceinline__ float squares(int g, int64_t from, int64_t step, float mean) const {
    float q = 0.0f;
    for (int f = g * fold; f < (g + 1) * fold; ++f)
#pragma unroll 4
      for (int64_t i = from; i <= last; i += step) {
        const float2 p = parts[i * pitch + f];
        q += fmaf(count(i) * (p.x - mean), p.x - mean, p.y);
      }
    return q;
  }
};
constexpr int kFewPieces = 16;
template <typename T, bool BACK>
__global__ void __launch_bounds__(256)
k_norm_join(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c, const __grid_constant__ NormTiles t, int joins, int64_t lines) {
  wait_for_previous();
  if (BACK && (int)blockIdx.x < joins) {
    if (blockIdx.y == 0) join_columns<T>(s, c, blockIdx.x, lines);
    return;
  }
  __shared__ float2 part[256];
  float2* const to = BACK ? c.means : c.stats;
  const int groups = s.groups / t.fold;
  const auto put = [&](int64_t seg, int g, float a, float b, float inv) {
    to[seg * groups + g] = make_float2(a, BACK ? b * inv : rsqrtf(b * inv + c.eps));
  };
  const int64_t block = blockIdx.x - joins;
  uint32_t rest = 1;      // of the block's segments, for all its threads
  if (t.join_segments > 1) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t seg = block * t.join_segments + warp;
    int many = 0;
    if (seg < s.segments) {
      const RowRange r = segment_rows(s, seg);
      if (s.offsets && lane == 0 && bad_group(s.offsets, (int)seg, s.rows)) atomicOr(c.status, APT_FLAG_BAD_OFFSETS);
      const NormPieces p(s, c, t, seg, r);
      many = r.end > r.begin && p.last - p.first >= kFewPieces;
      if (!many)
        for (int g = lane; g < groups; g += 32) {
          if (r.end <= r.begin) {
            to[seg * groups + g] = make_float2(0.0f, 0.0f);
            continue;
          }
          const float2 v = p.sums<BACK>(g, p.first, 1);
          const float mean = v.x * p.inv;
          put(seg, g, mean, BACK ? v.y : p.squares(g, p.first, 1, mean), p.inv);
        }
    }
    if (!__syncthreads_or(many)) return;
    __shared__ uint32_t long_ones;
    if (threadIdx.x == 0) long_ones = 0;
    __syncthreads();
    if (many && lane == 0) atomicOr(&long_ones, 1u << warp);
    __syncthreads();
    rest = long_ones;
  }
  for (; rest; rest &= rest - 1) {
    const int64_t seg = block * t.join_segments + __ffs(rest) - 1;
    const RowRange r = segment_rows(s, seg);
    if (t.join_segments == 1 && s.offsets && blockIdx.y == 0 && threadIdx.x == 0 && bad_group(s.offsets, (int)seg, s.rows))
      atomicOr(c.status, APT_FLAG_BAD_OFFSETS);
    const NormPieces p(s, c, t, seg, r);
    const int width = t.join_groups, lane = threadIdx.x / width, lanes = 256 / width;
    for (int g0 = blockIdx.y * width; g0 < groups; g0 += gridDim.y * width) {
      const int g = g0 + threadIdx.x % width;
      const bool mine = g < groups && lane < lanes;
      if (r.end <= r.begin) {
        if (mine && lane == 0) to[seg * groups + g] = make_float2(0.0f, 0.0f);
        continue;
      }
      const auto together = [&](float2 v) {
        __syncthreads();
        if (mine) part[threadIdx.x] = v;
        __syncthreads();
        v = make_float2(0.0f, 0.0f);
        if (mine)
          for (int k = 0; k < lanes; ++k) v.x += part[k * width + threadIdx.x % width].x, v.y += part[k * width + threadIdx.x % width].y;
        return v;
      };
      const float2 v = together(mine ? p.sums<BACK>(g, p.first + lane, lanes) : make_float2(0.0f, 0.0f));
      const float mean = v.x * p.inv;
      float q = v.y;
      if constexpr (!BACK) q = together(make_float2(0.0f, mine ? p.squares(g, p.first + lane, lanes, mean) : 0.0f)).y;
      if (mine && lane == 0) put(seg, g, mean, q, p.inv);
    }
  }
}

// The rows themselves, and zeros for rows of no segment. Tiles from the last to the first: what k_norm_sums read last is still in L2.
// 151552 x 256 bf16 in 8 segments, silu and dropout, us: forwards 63 (HBM: 24 at most), backwards 60 (36 at most): 57 per cent of the issue slots, the integer
// pipe at half its rate. 55001 x 64 f16 in 2048 segments, gelu: 11 and 13, mostly the chain of loads in front of the first row.
template <typename T, int VE, int NC, int GN, bool BACK, bool WARP>
__global__ void __launch_bounds__(256, GN > 1 || NC > 1 ? 2 : 3)
k_norm_apply(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c, const __grid_constant__ NormTiles t) {
  wait_for_previous();
  const NormThread<VE, NC, GN> me(s, t, WARP ? threadIdx.x % 32 : threadIdx.x);
  const T* const x = (const T*)c.x;
  const T* const grad = (const T*)c.grad;
  T* const out = (T*)c.out;
  const int64_t tile = t.apply_tiles - 1 - ((int64_t)blockIdx.x * (WARP ? 8 : 1) + (WARP ? threadIdx.x / 32 : 0));
  if (tile < 0) return;
  const int64_t row0 = tile * t.apply_rows, row1 = min(row0 + t.apply_rows, s.rows), step = t.lines * s.dim;
  float gamma[NC][VE], beta[NC][VE];
  load_params<T>(c, me, gamma, beta);
  int64_t done = row0, seg = segment_at(s, row0);      // rows up to here are of segments
  if (!me.mine) return;
  for (; seg < s.segments; ++seg) {
    const RowRange whole = segment_rows(s, seg);
    if (whole.begin >= row1) break;
    const int64_t b = max(whole.begin, row0), e = min(whole.end, row1);
    if (e <= b) continue;
    if (e > done) done = e;
    float2 st[NC][GN], ab[BACK ? NC : 1][GN];
    load_stats(s, t, c.stats, me, seg, st);
    if constexpr (BACK) load_stats(s, t, c.means, me, seg, ab);
    // forwards (x - mean) (gamma / deviation) + beta
    float scale[BACK ? 1 : NC][VE];
    if constexpr (!BACK)
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) scale[j][i] = gamma[j][i] * st[j][i % GN].y;
    // two rows of single elements at once, for each slice and row has code of its own: 18305 x 319 bf16 in 1651 segments 34 us, with four rows 47; in 8
    // segments, 150000 rows, 127 and 134. One row at a time backwards: 38 for 41, but 165 for 148.
    constexpr int U = BACK || NC > 4 ? 2 : 4;
    int left = (int)(e - b) - me.line;
    for (int64_t at0 = (b + me.line) * s.dim; left > 0; left -= U * t.lines, at0 += U * step) {
      Raw<T, VE> rx[U][NC], rg[BACK ? U : 1][NC];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (me.in[j] && left > u * t.lines) {
            rx[u][j] = load_raw<T, VE>(x + at0 + u * step + me.col[j]);
            if constexpr (BACK) rg[u][j] = load_raw<T, VE>(grad + at0 + u * step + me.col[j]);
          }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (left <= u * t.lines) break;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          if (!me.in[j]) continue;
          const int64_t at = at0 + u * step + me.col[j];
          float v[VE];
          if constexpr (BACK) {
#pragma unroll
            for (int i = 0; i < VE; ++i) v[i] = rx[u][j].get(i);
            normalise(v, st[j]);
            float dz[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) dz[i] = rg[u][j].get(i);
            begin_backward<T, kMaskTaken>(c, at, v, dz, gamma[j], beta[j]);
#pragma unroll
            for (int i = 0; i < VE; ++i) dz[i] = __fmul_rn(dz[i], gamma[j][i]);
            finish_backward(v, dz, st[j], ab[j]);
          } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) v[i] = rx[u][j].get(i) - st[j][i % GN].x;
            finish_forward<T>(c, at, v, scale[j], beta[j]);
          }
          store_all<T, VE>(out + at, v);
        }
      }
    }
  }
  const float zeros[VE] = {};
  for (int64_t r = done + me.line; r < row1; r += t.lines)
#pragma unroll
    for (int j = 0; j < NC; ++j)
      if (me.in[j]) store_all<T, VE>(out + r * s.dim + me.col[j], zeros);
}

// --------------------------------------------------------------------------------------- groups of very many channels
// Rows by themselves of more than 1024 slices, and groups of segments of more than 2048 channels that cannot be cut into equal parts.
// 4096 x 8192 fp32, gelu: forwards 86 us (HBM: 41), backwards 498 (62), of which the columns 300: three walks and two, the later ones out of L2. 20000 x 2053 bf16
// in two segments 55 and 96 ms: two blocks.
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
// A sum of however many numbers: what each addition loses is kept beside it (Knuth's two-sum). One thread may have a 256th of all of a long segment's, whose
// running mean stands still, and whose squares, of few different values in 16 bits, are rounded the same way every time (1e-4 of 20000 x 2053). A sum of
// 32 (LONG false) loses nothing to speak of.
template <bool LONG>
struct LongSum {
  float sum = 0.0f, lost = 0.0f;
  __device__ __forceinline__ void add(float v) {
    if (!LONG) {
      sum += v;
      return;
    }
    const float all = sum + v, added = all - sum;
    lost += (sum - (all - added)) + (v - added);
    sum = all;
  }
  __device__ __forceinline__ float get() const { return sum + lost; }
};
template <typename T>
__device__ __forceinline__ float2 wide_xh_dz(const NormCall& c, int64_t e, int64_t col, float2 st, float* gamma) {
  const float g = *gamma = param<T>(c.weight, c.wide_params, col, 1.0f);
  float xh[1] = {(Elem<T>::to_f(((const T*)c.x)[e]) - st.x) * st.y}, dz[1] = {Elem<T>::to_f(((const T*)c.grad)[e])};
  const float gs[1] = {g}, bs[1] = {param<T>(c.bias, c.wide_params, col, 0.0f)};
  begin_backward<T, kMaskMade>(c, e, xh, dz, gs, bs);
  return make_float2(xh[0], dz[0]);
}
template <typename T, bool BACK, bool LONG>
__global__ void __launch_bounds__(256) k_norm_wide(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c) {
  wait_for_previous();
  __shared__ float shared[8];
  const T* const x = (const T*)c.x;
  T* const out = (T*)c.out;
  for (int64_t item = blockIdx.x; item < s.segments * s.groups; item += gridDim.x) {
    const int64_t seg = item / s.groups, c0 = item % s.groups * s.per;
    const RowRange r = segment_rows(s, seg);
    if (s.offsets && c0 == 0 && threadIdx.x == 0 && bad_group(s.offsets, (int)seg, s.rows)) atomicOr(c.status, APT_FLAG_BAD_OFFSETS);
    const float inv = 1.0f / ((float)(r.end - r.begin) * (float)s.per);
    const auto walk = [&](auto&& f) {
      for (int64_t row = r.begin; row < r.end; ++row)
        for (int k = threadIdx.x; k < s.per; k += 256) f(row * s.dim + c0 + k, c0 + k);
    };
    if constexpr (!BACK) {
      LongSum<LONG> all, squares;
      walk([&](int64_t e, int64_t) { all.add(Elem<T>::to_f(x[e])); });
      const float mean = block_sum(all.get(), shared) * inv;
      walk([&](int64_t e, int64_t) {
        const float d = Elem<T>::to_f(x[e]) - mean;
        squares.add(d * d);
      });
      const float rstd = rsqrtf(block_sum(squares.get(), shared) * inv + c.eps);
      if (threadIdx.x == 0) c.stats[item] = r.end > r.begin ? make_float2(mean, rstd) : make_float2(0.0f, 0.0f);
      walk([&](int64_t e, int64_t col) {
        float v[1] = {(Elem<T>::to_f(x[e]) - mean) * rstd};
        const float g[1] = {param<T>(c.weight, c.wide_params, col, 1.0f)}, b[1] = {param<T>(c.bias, c.wide_params, col, 0.0f)};
        finish_forward<T>(c, e, v, g, b);
        out[e] = Elem<T>::from_f(v[0]);
      });
    } else {
      const float2 st = c.stats[item];
      LongSum<LONG> dxhs, dxh_xhs;
      float gamma;
      walk([&](int64_t e, int64_t col) {
        const float2 v = wide_xh_dz<T>(c, e, col, st, &gamma);
        const float dxh = __fmul_rn(v.y, gamma);
        dxhs.add(dxh), dxh_xhs.add(dxh * v.x);
      });
      const float a = block_sum(dxhs.get(), shared) * inv, b = block_sum(dxh_xhs.get(), shared) * inv;
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
// Sums for dgamma and dbeta of some rows, a channel a thread.
template <typename T>
__global__ void __launch_bounds__(256) k_norm_wide_columns(const __grid_constant__ NormShape s, const __grid_constant__ NormCall c) {
  wait_for_previous();
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x, some = (s.rows + gridDim.y - 1) / gridDim.y;
  const int64_t row0 = blockIdx.y * some, row1 = min(row0 + some, s.rows);
  int64_t seg = row0 < row1 ? segment_at(s, row0) : s.segments;
  if (col >= s.dim) return;
  float dgamma = 0.0f, dbeta = 0.0f, gamma;
  for (; seg < s.segments; ++seg) {
    const RowRange r = segment_rows(s, seg);
    if (r.begin >= row1) break;
    float a = 0.0f, b = 0.0f;
    const float2 st = r.end > r.begin ? c.stats[seg * s.groups + col / s.per] : make_float2(0.0f, 0.0f);
#pragma unroll 4
    for (int64_t row = max(r.begin, row0); row < min(r.end, row1); ++row) {
      const float2 v = wide_xh_dz<T>(c, row * s.dim + col, col, st, &gamma);
      a = fmaf(v.x, v.y, a), b += v.y;
    }
    dgamma += a, dbeta += b;
  }
  c.columns[(int64_t)blockIdx.y * 2 * s.dim + col] = dgamma;
  c.columns[((int64_t)blockIdx.y * 2 + 1) * s.dim + col] = dbeta;
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
  bool warps;             // tiles by warps
};

template <typename T, int VE, bool BACK>
static int norm_rows(const NormShape& s, const NormCall& c, const NormPlan& p, cudaStream_t st) {
  const int64_t grid = p.blocks * p.chunks;
  if (p.lanes.width > 32) {
    if (p.held == 1) APT_FOLLOW((k_norm_rows<T, VE, 1, BACK ? 1 : 2, true, BACK>), grid, 256, 0, st, s, c, p.lanes);
    else if (p.held == 2) APT_FOLLOW((k_norm_rows<T, VE, 2, 1, true, BACK>), grid, 256, 0, st, s, c, p.lanes);
    else APT_FOLLOW((k_norm_rows<T, VE, 4, 1, true, BACK>), grid, 256, 0, st, s, c, p.lanes);
  } else {
    if constexpr (VE <= 2)
      if (p.held == 2) APT_FOLLOW((k_norm_rows<T, VE, 2, BACK ? 1 : 2, false, BACK>), grid, 256, 0, st, s, c, p.lanes);
    if (p.held == 1) APT_FOLLOW((k_norm_rows<T, VE, 1, BACK ? 2 : 4, false, BACK>), grid, 256, 0, st, s, c, p.lanes);
  }
  if (BACK && c.columns) APT_FOLLOW((k_norm_columns<T>), ceil_div(2 * s.dim, 32), 256, 0, st, s, c, p.blocks);
  return APT_OK;
}
template <typename T, int VE, int NC, int GN, bool BACK, bool WARP>
static int norm_tiles(const NormShape& s, const NormCall& c, const NormPlan& p, cudaStream_t st) {
  const NormTiles& t = p.tiles;
  const dim3 sums((unsigned)p.blocks, (unsigned)p.chunks), apply((unsigned)ceil_div(t.apply_tiles, WARP ? 8 : 1), (unsigned)p.chunks);
  NormShape parts = s;
  parts.groups *= t.fold, parts.per /= t.fold;
  APT_FOLLOW((k_norm_sums<T, VE, NC, GN, BACK, WARP>), sums, 256, 0, st, parts, c, t);
  const int joins = BACK && c.columns ? (int)ceil_div(2 * s.dim, 32) : 0;
  const dim3 join((unsigned)(joins + ceil_div(s.segments, t.join_segments)), t.join_segments > 1 ? 1u : (unsigned)std::min<int64_t>(65535, ceil_div(s.groups, t.join_groups)));
  APT_FOLLOW((k_norm_join<T, BACK>), join, 256, 0, st, parts, c, t, joins, p.blocks);
  APT_FOLLOW((k_norm_apply<T, VE, NC, GN, BACK, WARP>), apply, 256, 0, st, parts, c, t);
  return APT_OK;
}
template <typename T, int VE, int NC, bool BACK>
static int norm_held(const NormShape& s, const NormCall& c, const NormPlan& p, cudaStream_t st) {
  if constexpr (VE > 1)
    if (s.per / p.tiles.fold % VE) return p.warps ? norm_tiles<T, VE, NC, VE, BACK, true>(s, c, p, st) : norm_tiles<T, VE, NC, VE, BACK, false>(s, c, p, st);
  return p.warps ? norm_tiles<T, VE, NC, 1, BACK, true>(s, c, p, st) : norm_tiles<T, VE, NC, 1, BACK, false>(s, c, p, st);
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
    // a thread's share of a row of up to 8192 channels is a sum of 32: 4096 x 8192 fp32, forwards, gelu 86 us, 97 with what additions lose kept beside
    const int64_t grid = wave_grid(s.segments * s.groups, 8);
    if (s.rows && !s.offsets && s.per_segment == 1 && s.per <= 32 * 256) APT_FOLLOW((k_norm_wide<T, BACK, false>), grid, 256, 0, st, s, c);
    else if (s.rows) APT_FOLLOW((k_norm_wide<T, BACK, true>), grid, 256, 0, st, s, c);
    if (BACK && c.columns) {
      APT_FOLLOW((k_norm_wide_columns<T>), dim3((unsigned)ceil_div(s.dim, 256), (unsigned)p.blocks), 256, 0, st, s, c);
      APT_FOLLOW((k_norm_columns<T>), ceil_div(2 * s.dim, 32), 256, 0, st, s, c, p.blocks);
    }
    return APT_OK;
  }
  if (p.slice == 16 / (int)sizeof(T)) return norm_slices<T, 16 / (int)sizeof(T), BACK>(s, c, p, st);
  if (p.slice == 8 / (int)sizeof(T)) return norm_slices<T, 8 / (int)sizeof(T), BACK>(s, c, p, st);
  if constexpr (sizeof(T) == 2)
    if (p.slice == 2) return norm_slices<T, 2, BACK>(s, c, p, st);
  return norm_slices<T, 1, BACK>(s, c, p, st);
}

}  // namespace apt
