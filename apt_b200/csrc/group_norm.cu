// Group norm with an activation and dropout behind it, channels last.
//
// A segment of rows (each row, equal blocks of rows, or ragged groups) and a group of neighbouring channels have one mean and one
// variance. xh = (x - mean) rstd, z = xh gamma + beta, y = drop(act(z)); backwards dz = drop(dy) act'(z), dgamma = sum dz xh,
// dbeta = sum dz, and with dxh = dz gamma: dx = rstd (dxh - mean(dxh) - xh mean(dxh xh)).
// Everything is held in 32 bits; the variance is taken around the mean, in a second walk, so that a mean far from zero costs nothing.
#include "dense.cuh"

namespace apt {

struct NormShape {
  int64_t rows, dim, segments, per_segment;      // per_segment: rows of each where there are no offsets
  const int64_t* offsets;
  int groups, per;                               // channels of a group
};
__device__ __forceinline__ RowRange segment_rows(const NormShape& s, int64_t k) {
  if (s.offsets) return group_rows(s.offsets, (int)k, s.rows);
  return {k * s.per_segment, (k + 1) * s.per_segment};
}
// The segment of a row, -1: of none.
__device__ __forceinline__ int64_t segment_of(const NormShape& s, int64_t row) {
  if (!s.offsets) return row / s.per_segment;
  int64_t lo = 0, hi = s.segments;
  while (lo < hi) {
    const int64_t m = (lo + hi) / 2;
    if (s.offsets[m + 1] <= row) lo = m + 1; else hi = m;
  }
  return lo < s.segments && s.offsets[lo] <= row ? lo : -1;
}

__device__ __forceinline__ float block_sum(float v, float* shared) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) shared[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.0f;
  for (int k = 0; k < (int)blockDim.x / 32; ++k) v += shared[k];
  return v;
}

template <typename T>
__global__ void __launch_bounds__(256) k_norm_stats(const T* __restrict__ x, const __grid_constant__ NormShape s, float eps, float2* __restrict__ stats,
                                                    int32_t* status) {
  wait_for_previous();
  __shared__ float shared[8];
  for (int64_t item = blockIdx.x; item < s.segments * s.groups; item += gridDim.x) {
    const int64_t seg = item / s.groups, g = item % s.groups;
    const RowRange r = segment_rows(s, seg);
    if (s.offsets && g == 0 && threadIdx.x == 0 && bad_group(s.offsets, (int)seg, s.rows)) atomicOr(status, APT_FLAG_BAD_OFFSETS);
    const int64_t n = (r.end - r.begin) * s.per;
    float sum = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += 256) sum += Elem<T>::to_f(x[(r.begin + i / s.per) * s.dim + g * s.per + i % s.per]);
    const float mean = block_sum(sum, shared) / (float)n;
    sum = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += 256) {
      const float d = Elem<T>::to_f(x[(r.begin + i / s.per) * s.dim + g * s.per + i % s.per]) - mean;
      sum += d * d;
    }
    const float var = block_sum(sum, shared) / (float)n;
    if (threadIdx.x == 0) stats[item] = make_float2(mean, rsqrtf(var + eps));
  }
}

template <typename P>
__device__ __forceinline__ float param(const P* p, int64_t c, float otherwise) { return p ? Elem<P>::to_f(p[c]) : otherwise; }

template <typename T, typename P, int ACT>
__global__ void __launch_bounds__(256)
k_norm_apply(const T* __restrict__ x, const __grid_constant__ NormShape s, const float2* __restrict__ stats, const P* weight, const P* bias,
             bool drop, const __grid_constant__ Drop d, T* __restrict__ out) {
  wait_for_previous();
  for (int64_t row = blockIdx.x; row < s.rows; row += gridDim.x) {
    const int64_t seg = segment_of(s, row);
    for (int64_t c = threadIdx.x; c < s.dim; c += 256) {
      const int64_t e = row * s.dim + c;
      float y = 0.0f;
      if (seg >= 0) {
        const float2 st = stats[seg * s.groups + c / s.per];
        y = act_of<ACT>((Elem<T>::to_f(x[e]) - st.x) * st.y * param(weight, c, 1.0f) + param(bias, c, 0.0f));
        if (drop) y = dropped(d, drop_words(d, e >> 2).w[e & 3], y);
      }
      out[e] = Elem<T>::from_f(y);
    }
  }
}

// xh and dz of an element.
template <typename T, typename P, int ACT>
__device__ __forceinline__ float2 xh_dz(const T* x, const T* grad, int64_t e, int64_t c, float2 st, const P* weight, const P* bias, bool drop, const Drop& d) {
  const float xh = (Elem<T>::to_f(x[e]) - st.x) * st.y;
  float g = Elem<T>::to_f(grad[e]);
  if (drop) g = dropped(d, drop_words(d, e >> 2).w[e & 3], g);
  return make_float2(xh, g * act_slope<ACT>(xh * param(weight, c, 1.0f) + param(bias, c, 0.0f)));
}

// means of dxh and of dxh xh for each segment and group
template <typename T, typename P, int ACT>
__global__ void __launch_bounds__(256)
k_norm_means(const T* __restrict__ x, const T* __restrict__ grad, const __grid_constant__ NormShape s, const float2* __restrict__ stats, const P* weight,
             const P* bias, bool drop, const __grid_constant__ Drop d, float2* __restrict__ means) {
  wait_for_previous();
  __shared__ float shared[8];
  for (int64_t item = blockIdx.x; item < s.segments * s.groups; item += gridDim.x) {
    const int64_t seg = item / s.groups, g = item % s.groups;
    const RowRange r = segment_rows(s, seg);
    const int64_t n = (r.end - r.begin) * s.per;
    float a = 0.0f, b = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += 256) {
      const int64_t c = g * s.per + i % s.per;
      const float2 v = xh_dz<T, P, ACT>(x, grad, (r.begin + i / s.per) * s.dim + c, c, stats[item], weight, bias, drop, d);
      const float dxh = __fmul_rn(v.y, param(weight, c, 1.0f));
      a += dxh;
      b += dxh * v.x;
    }
    a = block_sum(a, shared);
    b = block_sum(b, shared);
    if (threadIdx.x == 0) means[item] = make_float2(a / (float)n, b / (float)n);
  }
}

template <typename T, typename P, int ACT>
__global__ void __launch_bounds__(256)
k_norm_grad(const T* __restrict__ x, const T* __restrict__ grad, const __grid_constant__ NormShape s, const float2* __restrict__ stats,
            const float2* __restrict__ means, const P* weight, const P* bias, bool drop, const __grid_constant__ Drop d, T* __restrict__ grad_x) {
  wait_for_previous();
  for (int64_t row = blockIdx.x; row < s.rows; row += gridDim.x) {
    const int64_t seg = segment_of(s, row);
    for (int64_t c = threadIdx.x; c < s.dim; c += 256) {
      const int64_t e = row * s.dim + c;
      float dx = 0.0f;
      if (seg >= 0) {
        const float2 st = stats[seg * s.groups + c / s.per], m = means[seg * s.groups + c / s.per];
        const float2 v = xh_dz<T, P, ACT>(x, grad, e, c, st, weight, bias, drop, d);
        // the product as the means have it, rounded by itself: a group of one element has a gradient of zero
        dx = st.y * (__fmul_rn(v.y, param(weight, c, 1.0f)) - m.x - v.x * m.y);
      }
      grad_x[e] = Elem<T>::from_f(dx);
    }
  }
}

template <typename T, typename P, int ACT>
__global__ void __launch_bounds__(256)
k_norm_params(const T* __restrict__ x, const T* __restrict__ grad, const __grid_constant__ NormShape s, const float2* __restrict__ stats, const P* weight,
              const P* bias, bool drop, const __grid_constant__ Drop d, P* grad_weight, P* grad_bias) {
  wait_for_previous();
  __shared__ float shared[8];
  const int64_t c = blockIdx.x;
  float a = 0.0f, b = 0.0f;
  for (int64_t row = threadIdx.x; row < s.rows; row += 256) {
    const int64_t seg = segment_of(s, row);
    if (seg < 0) continue;
    const float2 v = xh_dz<T, P, ACT>(x, grad, row * s.dim + c, c, stats[seg * s.groups + c / s.per], weight, bias, drop, d);
    a += v.y * v.x;
    b += v.y;
  }
  a = block_sum(a, shared);
  b = block_sum(b, shared);
  if (threadIdx.x == 0 && grad_weight) grad_weight[c] = Elem<P>::from_f(a);
  if (threadIdx.x == 0 && grad_bias) grad_bias[c] = Elem<P>::from_f(b);
}

struct NormCall {
  const void *x, *grad, *weight, *bias;
  void *out, *grad_weight, *grad_bias;      // out: y, or the gradient of x
  float2 *stats, *means;
  float eps;
  bool drop;
  Drop d;
  int32_t* status;
};

template <typename T, typename P, int ACT>
static int norm_forward(const NormShape& s, const NormCall& c, cudaStream_t st) {
  APT_FOLLOW((k_norm_stats<T>), wave_grid(s.segments * s.groups, 8), 256, 0, st, (const T*)c.x, s, c.eps, c.stats, c.status);
  APT_FOLLOW((k_norm_apply<T, P, ACT>), wave_grid(s.rows, 8), 256, 0, st, (const T*)c.x, s, (const float2*)c.stats, (const P*)c.weight, (const P*)c.bias,
             c.drop, c.d, (T*)c.out);
  return APT_OK;
}
template <typename T, typename P, int ACT>
static int norm_backward(const NormShape& s, const NormCall& c, cudaStream_t st) {
  const T *x = (const T*)c.x, *g = (const T*)c.grad;
  const P *w = (const P*)c.weight, *b = (const P*)c.bias;
  const float2 *stats = c.stats, *means = c.means;
  if (s.rows) {
    APT_FOLLOW((k_norm_means<T, P, ACT>), wave_grid(s.segments * s.groups, 8), 256, 0, st, x, g, s, stats, w, b, c.drop, c.d, c.means);
    APT_FOLLOW((k_norm_grad<T, P, ACT>), wave_grid(s.rows, 8), 256, 0, st, x, g, s, stats, means, w, b, c.drop, c.d, (T*)c.out);
  }
  if (c.grad_weight || c.grad_bias)
    APT_FOLLOW((k_norm_params<T, P, ACT>), s.dim, 256, 0, st, x, g, s, stats, w, b, c.drop, c.d, (P*)c.grad_weight, (P*)c.grad_bias);
  return APT_OK;
}

template <typename T, typename P>
static int norm(const NormShape& s, const NormCall& c, int act, cudaStream_t st) {
  const bool back = c.grad;
  switch (act) {
    case APT_ACT_NONE: return back ? norm_backward<T, P, APT_ACT_NONE>(s, c, st) : norm_forward<T, P, APT_ACT_NONE>(s, c, st);
    case APT_ACT_RELU: return back ? norm_backward<T, P, APT_ACT_RELU>(s, c, st) : norm_forward<T, P, APT_ACT_RELU>(s, c, st);
    case APT_ACT_SILU: return back ? norm_backward<T, P, APT_ACT_SILU>(s, c, st) : norm_forward<T, P, APT_ACT_SILU>(s, c, st);
    default: return back ? norm_backward<T, P, APT_ACT_GELU>(s, c, st) : norm_forward<T, P, APT_ACT_GELU>(s, c, st);
  }
}
static int norm_typed(int dtype, int param_dtype, const NormShape& s, const NormCall& c, int act, cudaStream_t st) {
  if (dtype == APT_F32) return norm<float, float>(s, c, act, st);
  if (dtype == APT_BF16) return param_dtype == APT_F32 ? norm<__nv_bfloat16, float>(s, c, act, st) : norm<__nv_bfloat16, __nv_bfloat16>(s, c, act, st);
  return param_dtype == APT_F32 ? norm<__half, float>(s, c, act, st) : norm<__half, __half>(s, c, act, st);
}

static int norm_check(const char* who, int dtype, int param_dtype, int64_t rows, int64_t dim, int groups, const int64_t* offsets, int64_t segments,
                      double eps, int act, double p) {
  APT_CHECK_ARG(dtype == APT_F32 || dtype == APT_BF16 || dtype == APT_F16, "%s: unsupported dtype %d", who, dtype);
  APT_CHECK_ARG(param_dtype == dtype || param_dtype == APT_F32, "%s: parameters of type %d beside type %d", who, param_dtype, dtype);
  APT_CHECK_ARG(rows >= 0 && dim > 0 && dim < (1 << 30) && groups > 0 && dim % groups == 0, "%s: %lld channels in %d groups", who, (long long)dim, groups);
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

extern "C" size_t apt_group_norm_workspace_bytes(int64_t rows, int64_t dim, int groups, int64_t segments, int backward) {
  if (rows < 0 || dim <= 0 || groups <= 0 || segments < 0) return 0;
  return apt::align_up((size_t)segments * groups * 8, 256);
}

extern "C" int apt_group_norm_forward(int dtype, int param_dtype, const void* x, int64_t rows, int64_t dim, int groups, const int64_t* offsets,
                                      int64_t segments, double eps, int act, const void* weight, const void* bias, double p, uint64_t key,
                                      uint32_t call_id, void* out, float* stats, void* workspace, size_t workspace_bytes, int32_t* status_word,
                                      void* stream) {
  using namespace apt;
  if (const int e = norm_check("apt_group_norm_forward", dtype, param_dtype, rows, dim, groups, offsets, segments, eps, act, p)) return e;
  if (rows == 0) return APT_OK;
  APT_CHECK_ARG(x && out && status_word && stats, "apt_group_norm_forward: null buffer");
  APT_CHECK_ARG(workspace && workspace_bytes >= apt_group_norm_workspace_bytes(rows, dim, groups, segments, 0), "apt_group_norm_forward: workspace too small");
  const NormCall c{x, nullptr, weight, bias, out, nullptr, nullptr, (float2*)stats, nullptr, (float)eps, p > 0.0, make_drop(p, key, call_id), status_word};
  return norm_typed(dtype, param_dtype, norm_shape(rows, dim, groups, offsets, segments), c, act, (cudaStream_t)stream);
}

extern "C" int apt_group_norm_backward(int dtype, int param_dtype, const void* x, const void* grad_out, int64_t rows, int64_t dim, int groups,
                                       const int64_t* offsets, int64_t segments, double eps, int act, const void* weight, const void* bias, double p,
                                       uint64_t key, uint32_t call_id, const float* stats, void* grad_x, void* grad_weight, void* grad_bias,
                                       void* workspace, size_t workspace_bytes, int32_t* status_word, void* stream) {
  using namespace apt;
  if (const int e = norm_check("apt_group_norm_backward", dtype, param_dtype, rows, dim, groups, offsets, segments, eps, act, p)) return e;
  APT_CHECK_ARG(status_word && (rows == 0 || (x && grad_out && grad_x && stats)), "apt_group_norm_backward: null buffer");
  APT_CHECK_ARG(workspace && workspace_bytes >= apt_group_norm_workspace_bytes(rows, dim, groups, segments, 1), "apt_group_norm_backward: workspace too small");
  const int any = 0;      // no rows: the parameters' gradients are written all the same
  const NormCall c{x, grad_out ? grad_out : &any, weight, bias, grad_x, grad_weight, grad_bias, (float2*)stats, (float2*)workspace, (float)eps, p > 0.0,
                   make_drop(p, key, call_id), status_word};
  return norm_typed(dtype, param_dtype, norm_shape(rows, dim, groups, offsets, segments), c, act, (cudaStream_t)stream);
}
