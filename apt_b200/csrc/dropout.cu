// Dropout whose mask is made anew wherever it is needed.
//
// y = x / (1 - p) where the element's word is at least p 2^32, else 0; the gradient is the same map. Nothing but x is read and nothing
// but y is written. 151552 x 256 bf16: 41 us (155 MB; a copy takes 24 to 28), bound by the generator's integer products and logic, 29 us of them:
// 63 per cent of the issue slots and 60 of the integer pipes' cycles.
#include "dense.cuh"

namespace apt {

// A thread has quads of elements, whose words one call of the generator makes.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_dropout(const T* __restrict__ in, int64_t n, const __grid_constant__ Drop d, T* __restrict__ out) {
  wait_for_previous();
  constexpr int VE = 16 / sizeof(T);
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VE; i < n; i += (int64_t)gridDim.x * 256 * VE) {
    if (VEC && i + VE <= n) {
      const Raw<T, VE> v = load_raw<T, VE>(in + i);
      float r[VE];
#pragma unroll
      for (int q = 0; q < VE / 4; ++q) {
        const Philox4 w = drop_words(d, (i >> 2) + q);
#pragma unroll
        for (int k = 0; k < 4; ++k) r[4 * q + k] = dropped(d, w.w[k], v.get(4 * q + k));
      }
      store_all<T, VE>(out + i, r);
    } else {
      for (int q = 0; q < VE / 4; ++q) {
        const Philox4 w = drop_words(d, (i >> 2) + q);
        for (int k = 0; k < 4; ++k) {
          const int64_t e = i + 4 * q + k;
          if (e < n) out[e] = Elem<T>::from_f(dropped(d, w.w[k], Elem<T>::to_f(in[e])));
        }
      }
    }
  }
}

template <typename T>
static int dropout(const void* in, int64_t n, const Drop& d, void* out, cudaStream_t s) {
  const int64_t blocks = ceil_div(n, 256 * (16 / (int64_t)sizeof(T)));
  if (((uintptr_t)in | (uintptr_t)out) % 16 == 0)
    APT_FOLLOW((k_dropout<T, true>), wave_grid(blocks, 8), 256, 0, s, (const T*)in, n, d, (T*)out);
  else
    APT_FOLLOW((k_dropout<T, false>), wave_grid(blocks, 8), 256, 0, s, (const T*)in, n, d, (T*)out);
  return APT_OK;
}

}  // namespace apt

extern "C" int apt_dropout(int dtype, const void* in, int64_t n, double p, uint64_t key, uint32_t call_id, void* out, void* stream) {
  using namespace apt;
  APT_CHECK_ARG(dtype == APT_F32 || dtype == APT_BF16 || dtype == APT_F16, "apt_dropout: unsupported dtype %d", dtype);
  APT_CHECK_ARG(n >= 0 && (n == 0 || (in && out)), "apt_dropout: null buffer or negative size");
  APT_CHECK_ARG(p >= 0.0 && p <= 1.0, "apt_dropout: p = %g is no probability", p);
  if (n == 0) return APT_OK;
  const Drop d = make_drop(p, key, call_id);
  const cudaStream_t s = (cudaStream_t)stream;
  if (dtype == APT_F32) return dropout<float>(in, n, d, out, s);
  if (dtype == APT_BF16) return dropout<__nv_bfloat16>(in, n, d, out, s);
  return dropout<__half>(in, n, d, out, s);
}
