// What the operators of a layer's dense half share: the generator of dropout, activations with their derivatives, and ragged groups
// of rows whose ends are on the device.
#pragma once

#include "rows.cuh"

namespace apt {

// ---- dropout --------------------------------------------------------------------
// Word i of the stream (key, call) decides on element i, counted row by row: Philox4x32-10 with counter (i / 4 low, i / 4 high, call,
// "drop"), word i % 4. So the mask is a function of numbers that forward and backward both have, whatever kernel makes it, and is never
// stored. An element goes where its word is below threshold = floor(p 2^32).
//
// What the first two rounds make of the numbers that are the same for all elements (the call, the tag, and the upper word of the quad's
// number while it is 0) is worked out on the host, and so are the rounds' keys: 18 products and 19 logical operations a quad instead of 20,
// 20 and 20 additions (151552 x 256 bf16, both ways: 81 -> 79 us). A product of 32 by 32 bits takes its pipe for four cycles a warp, so that the
// words alone of that matrix are 29 us, as long as reading and writing it; the upper half from a product in 64-bit floating point took 33.
struct Drop {
  uint32_t k0[10], k1[10];      // the rounds' keys
  uint32_t a0, a1, a2;          // behind the first round: the first word but for the quad's upper one, the second, part of the third
  uint32_t b2, b3;              // behind the second: part of the third, the fourth
  uint32_t threshold;
  float scale;                  // 1 / (1 - p); 0: everything goes
};
constexpr uint32_t kDropTag = 0x64726f70u, kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u;

// p in [0, 1] (checked by the caller).
inline Drop make_drop(double p, uint64_t key, uint32_t call) {
  Drop d;
  for (int r = 0; r < 10; ++r) d.k0[r] = (uint32_t)key + r * 0x9E3779B9u, d.k1[r] = (uint32_t)(key >> 32) + r * 0xBB67AE85u;
  const uint64_t first = (uint64_t)kPhiloxM1 * call;
  d.a0 = (uint32_t)(first >> 32) ^ d.k0[0], d.a1 = (uint32_t)first, d.a2 = kDropTag ^ d.k1[0];
  const uint64_t second = (uint64_t)kPhiloxM0 * d.a0;
  d.b2 = (uint32_t)(second >> 32), d.b3 = (uint32_t)second;
  const bool all = p >= 1.0;
  d.threshold = all ? 0u : (uint32_t)(p * 4294967296.0);
  d.scale = all ? 0.0f : (float)(1.0 / (1.0 - p));
  return d;
}

__device__ __forceinline__ Philox4 drop_words(const Drop& d, int64_t quad) {
  uint64_t p = (uint64_t)kPhiloxM0 * (uint32_t)quad, q;
  uint32_t c2 = (uint32_t)(p >> 32) ^ d.a2, c3 = (uint32_t)p, b2 = d.b2, b3 = d.b3;
  const uint32_t upper = (uint32_t)((uint64_t)quad >> 32);
  if (upper) {
    p = (uint64_t)kPhiloxM0 * (d.a0 ^ upper);
    b2 = (uint32_t)(p >> 32), b3 = (uint32_t)p;
  }
  q = (uint64_t)kPhiloxM1 * c2;
  uint32_t c0 = (uint32_t)(q >> 32) ^ d.a1 ^ d.k0[1], c1 = (uint32_t)q;
  c2 = b2 ^ c3 ^ d.k1[1], c3 = b3;
#pragma unroll
  for (int r = 2; r < 10; ++r) {
    p = (uint64_t)kPhiloxM0 * c0, q = (uint64_t)kPhiloxM1 * c2;
    c0 = (uint32_t)(q >> 32) ^ c1 ^ d.k0[r], c2 = (uint32_t)(p >> 32) ^ c3 ^ d.k1[r];
    c1 = (uint32_t)q, c3 = (uint32_t)p;
  }
  return {{c0, c1, c2, c3}};
}
// An element that goes is zero whatever it was, infinities and NaN among it.
__device__ __forceinline__ float dropped(const Drop& d, uint32_t word, float v) {
  return word >= d.threshold && d.scale != 0.0f ? v * d.scale : 0.0f;
}

// ---- activations ----------------------------------------------------------------
// Exponential and reciprocal are single instructions, off by two units in the last place and one (and the exponential by |z| units more
// for its rounded argument, which counts where silu and the normal density are small); results below 2^-126 are zero. With the
// functions that take denormals, silu is 20 instructions instead of 5, in kernels that their instructions bound.
__device__ __forceinline__ float exp2_short(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float logistic(float z) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + exp2_short(-1.4426950408889634f * z)));
  return r;
}
// The normal distribution's mass below z, given q = exp(-z z / 2), which the density needs too: the tail beyond |z| is q times a polynomial in
// t = 1 / (1 + c |z|) without a constant term, fitted to erfcx(|z| / sqrt 2) / 2 for the least largest relative error on |z| <= 14 (a linear programme over
// 1500 points), so that gelu keeps its digits where it is small; what it is off there comes from q. fp32: nine terms, 1e-8 (in fp32 arithmetic 4e-7).
// T of 16 bits: seven, 9e-7 (1.2e-6). The library's error function takes 30 instructions and a branch, these 14 and 12, and 1 + erf is 2.7e-4 off at
// z = -4. Abramowitz and Stegun's 7.1.26, which bounds the error of erf and not of the tail, is one instruction less than the shorter one and is 5e-5 off
// at -3, 5e-4 at -4, 4e-3 at -6.
template <typename T>
__device__ __forceinline__ float normal_below(float z, float q) {
  constexpr bool kLong = sizeof(T) == 4;
  float t;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(kLong ? 0.35f : 0.36f, fabsf(z), 1.0f)));
  float p;
  if constexpr (kLong) {
    p = fmaf(-0.0287085366f, t, 0.142167712f);
    p = fmaf(p, t, -0.252693937f);
    p = fmaf(p, t, 0.156555375f);
    p = fmaf(p, t, -0.0218758071f);
    p = fmaf(p, t, 0.105213384f);
    p = fmaf(p, t, 0.119856455f);
    p = fmaf(p, t, 0.139864332f);
    p = fmaf(p, t, 0.139621022f);
  } else {
    p = fmaf(0.047022188f, t, -0.179647118f);
    p = fmaf(p, t, 0.180795716f);
    p = fmaf(p, t, 0.0266545596f);
    p = fmaf(p, t, 0.139683226f);
    p = fmaf(p, t, 0.141778465f);
    p = fmaf(p, t, 0.143712663f);
  }
  const float tail = q * (p * t);
  return z < 0.0f ? tail : 1.0f - tail;
}
// A NaN stays one, in relu too.
template <typename T, int ACT>
__device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == APT_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if constexpr (ACT == APT_ACT_SILU) return z * logistic(z);
  if constexpr (ACT == APT_ACT_GELU) return z * normal_below<T>(z, exp2_short(-0.72134752044448170f * z * z));
  return z;
}
template <typename T, int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == APT_ACT_RELU) return z <= 0.0f ? 0.0f : 1.0f;
  if constexpr (ACT == APT_ACT_SILU) {
    const float s = logistic(z);
    return fmaf(s * z, 1.0f - s, s);
  }
  if constexpr (ACT == APT_ACT_GELU) {
    const float q = exp2_short(-0.72134752044448170f * z * z);
    return fmaf(0.39894228040143268f * z, q, normal_below<T>(z, q));
  }
  return 1.0f;
}

// Two 16-bit elements, rounded by one instruction.
template <typename T>
__device__ __forceinline__ uint32_t rounded_pair(float a, float b) {
  if constexpr (Elem<T>::kIsBf16) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&r;
  } else {
    const __half2 r = __floats2half2_rn(a, b);
    return *(const uint32_t*)&r;
  }
}
// A 16-byte slice of elements from v on, rounded.
template <typename T>
__device__ __forceinline__ uint4 rounded_slice(const float* v) {
  if constexpr (sizeof(T) == 4) return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  else return make_uint4(rounded_pair<T>(v[0], v[1]), rounded_pair<T>(v[2], v[3]), rounded_pair<T>(v[4], v[5]), rounded_pair<T>(v[6], v[7]));
}
// N neighbouring elements, rounded.
template <typename T, int N>
__device__ __forceinline__ void store_all(T* p, const float (&v)[N]) {
  if constexpr (N * sizeof(T) == 16) {
    *(uint4*)p = rounded_slice<T>(v);
  } else {
    Pack<T, N> r;
#pragma unroll
    for (int k = 0; k < N; ++k) r.v[k] = Elem<T>::from_f(v[k]);
    store_pack<T, N>(p, r);
  }
}

// ---- ragged groups --------------------------------------------------------------
// Group g has the rows [offsets[g], offsets[g + 1]). Ends that do not ascend, begin elsewhere than at 0 or lie beyond the rows are
// flagged, and whatever they are no row outside [0, rows) is touched.
struct RowRange {
  int64_t begin, end;
};
__device__ __forceinline__ RowRange group_rows(const int64_t* offsets, int g, int64_t rows) {
  const int64_t b = min(max(offsets[g], (int64_t)0), rows);
  return {b, min(max(offsets[g + 1], b), rows)};
}
__device__ __forceinline__ bool bad_group(const int64_t* offsets, int g, int64_t rows) {
  return offsets[g + 1] < offsets[g] || offsets[g + 1] > rows || (g == 0 && offsets[0] != 0);
}
// The same of all groups, where there are no rows and so no kernel that looks at them (group_norm.cu).
int look_at_ends(const int64_t* offsets, int64_t groups, int64_t rows, int32_t* status, cudaStream_t s);

}  // namespace apt
