// What the operators of a layer's dense half share: the generator of dropout, activations with their derivatives, and ragged groups
// of rows whose ends are on the device.
#pragma once

#include "rows.cuh"

namespace apt {

// ---- dropout --------------------------------------------------------------------
// Word i of the stream (key, call) decides on element i, counted row by row: Philox4x32-10 with counter (i / 4 low, i / 4 high, call,
// "drop"), word i % 4. So the mask is a function of numbers that forward and backward both have, whatever kernel makes it, and is never
// stored. An element goes where its word is below threshold = floor(p 2^32).
struct Drop {
  uint32_t key_low, key_high, call, threshold;
  float scale;      // 1 / (1 - p); 0: everything goes
};
constexpr uint32_t kDropTag = 0x64726f70u;

// p in [0, 1] (checked by the caller).
inline Drop make_drop(double p, uint64_t key, uint32_t call) {
  const bool all = p >= 1.0;
  return {(uint32_t)key, (uint32_t)(key >> 32), call, all ? 0u : (uint32_t)(p * 4294967296.0), all ? 0.0f : (float)(1.0 / (1.0 - p))};
}

__device__ __forceinline__ Philox4 drop_words(const Drop& d, int64_t quad) {
  return philox4x32_10((uint32_t)quad, (uint32_t)((uint64_t)quad >> 32), d.call, kDropTag, d.key_low, d.key_high);
}
// An element that goes is zero whatever it was, infinities and NaN among it.
__device__ __forceinline__ float dropped(const Drop& d, uint32_t word, float v) {
  return word >= d.threshold && d.scale != 0.0f ? v * d.scale : 0.0f;
}

// ---- activations ----------------------------------------------------------------
// A NaN stays one, in relu too.
template <int ACT>
__device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == APT_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if constexpr (ACT == APT_ACT_SILU) return z / (1.0f + expf(-z));
  if constexpr (ACT == APT_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == APT_ACT_RELU) return z <= 0.0f ? 0.0f : 1.0f;
  if constexpr (ACT == APT_ACT_SILU) {
    const float s = 1.0f / (1.0f + expf(-z));
    return s * (1.0f + z * (1.0f - s));
  }
  if constexpr (ACT == APT_ACT_GELU)
    return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
  return 1.0f;
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

}  // namespace apt
