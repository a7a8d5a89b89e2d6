// Group norm with an activation: what kernels a call takes, and its entry points. The kernels (group_norm.cuh) are compiled a type a file.
#include "group_norm.cuh"

namespace apt {

extern template int norm<float, false>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
extern template int norm<float, true>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
extern template int norm<__nv_bfloat16, false>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
extern template int norm<__nv_bfloat16, true>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
extern template int norm<__half, false>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
extern template int norm<__half, true>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);

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
  t.chunk = chunk;
  p.chunks = ceil_div(s.groups, chunk);
  // Short segments by warps where there are enough to fill the chip and a warp holds a row; by blocks where there are fewer. Where the mean
  // is well above what those do whole, nothing is looked for and all segments are long.
  p.held = slices <= 256 ? 1 : 8 / p.slice;
  p.warps = p.chunks == 1 && slices <= 32 * (8 / p.slice) && s.segments >= kNumSMs * 8;
  if (p.warps) p.held = slices <= 32 ? 1 : 8 / p.slice;
  t.slots = (int)ceil_div(slices, p.held);
  t.lines = t.slots <= 32 ? 8 * (32 / t.slots) : 256 / t.slots;
  const int rows = held_rows(back, p.held);
  t.cap = p.warps ? rows * (t.lines / 8) * kWarpChunks : rows * t.lines;
  if (s.rows / s.segments > 4 * (int64_t)t.cap) t.cap = 0;
  t.short_blocks = t.cap ? (int)std::min<int64_t>(p.warps ? ceil_div(s.segments, 8) : s.segments, kNumSMs * 4) : 0;
  // one round of blocks, of eight rounds of rows at least
  const int64_t blocks = ceil_div(kNumSMs * (t.cap || back ? 2 : 4), p.chunks);
  t.tile = std::max<int64_t>(8 * t.lines, ceil_div(ceil_div(s.rows, blocks), t.lines) * t.lines);
  t.tiles = ceil_div(s.rows, t.tile);
  p.blocks = t.tiles + t.short_blocks;
  return p;
}

static size_t norm_room(const NormShape& s, const NormPlan& p, bool back) {
  const size_t columns = back && p.kind != kNormWide ? align_up((size_t)p.blocks * 2 * s.dim * 4, 256) : 0;
  return columns + (p.kind == kNormTiles ? (size_t)(p.tiles.tiles + s.segments) * s.groups * 8 : 0);
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
