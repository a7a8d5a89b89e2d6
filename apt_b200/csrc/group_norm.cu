// Group norm with an activation: what kernels a call takes, and its entry points. The kernels (group_norm.cuh) are compiled a type a file.
#include "group_norm.cuh"

namespace apt {

extern template int norm<float, false>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
extern template int norm<float, true>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
extern template int norm<__nv_bfloat16, false>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
extern template int norm<__nv_bfloat16, true>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
extern template int norm<__half, false>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
extern template int norm<__half, true>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);

__global__ void __launch_bounds__(256) k_look_at_ends(const int64_t* __restrict__ offsets, int groups, int64_t rows, int32_t* status) {
  wait_for_previous();
  const int g = blockIdx.x * 256 + threadIdx.x;
  if (g < groups && bad_group(offsets, g, rows)) atomicOr(status, APT_FLAG_BAD_OFFSETS);
}
int look_at_ends(const int64_t* offsets, int64_t groups, int64_t rows, int32_t* status, cudaStream_t s) {
  if (offsets && groups > 0 && status) APT_FOLLOW(k_look_at_ends, ceil_div(groups, 256), 256, 0, s, offsets, (int)groups, rows, status);
  return APT_OK;
}

// Elements of an access that `run` elements from any of the addresses on are a whole number of: 16, 8 or 4 bytes, or one.
static int slice_of(int64_t run, size_t size, uintptr_t addresses) {
  for (const int bytes : {16, 8, 4})
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
      // Rows of more slices than a warp's lanes are several warps', as few as will do: us backwards (forwards), 131072 x 512 bf16 with 64 lanes
      // 149 (82), a warp with two slices a lane 236 (100); 65536 x 1024 bf16 with 128 lanes 215 (88), with 256 399 (127). Slices of one or two
      // elements are little work for the barriers: two a lane of a warp (657930 x 102 fp32 291 (182), with 64 lanes 336 (188)), then four a lane of 128
      // up to 512 (187980 x 357 bf16 430 (257), with 256 lanes 609 (385)).
      if (slices > (p.slice <= 2 ? 64 : 32))
        while (w < (p.slice <= 2 && slices <= 512 ? 128 : 256) && w < slices) w *= 2;
      p.held = (int)ceil_div(slices, w);
      if (p.held == 3) p.held = 4;
      p.lanes.width = w;
      p.lanes.groups = (int)std::min<int64_t>(s.groups, 256 / w);
      p.lanes.rows = 256 / (w * p.lanes.groups);
      p.chunks = ceil_div(s.groups, p.lanes.groups);
      p.blocks = std::max<int64_t>(1, std::min<int64_t>(ceil_div(s.rows, p.lanes.rows * (back ? 2 : 4)), ceil_div(kNumSMs * (back ? 4 : 8), p.chunks)));
      p.lanes.blocks = (int)p.blocks;
      return p;
    }
  }
  NormTiles& t = p.tiles;
  // A group wider than a block's columns is cut into equal parts (rows by themselves that come here stay a block's, walk by walk), and a block has whole
  // groups (or parts), a chunk of them that begins on an access. Where whole accesses leave no such chunk (eight groups of 513 channels of 16 bits: not even
  // one of them is a number of 16-byte slices) accesses are narrower, down to single elements: 40000 x 4104 in 8 groups of 4 segments, bf16, gelu, 0.64 and 1.05 ms
  // where a block that walks over a segment's group took 29 and 25.
  int per, groups, chunk;
  int64_t slices;
  bool fits;
  for (p.slice = slice_of(s.dim, size, addresses);; p.slice /= 2) {
    t.fold = 1;
    if (s.per > kMostColumns && (s.offsets || s.per_segment > 1)) {
      t.fold = (int)ceil_div(s.per, kMostColumns);
      while (s.per / t.fold >= 64 && s.per % (t.fold * p.slice)) ++t.fold;
    }
    per = s.per / t.fold, groups = s.groups * t.fold, chunk = groups;
    if (s.dim > kMostColumns || groups > kMostColumns / 4) {
      chunk = std::min<int>(kMostColumns / per, kMostColumns / 4);
      while (chunk > 0 && (int64_t)chunk * per % p.slice) --chunk;
    }
    slices = chunk > 0 ? ceil_div((int64_t)std::min(chunk, groups) * per, p.slice) : 0;
    fits = chunk > 0 && per * t.fold == s.per && slices <= 256 * (8 / p.slice) && s.segments > 0;
    if (fits || p.slice == 1) break;
  }
  if (!fits) {
    p.kind = kNormWide;
    p.blocks = std::max<int64_t>(1, std::min<int64_t>(ceil_div(s.rows, 32), kNumSMs * 8 / ceil_div(s.dim, 256)));
    return p;
  }
  p.kind = kNormTiles;
  t.chunk = chunk;
  p.chunks = ceil_div(groups, chunk);
  p.warps = p.chunks == 1 && slices <= 32 * (8 / p.slice);
  const int team = p.warps ? 32 : 256;
  p.held = slices <= team ? 1 : 8 / p.slice;
  t.slots = (int)ceil_div(slices, p.held);
  t.lines = team / t.slots;
  // a round of blocks each, two or three an SM (registers)
  const auto tiles_of = [&](int per_sm, int64_t* rows, int64_t* tiles) {
    const int64_t teams = ceil_div(kNumSMs * per_sm, p.chunks) * (256 / team);
    *rows = ceil_div(ceil_div(s.rows, teams), t.lines) * t.lines;
    *tiles = ceil_div(s.rows, *rows);
  };
  tiles_of(back ? 2 : 3, &t.sum_rows, &t.sum_tiles);
  tiles_of(p.held > 1 || per % p.slice ? 2 : 3, &t.apply_rows, &t.apply_tiles);
  // threads for all pieces of a mean segment, or a number of them
  t.join_groups = 1;
  while (t.join_groups < 64 && t.join_groups < s.groups && 256 / (2 * t.join_groups) >= t.sum_tiles / s.segments + 1) t.join_groups *= 2;
  t.join_groups = std::max(t.join_groups, std::min(4, s.groups));
  t.join_segments = s.segments >= kNumSMs * 8 ? 8 : 1;
  p.blocks = ceil_div(t.sum_tiles, 256 / team);
  return p;
}

// Sums for dgamma and dbeta, sums of pieces, means of segments, what stays.
struct NormRoom {
  size_t columns, parts, means, mask;
  size_t all() const { return columns + parts + means + mask; }
};
static NormRoom norm_room(const NormShape& s, const NormPlan& p, bool back) {
  const bool tiles = p.kind == kNormTiles;
  return {back ? align_up((size_t)p.blocks * 2 * s.dim * 4, 256) : 0,
          tiles ? align_up((size_t)(p.tiles.sum_tiles + s.segments) * s.groups * p.tiles.fold * 8, 256) : 0,
          back && tiles ? align_up((size_t)s.segments * s.groups * 8, 256) : 0, back && tiles && p.slice % 4 == 0 ? (size_t)(s.rows * s.dim) / p.slice : 0};
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
  for (const uintptr_t addresses : {0, 8, 4, 2}) most = std::max(most, norm_room(s, norm_plan(s, dtype == APT_F32 ? 4 : 2, addresses, backward), backward).all());
  return most;
}

extern "C" int apt_group_norm_forward(int dtype, int param_dtype, const void* x, int64_t rows, int64_t dim, int groups, const int64_t* offsets,
                                      int64_t segments, double eps, int act, const void* weight, const void* bias, double p, uint64_t key,
                                      uint32_t call_id, void* out, float* stats, void* workspace, size_t workspace_bytes, int32_t* status_word,
                                      void* stream) {
  using namespace apt;
  if (const int e = norm_check("apt_group_norm_forward", dtype, param_dtype, rows, dim, groups, offsets, segments, eps, act, p)) return e;
  if (rows == 0) {
    if (stats) APT_CUDA(cudaMemsetAsync(stats, 0, (size_t)segments * groups * 8, (cudaStream_t)stream));
    return look_at_ends(offsets, segments, 0, status_word, (cudaStream_t)stream);
  }
  const NormShape s = norm_shape(rows, dim, groups, offsets, segments);
  APT_CHECK_ARG(x && out && status_word && (stats || (!offsets && segments == rows && dim / groups <= APT_GROUP_NORM_ROW_CHANNELS)), "apt_group_norm_forward: null buffer");
  APT_CHECK_ARG(workspace_bytes >= apt_group_norm_workspace_bytes(dtype, rows, dim, groups, offsets, segments, 0), "apt_group_norm_forward: workspace too small");
  const NormPlan plan = norm_plan(s, dtype == APT_F32 ? 4 : 2, (uintptr_t)x | (uintptr_t)out, false);
  const NormCall c{x, nullptr, weight, bias, out, nullptr, nullptr, (float2*)stats, (float)eps, act, param_dtype == APT_F32, p > 0.0,
                   make_drop(p, key, call_id), status_word, nullptr, (float2*)workspace, nullptr, nullptr};
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
    return look_at_ends(offsets, segments, 0, status_word, st);
  }
  APT_CHECK_ARG(x && grad_out && grad_x && status_word && (stats || (!offsets && segments == rows && dim / groups <= APT_GROUP_NORM_ROW_CHANNELS)), "apt_group_norm_backward: null buffer");
  APT_CHECK_ARG(workspace_bytes >= apt_group_norm_workspace_bytes(dtype, rows, dim, groups, offsets, segments, 1), "apt_group_norm_backward: workspace too small");
  const NormShape s = norm_shape(rows, dim, groups, offsets, segments);
  const NormPlan plan = norm_plan(s, dtype == APT_F32 ? 4 : 2, (uintptr_t)x | (uintptr_t)grad_out | (uintptr_t)grad_x, true);
  const bool params = grad_weight || grad_bias;
  const NormRoom room = norm_room(s, plan, true);
  char* const ws = (char*)workspace;
  const NormCall c{x, grad_out, weight, bias, grad_x, grad_weight, grad_bias, (float2*)stats, (float)eps, act, param_dtype == APT_F32, p > 0.0,
                   make_drop(p, key, call_id), status_word, params ? (float*)ws : nullptr, (float2*)(ws + room.columns),
                   (float2*)(ws + room.columns + room.parts), (uint8_t*)(ws + room.columns + room.parts + room.means)};
  return norm_typed<true>(dtype, s, c, plan, st);
}
