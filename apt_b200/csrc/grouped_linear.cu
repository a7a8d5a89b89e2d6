// Products of rows in ragged groups with the weights of their group: the calls of the kernel in grouped.cuh.
#include "grouped.cuh"

namespace apt {

template <typename T>
static int linear_forward(const void* x, int64_t rows, int64_t dim, const void* weight, const void* bias, int64_t out_dim, const int64_t* offsets, int groups,
                          void* out, char* room, int32_t* status, cudaStream_t s) {
  char* const carry = room;
  room += carry_room<T>(rows, dim, out_dim, false);
  Operand a, w;
  if (const int e = laid_out(x, 0, rows, dim, sizeof(T), &room, &a, s)) return e;
  if (const int e = laid_out(weight, groups, out_dim, dim, sizeof(T), &room, &w, s)) return e;
  return rows_product<T, kOut>(a, w, out_dim, bias, offsets, groups, out, carry, status, s);
}

template <typename T>
static size_t linear_room(int64_t rows, int64_t dim, int64_t out_dim, int64_t groups, bool backward) {
  size_t bytes = carry_room<T>(rows, dim, out_dim, backward) + room_of(rows, dim, sizeof(T)) + room_of(groups * out_dim, dim, sizeof(T));
  if (backward) {
    const WeightPlan p = weight_plan<T>(rows, dim, out_dim, groups);
    bytes += room_of(rows, out_dim, sizeof(T)) + align_up((size_t)(2 + kPlanWords * p.ranges) * 8, 256) + (size_t)p.pieces * kTileM * (p.tile_n + 1) * 4;
  }
  return bytes;
}

template <typename T>
static int linear_backward(const void* x, int64_t rows, int64_t dim, const void* weight, int64_t out_dim, const int64_t* offsets, int groups,
                           const void* grad, void* grad_x, void* grad_weight, void* grad_bias, char* room, int32_t* status, cudaStream_t s) {
  if (grad_bias && !grad_weight) {
    const dim3 grid((unsigned)ceil_div(out_dim, 32), (unsigned)groups);
    APT_FOLLOW((k_bias_sums<T>), grid, 1024, 0, s, (const T*)grad, rows, out_dim, offsets, (T*)grad_bias, status);
  }
  if (rows == 0) {
    if (grad_weight) APT_CUDA(cudaMemsetAsync(grad_weight, 0, (size_t)groups * out_dim * dim * sizeof(T), s));
    if (grad_weight && grad_bias) APT_CUDA(cudaMemsetAsync(grad_bias, 0, (size_t)groups * out_dim * sizeof(T), s));
    return look_at_ends(offsets, groups, 0, status, s);
  }
  if (!grad_x && !grad_weight) return APT_OK;
  char* const carry = room;
  room += carry_room<T>(rows, dim, out_dim, true);
  Operand dy;
  if (const int e = laid_out(grad, 0, rows, out_dim, sizeof(T), &room, &dy, s)) return e;
  if (grad_x) {
    Operand w;
    if (const int e = laid_out(weight, groups, out_dim, dim, sizeof(T), &room, &w, s)) return e;
    if (const int e = rows_product<T, kGradX>(dy, w, dim, nullptr, offsets, groups, grad_x, carry, status, s)) return e;
  }
  if (grad_weight) {
    using Tr = GroupedTraits<T, kGradW>;
    Operand in;
    if (const int e = laid_out(x, 0, rows, dim, sizeof(T), &room, &in, s)) return e;
    const WeightPlan p = weight_plan<T>(rows, dim, out_dim, groups);
    GroupedCall c = {};
    c.offsets = offsets, c.rows = rows, c.groups = groups;
    c.num_m = (int)out_dim, c.num_n = (int)dim;
    c.tile_n = p.tile_n, c.tiles_m = p.tiles_m, c.tiles_n = p.tiles_n, c.ranges = p.ranges;
    c.a = dy.data, c.b = in.data, c.pitch_a = dy.pitch, c.pitch_b = in.pitch;
    c.out = grad_weight, c.grad_bias = grad_bias, c.carry = (float*)carry, c.status = status;
    c.plan = (int64_t*)room;
    c.partial = (float*)(room + align_up((size_t)(2 + kPlanWords * p.ranges) * 8, 256));
    c.partial_bias = c.partial + (size_t)p.pieces * kTileM * p.tile_n;
    CUtensorMap a, b;
    if (const int e = make_map(&a, code_of<T>(), dy, Tr::kBox, Tr::kBlock)) return e;
    if (const int e = make_map(&b, code_of<T>(), in, Tr::kBox, Tr::kBlock)) return e;
    if (const int e = launch_grouped<T, kGradW>(c, a, b, p.ranges, s)) return e;
    if (p.ranges > 1) {
      const dim3 grid(kJoinParts, (unsigned)(p.ranges - 1));
      APT_FOLLOW((k_join_weights<T>), grid, 256, 0, s, c);
    }
  }
  return APT_OK;
}

static int linear_check(const char* who, int dtype, int64_t rows, int64_t dim, int64_t out_dim, int64_t groups, const void* workspace, size_t workspace_bytes,
                        int backward) {
  APT_CHECK_ARG(dtype == APT_F32 || dtype == APT_BF16 || dtype == APT_F16, "%s: unsupported dtype %d", who, dtype);
  APT_CHECK_ARG(rows >= 0 && rows < (1ll << 31) - (1 << 20) && dim > 0 && out_dim > 0 && dim <= APT_GROUPED_LINEAR_MAX_DIM && out_dim <= APT_GROUPED_LINEAR_MAX_DIM,
                "%s: %lld rows of %lld by %lld (1 to %d are possible)", who, (long long)rows, (long long)dim, (long long)out_dim, APT_GROUPED_LINEAR_MAX_DIM);
  APT_CHECK_ARG(groups > 0 && groups <= APT_GROUPED_LINEAR_MAX_GROUPS, "%s: %lld groups (1 to %d are possible)", who, (long long)groups,
                APT_GROUPED_LINEAR_MAX_GROUPS);
  APT_CHECK_ARG(rows == 0 || workspace_bytes >= apt_grouped_linear_workspace_bytes(dtype, rows, dim, out_dim, groups, backward), "%s: workspace too small", who);
  APT_CHECK_ARG((uintptr_t)workspace % 16 == 0, "%s: workspace not aligned to 16 bytes", who);
  return APT_OK;
}

}  // namespace apt

extern "C" size_t apt_grouped_linear_workspace_bytes(int dtype, int64_t rows, int64_t dim, int64_t out_dim, int64_t groups, int backward) {
  if (rows <= 0 || dim <= 0 || out_dim <= 0 || groups <= 0) return 0;
  return dtype == APT_F32 ? apt::linear_room<float>(rows, dim, out_dim, groups, backward) : apt::linear_room<__half>(rows, dim, out_dim, groups, backward);
}

extern "C" int apt_grouped_linear_forward(int dtype, const void* x, int64_t rows, int64_t dim, const void* weight, const void* bias, int64_t out_dim,
                                          const int64_t* offsets, int64_t groups, void* out, void* workspace, size_t workspace_bytes,
                                          int32_t* status_word, void* stream) {
  using namespace apt;
  if (const int e = linear_check("apt_grouped_linear_forward", dtype, rows, dim, out_dim, groups, workspace, workspace_bytes, 0)) return e;
  if (rows == 0) return look_at_ends(offsets, groups, 0, status_word, (cudaStream_t)stream);
  APT_CHECK_ARG(x && weight && offsets && out && status_word, "apt_grouped_linear_forward: null buffer");
  APT_CHECK_ARG(((uintptr_t)x | (uintptr_t)weight | (uintptr_t)out) % 16 == 0, "apt_grouped_linear_forward: buffers not aligned to 16 bytes");
  const cudaStream_t s = (cudaStream_t)stream;
  char* const room = (char*)workspace;
  if (dtype == APT_F32) return linear_forward<float>(x, rows, dim, weight, bias, out_dim, offsets, (int)groups, out, room, status_word, s);
  if (dtype == APT_BF16) return linear_forward<__nv_bfloat16>(x, rows, dim, weight, bias, out_dim, offsets, (int)groups, out, room, status_word, s);
  return linear_forward<__half>(x, rows, dim, weight, bias, out_dim, offsets, (int)groups, out, room, status_word, s);
}

extern "C" int apt_grouped_linear_backward(int dtype, const void* x, int64_t rows, int64_t dim, const void* weight, int64_t out_dim,
                                           const int64_t* offsets, int64_t groups, const void* grad_out, void* grad_x, void* grad_weight,
                                           void* grad_bias, void* workspace, size_t workspace_bytes, int32_t* status_word, void* stream) {
  using namespace apt;
  if (const int e = linear_check("apt_grouped_linear_backward", dtype, rows, dim, out_dim, groups, workspace, workspace_bytes, 1)) return e;
  APT_CHECK_ARG(offsets && status_word && (rows == 0 || grad_out) && (!grad_x || rows == 0 || weight) && (!grad_weight || rows == 0 || x),
                "apt_grouped_linear_backward: null buffer");
  APT_CHECK_ARG(((uintptr_t)x | (uintptr_t)weight | (uintptr_t)grad_out | (uintptr_t)grad_x | (uintptr_t)grad_weight) % 16 == 0,
                "apt_grouped_linear_backward: buffers not aligned to 16 bytes");
  const cudaStream_t s = (cudaStream_t)stream;
  const int g = (int)groups;
  char* const room = (char*)workspace;
  if (dtype == APT_F32) return linear_backward<float>(x, rows, dim, weight, out_dim, offsets, g, grad_out, grad_x, grad_weight, grad_bias, room, status_word, s);
  if (dtype == APT_BF16)
    return linear_backward<__nv_bfloat16>(x, rows, dim, weight, out_dim, offsets, g, grad_out, grad_x, grad_weight, grad_bias, room, status_word, s);
  return linear_backward<__half>(x, rows, dim, weight, out_dim, offsets, g, grad_out, grad_x, grad_weight, grad_bias, room, status_word, s);
}
