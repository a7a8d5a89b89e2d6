// The group norm's kernels of bf16 rows.
#include "group_norm.cuh"

namespace apt {
template int norm<__nv_bfloat16, false>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
template int norm<__nv_bfloat16, true>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
}  // namespace apt
