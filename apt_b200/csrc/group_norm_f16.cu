// The group norm's kernels of f16 rows.
#include "group_norm.cuh"

namespace apt {
template int norm<__half, false>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
template int norm<__half, true>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
}  // namespace apt
