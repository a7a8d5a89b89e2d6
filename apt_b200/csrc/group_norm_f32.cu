// The group norm's kernels of fp32 rows.
#include "group_norm.cuh"

namespace apt {
template int norm<float, false>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
template int norm<float, true>(const NormShape&, const NormCall&, const NormPlan&, cudaStream_t);
}  // namespace apt
