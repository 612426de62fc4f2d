// The objectives over float logits.
#include "objectives_kernels.cuh"

namespace rgc {

template cudaError_t Objectives<float>::log_prob(const RowView&, const int32_t*, void*, void*, cudaStream_t);
template cudaError_t Objectives<float>::log_prob_grad(const RowView&, const int32_t*, const void*, const void*, const RowOut&, cudaStream_t);
template cudaError_t Objectives<float>::policy(const RowView&, const int32_t*, const PolicyArgs&, void*, void*, void*, const RowOut&, cudaStream_t);
template cudaError_t Objectives<float>::preference(const RowView&, const int32_t*, const PreferenceArgs&, void*, void*, void*, const RowOut&, void*, cudaStream_t);
template cudaError_t Objectives<float>::distill(const RowView&, const DistillArgs&, void*, void*, const RowOut&, cudaStream_t);

}  // namespace rgc
