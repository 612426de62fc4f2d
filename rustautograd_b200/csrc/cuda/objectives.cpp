// The objectives over logits by the logits' type (objectives_f32.cu and objectives_f64.cu hold the kernels).
#include "objectives.cuh"

namespace rgc {

cudaError_t token_log_prob(EType t, const RowView& x, const int32_t* labels, void* logp, void* stats, cudaStream_t s) {
  return t == EType::F64 ? Objectives<double>::log_prob(x, labels, logp, stats, s) : Objectives<float>::log_prob(x, labels, logp, stats, s);
}

cudaError_t token_log_prob_grad(EType t, const RowView& x, const int32_t* labels, const void* stats, const void* dlogp, const RowOut& grad,
                                cudaStream_t s) {
  return t == EType::F64 ? Objectives<double>::log_prob_grad(x, labels, stats, dlogp, grad, s)
                         : Objectives<float>::log_prob_grad(x, labels, stats, dlogp, grad, s);
}

cudaError_t policy_loss(EType t, const RowView& x, const int32_t* labels, const PolicyArgs& a, void* loss, void* terms, void* logp,
                        const RowOut& grad, cudaStream_t s) {
  return t == EType::F64 ? Objectives<double>::policy(x, labels, a, loss, terms, logp, grad, s)
                         : Objectives<float>::policy(x, labels, a, loss, terms, logp, grad, s);
}

// A log-probability and the statistics of each row, a coefficient of each sequence (and a number of each pair that is spare).
size_t preference_workspace_bytes(EType t, long long sequences, long long length) {
  return (size_t)(3 * sequences * length + 3 * (sequences / 2)) * esize(t);
}

cudaError_t preference_loss(EType t, const RowView& x, const int32_t* labels, const PreferenceArgs& a, void* loss, void* margins, void* logp,
                            const RowOut& grad, void* workspace, cudaStream_t s) {
  return t == EType::F64 ? Objectives<double>::preference(x, labels, a, loss, margins, logp, grad, workspace, s)
                         : Objectives<float>::preference(x, labels, a, loss, margins, logp, grad, workspace, s);
}

cudaError_t distill_loss(EType t, const RowView& x, const DistillArgs& a, void* loss, void* terms, const RowOut& grad, cudaStream_t s) {
  return t == EType::F64 ? Objectives<double>::distill(x, a, loss, terms, grad, s) : Objectives<float>::distill(x, a, loss, terms, grad, s);
}

}  // namespace rgc
