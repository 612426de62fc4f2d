// Objectives over rows of logits (graph.h LogProb .. DistillLoss; include/rgc.h rgc_token_log_prob ..):
// the log-probability of given tokens, the clipped policy loss with a KL term, the preference loss
// over pairs of sequences and the distillation from a teacher's top logits, with their gradients.
//
// For a row x of V logits: m = max_j x_j, s = sum_j exp(x_j - m), p_j = exp(x_j - m) / s, and for a label
// l (clamped to [0, V), as rg clamps indices) lp = (x_l - m) - log s. Every gradient with respect to the
// row has the form c (onehot(l) - p) with one coefficient c per row, or c (p - sum_k q_k onehot(i_k))
// for the distillation.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "kernels.cuh"

namespace rgc {

// outer x inner rows of `vocab` adjacent elements; row (a, b) starts at element a * so + b * si.
struct RowView {
  const void* data = nullptr;
  long long outer = 0, inner = 0, vocab = 0;
  long long so = 0, si = 0;
  long long rows() const { return outer * inner; }
};
// Where a gradient of that many rows goes (`data` null: no gradient is asked for). It may be the
// logits themselves with the logits' strides: a row is read before it is written.
struct RowOut {
  void* data = nullptr;
  long long so = 0, si = 0;
};

// logp[r] = lp; stats[2 r], stats[2 r + 1] = m, s. Either may be null.
cudaError_t token_log_prob(EType t, const RowView& x, const int32_t* labels, void* logp, void* stats, cudaStream_t s);
// grad = dlogp[r] (onehot - p), p from the stats of the forward. A row with dlogp = 0 is not read.
cudaError_t token_log_prob_grad(EType t, const RowView& x, const int32_t* labels, const void* stats, const void* dlogp, const RowOut& grad,
                                cudaStream_t s);

// loss = sum_r terms[r], terms[r] = w (-min(r A, clip(r, 1 - low, 1 + high) A) + kl (exp(d) - d - 1)) with
// r = exp(lp - old), d = ref - lp. Rows with w = 0 are not read: term, lp and gradient are 0.
// `ref` is read only when kl != 0. loss and logp may be null.
struct PolicyArgs {
  const void *old_logp = nullptr, *ref_logp = nullptr, *advantage = nullptr, *weight = nullptr;
  double clip_low = 0, clip_high = 0, kl = 0;
};
cudaError_t policy_loss(EType t, const RowView& x, const int32_t* labels, const PolicyArgs& a, void* loss, void* terms, void* logp,
                        const RowOut& grad, cudaStream_t s);

// 2B sequences of T rows (x.outer = 2B, x.inner = T), chosen ones first. S_b = sum_t w lp;
// h_k = beta ((S_k - ref_k) - (S_{B+k} - ref_{B+k})); loss = mean_k -(1 - e) log sigma(h_k) - e log sigma(-h_k).
// margins[k] = h_k, logp[b] = S_b (either may be null). `workspace`: preference_workspace_bytes bytes.
struct PreferenceArgs {
  const void *weight = nullptr, *ref_logp = nullptr;
  double beta = 0, smoothing = 0;
};
size_t preference_workspace_bytes(EType t, long long sequences, long long length);
cudaError_t preference_loss(EType t, const RowView& x, const int32_t* labels, const PreferenceArgs& a, void* loss, void* margins, void* logp,
                            const RowOut& grad, void* workspace, cudaStream_t s);

// q = softmax(teacher / T) over the k entries of a row (entries of -inf are absent), p = softmax(x / T);
// terms[r] = w T^2 sum_k q_k (log q_k - log p_{i_k}), loss their sum. An index given twice counts twice;
// rows with w = 0 or without entries give 0. Indices are clamped to [0, V).
struct DistillArgs {
  const int32_t* index = nullptr;
  const void *teacher = nullptr, *weight = nullptr;
  long long k = 0;
  double temperature = 1;
};
cudaError_t distill_loss(EType t, const RowView& x, const DistillArgs& a, void* loss, void* terms, const RowOut& grad, cudaStream_t s);

// The same by type.
template <typename T> struct Objectives {
  static cudaError_t log_prob(const RowView& x, const int32_t* labels, void* logp, void* stats, cudaStream_t s);
  static cudaError_t log_prob_grad(const RowView& x, const int32_t* labels, const void* stats, const void* dlogp, const RowOut& grad, cudaStream_t s);
  static cudaError_t policy(const RowView& x, const int32_t* labels, const PolicyArgs& a, void* loss, void* terms, void* logp, const RowOut& grad,
                            cudaStream_t s);
  static cudaError_t preference(const RowView& x, const int32_t* labels, const PreferenceArgs& a, void* loss, void* margins, void* logp, const RowOut& grad,
                                void* workspace, cudaStream_t s);
  static cudaError_t distill(const RowView& x, const DistillArgs& a, void* loss, void* terms, const RowOut& grad, cudaStream_t s);
};

}  // namespace rgc
