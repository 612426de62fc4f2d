// The objectives over rows of logits (graph.h LogProb, LogProbGrad, PolicyLoss, PreferenceLoss, DistillLoss;
// no counterpart in rg): the shapes they take and give. Graph construction, the device's lowering
// and the CPU interpreter read them from here.
#pragma once
#include <string>
#include <vector>

#include "graph.h"

namespace rg {

// The vocabulary, the rows (and a preference's sequences) and the teacher entries of a row that the device's kernels take.
constexpr size_t OBJECTIVE_MAX_VOCAB = size_t(1) << 30, OBJECTIVE_MAX_ROWS = 0x7fffffff, OBJECTIVE_MAX_ENTRIES = 1024;

struct Objective {
  size_t rows = 0, vocab = 0;
  size_t outer = 0, inner = 0;  // rows as outer x inner: PreferenceLoss's sequences x positions, else rows x 1
  size_t k = 1;                 // indices per row: DistillLoss's teacher entries
  std::vector<std::vector<size_t>> outs;  // the shapes of outputs 0, 1, ... (none for LogProbGrad)
  // Output 0 is the value that is differentiated; this output is its gradient with respect to the
  // logits (SIZE_MAX for LogProb, whose gradient is the LogProbGrad operation).
  size_t grad_out = SIZE_MAX;
  // The operands that say which indices (operand 1, k to a row) count: rows with weight 0 do not, nor do teacher entries of -inf.
  // SIZE_MAX: all do.
  size_t weight_arg = SIZE_MAX, teacher_arg = SIZE_MAX;
};

// The objective `op` on operands of the given shapes and dtypes; false and the reason when they do not fit.
bool objective_of(const Op& op, const std::vector<std::vector<size_t>>& shapes, const std::vector<DType>& dtypes, Objective* out, std::string* why);

// Attribute `i` of an objective (graph.h lists them).
inline double objective_attr(const Op& op, size_t i) { return op.value && i < op.value->n() ? op.value->data.get(i) : 0.0; }

}  // namespace rg
