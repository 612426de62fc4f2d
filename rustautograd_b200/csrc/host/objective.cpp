#include "objective.h"

#include <cmath>

namespace rg {

namespace {

bool attrs_ok(const Op& op, size_t n) {
  if (!op.value || op.value->n() != n) return false;
  for (size_t i = 0; i < n; ++i)
    if (!std::isfinite(op.value->data.get(i))) return false;
  return true;
}

}  // namespace

bool objective_of(const Op& op, const std::vector<std::vector<size_t>>& s, const std::vector<DType>& d, Objective* out, std::string* why) {
  auto no = [&](const char* reason) {
    *why = reason;
    return false;
  };
  size_t lo = 0, hi = 0;
  switch (op.kind) {
    case OpKind::LogProb: lo = hi = 2; break;
    case OpKind::LogProbGrad: lo = hi = 4; break;
    case OpKind::PolicyLoss: lo = 5; hi = 6; break;
    case OpKind::PreferenceLoss: case OpKind::DistillLoss: lo = hi = 4; break;
    default: return no("not_an_objective");
  }
  if (s.size() < lo || s.size() > hi || d.size() != s.size()) return no("wrong_input_count");
  if (d[0] == DType::I32) return no("logits_must_be_floating");
  for (size_t i = 1; i < d.size(); ++i)
    if (d[i] != (i == 1 ? DType::I32 : d[0])) return no(i == 1 ? "index_must_be_int32" : "implicit_promotion_not_allowed");
  if (s[0].empty() || s[0].back() == 0 || s[0].back() > OBJECTIVE_MAX_VOCAB) return no("logits_need_a_nonempty_last_axis");
  Objective o;
  const std::vector<size_t> lead(s[0].begin(), s[0].end() - 1);
  o.vocab = s[0].back();
  o.rows = o.outer = product(lead);
  if (o.rows > OBJECTIVE_MAX_ROWS || (op.kind == OpKind::PreferenceLoss && !lead.empty() && lead[0] > OBJECTIVE_MAX_ROWS)) return no("too_many_rows");
  o.inner = 1;
  auto with = [&](size_t n) {
    auto v = lead;
    v.push_back(n);
    return v;
  };
  switch (op.kind) {
    case OpKind::LogProb:
      if (s[1] != lead) return no("labels_need_the_leading_shape_of_the_logits");
      o.outs = {lead, with(2)};
      break;
    case OpKind::LogProbGrad:
      if (s[1] != lead || s[2] != with(2) || s[3] != lead) return no("operands_do_not_fit_the_logits");
      break;
    case OpKind::PolicyLoss: {
      for (size_t i = 1; i < s.size(); ++i)
        if (s[i] != lead) return no("operands_need_the_leading_shape_of_the_logits");
      if (!attrs_ok(op, 3)) return no("clip_low_clip_high_and_kl_must_be_finite");
      if (objective_attr(op, 0) < 0 || objective_attr(op, 1) < 0) return no("clip_ranges_must_not_be_negative");
      if ((objective_attr(op, 2) != 0) != (s.size() == 6)) return no("reference_log_probabilities_go_with_a_kl_coefficient");
      o.outs = {{}, lead, lead, s[0]};
      o.grad_out = 3;
      o.weight_arg = 4;
      break;
    }
    case OpKind::PreferenceLoss:
      if (s[0].size() != 3 || lead[0] == 0 || lead[0] % 2) return no("logits_must_be_pairs_of_sequences_by_positions_by_vocabulary");
      if (s[1] != lead || s[2] != lead || s[3] != std::vector<size_t>{lead[0]}) return no("operands_do_not_fit_the_logits");
      if (!attrs_ok(op, 2)) return no("beta_and_smoothing_must_be_finite");
      if (objective_attr(op, 1) < 0 || objective_attr(op, 1) > 1) return no("smoothing_must_be_between_zero_and_one");
      o.outer = lead[0];
      o.inner = lead[1];
      o.outs = {{}, {lead[0] / 2}, {lead[0]}, s[0]};
      o.grad_out = 3;
      o.weight_arg = 2;
      break;
    default:
      if (s[1].empty() || s[1].back() == 0 || s[1].back() > OBJECTIVE_MAX_ENTRIES) return no("teacher_needs_between_1_and_1024_entries_per_row");
      o.k = s[1].back();
      if (s[1] != with(o.k) || s[2] != s[1] || s[3] != lead) return no("operands_do_not_fit_the_logits");
      // Beyond these bounds 1 / T or T^2 leaves the range of a float.
      if (!attrs_ok(op, 1) || !(objective_attr(op, 0) >= 0x1p-60 && objective_attr(op, 0) <= 0x1p60)) return no("temperature_must_be_between_2^-60_and_2^60");
      o.outs = {{}, lead, s[0]};
      o.grad_out = 2;
      o.weight_arg = 3;
      o.teacher_arg = 2;
  }
  *out = std::move(o);
  return true;
}

}  // namespace rg
