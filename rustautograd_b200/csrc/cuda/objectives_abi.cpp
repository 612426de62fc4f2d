// The C ABI of the objectives over logits (include/rgc.h): argument checks around objectives.cuh.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <exception>
#include <string>

#include "objective.h"
#include "objectives.cuh"
#include "rgc.h"

namespace rgc {

int set_last_error(int code, const std::string& msg);

namespace {

struct Refused {
  int code;
  std::string why;
};

[[noreturn]] void refuse(const std::string& why) { throw Refused{RGC_ERR_INVALID, why}; }

struct Rows {
  RowView x;
  EType t = EType::F32;
  size_t es = 4;
  bool vouched = false;  // the caller knows that its pointers are the current device's
};

// A pointer the kernels will read or write: device memory of the current device. (A host pointer, or
// another device's, would fault on the GPU.) device < 0: its place is not looked up.
void check_pointer(const char* what, const void* p, size_t align, int device) {
  if (!p) refuse(std::string(what) + " is null");
  if ((uintptr_t)p % align) refuse(std::string(what) + " is not aligned to its element size");
  if (device < 0) return;
  cudaPointerAttributes a;
  const cudaError_t e = cudaPointerGetAttributes(&a, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    throw Refused{RGC_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e)};
  }
  if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) refuse(std::string(what) + " is not device memory");
  if (a.type == cudaMemoryTypeDevice && a.device != device) refuse(std::string(what) + " is on device " + std::to_string(a.device) + ", not the current device " + std::to_string(device));
}

int device_of(const Rows& r) {
  if (r.vouched) return -1;
  int d = 0;
  const cudaError_t e = cudaGetDevice(&d);
  if (e != cudaSuccess) {
    cudaGetLastError();
    throw Refused{RGC_ERR_UNAVAILABLE, std::string("no CUDA device: ") + cudaGetErrorString(e)};
  }
  return d;
}

// Elements from the first to behind the last one of `outer` x `inner` rows of `vocab`; 2^60 stands for more.
int64_t extent(const rgc_logits& x, int64_t so, int64_t si) {
  const double all = (double)(x.outer - 1) * (double)so + (double)(x.inner - 1) * (double)si + (double)x.vocab;
  return all < 0x1p60 ? (x.outer - 1) * so + (x.inner - 1) * si + x.vocab : int64_t(1) << 60;
}

// Rows, or either factor of them: sequences without positions have their pairs all the same.
bool too_many(int64_t outer, int64_t inner) {
  constexpr int64_t most = rg::OBJECTIVE_MAX_ROWS;
  return outer > most || inner > most || (inner && outer > most / inner);
}

// The sizes, types and strides (before any CUDA call).
Rows check_logits(const rgc_logits* x) {
  if (!x) refuse("null argument");
  const int dtype = x->dtype & ~RGC_VOUCHED;
  if (dtype != 0 && dtype != 1) refuse("dtype must be 0 (float32) or 1 (float64)");
  if (x->outer < 0 || x->inner < 0) refuse("negative row count");
  if (x->vocab < 1 || x->vocab > (int64_t)rg::OBJECTIVE_MAX_VOCAB) refuse("vocab must be between 1 and 2^30");
  constexpr int64_t LIMIT = int64_t(1) << 40;
  if (too_many(x->outer, x->inner)) refuse("too many rows (at most 2^31 - 1)");
  if (x->outer_stride < 0 || x->inner_stride < 0 || x->outer_stride > LIMIT || x->inner_stride > LIMIT) refuse("strides must be between 0 and 2^40");
  if (x->outer > 0 && x->inner > 0 && extent(*x, x->outer_stride, x->inner_stride) >= int64_t(1) << 60) refuse("the rows span 2^60 elements or more");
  Rows r;
  r.t = dtype == 1 ? EType::F64 : EType::F32;
  r.vouched = (x->dtype & RGC_VOUCHED) != 0;
  r.es = esize(r.t);
  r.x.data = x->data;
  r.x.outer = x->outer;
  r.x.inner = x->inner;
  r.x.vocab = x->vocab;
  r.x.so = x->outer_stride;
  r.x.si = x->inner_stride;
  return r;
}

RowOut check_gradient(const rgc_logits& x, const Rows& r, const rgc_gradient* g) {
  RowOut out;
  if (!g || !g->data) return out;
  const int64_t so = g->outer_stride, si = g->inner_stride;
  constexpr int64_t LIMIT = int64_t(1) << 40;
  if (so < 0 || si < 0 || so > LIMIT || si > LIMIT) refuse("gradient strides must be between 0 and 2^40");
  if (r.x.rows() > 0 && extent(x, so, si) >= int64_t(1) << 60) refuse("the gradient's rows span 2^60 elements or more");
  // Rows written at the same time may not overlap: the smaller stride steps over a row, the larger
  // one over all rows of the smaller.
  if (r.x.rows() > 0) {
    const bool io = x.inner <= 1 || (x.outer > 1 && so < si);  // outer is the faster one
    const int64_t fast_n = io ? x.outer : x.inner, fast = io ? so : si, slow_n = io ? x.inner : x.outer, slow = io ? si : so;
    if (fast_n > 1 && fast < x.vocab) refuse("gradient rows overlap");
    if (slow_n > 1 && slow < (fast_n - 1) * fast + x.vocab) refuse("gradient rows overlap");
    const char *a = (const char*)x.data, *b = (const char*)g->data;
    const bool same = a == b && (x.outer <= 1 || so == x.outer_stride) && (x.inner <= 1 || si == x.inner_stride);
    if (!same && b < a + extent(x, x.outer_stride, x.inner_stride) * (int64_t)r.es && a < b + extent(x, so, si) * (int64_t)r.es)
      refuse("the gradient overlaps the logits without being them");
  }
  out.data = g->data;
  out.so = so;
  out.si = si;
  return out;
}

void launched(cudaError_t e) {
  if (e != cudaSuccess) throw Refused{RGC_ERR_CUDA, std::string("launch: ") + cudaGetErrorString(e)};
}

template <typename F> int entry(const char* name, F f) {
  try {
    set_last_error(RGC_OK, "");
    f();
    return RGC_OK;
  } catch (const Refused& r) {
    return set_last_error(r.code, std::string(name) + ": " + r.why);
  } catch (const std::exception& e) {
    return set_last_error(RGC_ERR_INVALID, std::string(name) + ": " + e.what());
  }
}

}  // namespace
}  // namespace rgc

using namespace rgc;

#define RGC_EXPORT extern "C" __attribute__((visibility("default")))

RGC_EXPORT int rgc_token_log_prob(const rgc_logits* logits, const int32_t* labels, void* logp, void* stats, void* stream) {
  return entry("rgc_token_log_prob", [&] {
    const Rows r = check_logits(logits);
    if (r.x.rows() == 0) return;
    if (!logp && !stats) refuse("no output is asked for");
    const int dev = device_of(r);
    check_pointer("logits", logits->data, r.es, dev);
    check_pointer("labels", labels, 4, dev);
    if (logp) check_pointer("logp", logp, r.es, dev);
    if (stats) check_pointer("stats", stats, r.es, dev);
    launched(token_log_prob(r.t, r.x, labels, logp, stats, (cudaStream_t)stream));
  });
}

RGC_EXPORT int rgc_token_log_prob_grad(const rgc_logits* logits, const int32_t* labels, const void* stats, const void* dlogp, const rgc_gradient* grad,
                                       void* stream) {
  return entry("rgc_token_log_prob_grad", [&] {
    const Rows r = check_logits(logits);
    const RowOut g = check_gradient(*logits, r, grad);
    if (r.x.rows() == 0) return;
    const int dev = device_of(r);
    check_pointer("logits", logits->data, r.es, dev);
    check_pointer("labels", labels, 4, dev);
    check_pointer("stats", stats, r.es, dev);
    check_pointer("dlogp", dlogp, r.es, dev);
    check_pointer("grad", g.data, r.es, dev);
    launched(token_log_prob_grad(r.t, r.x, labels, stats, dlogp, g, (cudaStream_t)stream));
  });
}

RGC_EXPORT int rgc_policy_loss(const rgc_logits* logits, const int32_t* labels, const rgc_policy* p, void* loss, void* terms, void* logp,
                               const rgc_gradient* grad, void* stream) {
  return entry("rgc_policy_loss", [&] {
    const Rows r = check_logits(logits);
    if (!p) refuse("null argument");
    if (!std::isfinite(p->clip_low) || !std::isfinite(p->clip_high) || !std::isfinite(p->kl)) refuse("clip_low, clip_high and kl must be finite");
    if (p->clip_low < 0 || p->clip_high < 0) refuse("clip ranges must not be negative");
    const RowOut g = check_gradient(*logits, r, grad);
    const int dev = device_of(r);
    check_pointer("loss", loss, r.es, dev);
    if (r.x.rows() > 0) {
      check_pointer("logits", logits->data, r.es, dev);
      check_pointer("labels", labels, 4, dev);
      check_pointer("old_logp", p->old_logp, r.es, dev);
      check_pointer("advantage", p->advantage, r.es, dev);
      check_pointer("weight", p->weight, r.es, dev);
      if (p->kl != 0) check_pointer("ref_logp", p->ref_logp, r.es, dev);
      check_pointer("terms", terms, r.es, dev);
      if (logp) check_pointer("logp", logp, r.es, dev);
      if (g.data) check_pointer("grad", g.data, r.es, dev);
    }
    PolicyArgs a;
    a.old_logp = p->old_logp;
    a.ref_logp = p->ref_logp;
    a.advantage = p->advantage;
    a.weight = p->weight;
    a.clip_low = p->clip_low;
    a.clip_high = p->clip_high;
    a.kl = p->kl;
    launched(policy_loss(r.t, r.x, labels, a, loss, terms, logp, g, (cudaStream_t)stream));
  });
}

RGC_EXPORT size_t rgc_preference_workspace(int64_t sequences, int64_t length, int dtype) {
  if (sequences < 0 || length < 0 || too_many(sequences, length) || (dtype != 0 && dtype != 1)) return 0;
  return preference_workspace_bytes(dtype == 1 ? EType::F64 : EType::F32, sequences, length);
}

RGC_EXPORT int rgc_preference_loss(const rgc_logits* logits, const int32_t* labels, const rgc_preference* p, void* loss, void* margins, void* logp,
                                   const rgc_gradient* grad, void* workspace, size_t workspace_bytes, void* stream) {
  return entry("rgc_preference_loss", [&] {
    const Rows r = check_logits(logits);
    if (!p) refuse("null argument");
    if (r.x.outer < 2 || r.x.outer % 2) refuse("the logits are pairs of sequences: outer must be even and at least 2");
    if (!std::isfinite(p->beta) || !(p->smoothing >= 0 && p->smoothing <= 1)) refuse("beta must be finite and smoothing between 0 and 1");
    if (workspace_bytes < preference_workspace_bytes(r.t, r.x.outer, r.x.inner)) refuse("the workspace is too small");
    const RowOut g = check_gradient(*logits, r, grad);
    const int dev = device_of(r);
    check_pointer("loss", loss, r.es, dev);
    check_pointer("ref_logp", p->ref_logp, r.es, dev);
    check_pointer("workspace", workspace, 8, dev);
    if (margins) check_pointer("margins", margins, r.es, dev);
    if (logp) check_pointer("logp", logp, r.es, dev);
    if (r.x.rows() > 0) {
      check_pointer("logits", logits->data, r.es, dev);
      check_pointer("labels", labels, 4, dev);
      check_pointer("weight", p->weight, r.es, dev);
      if (g.data) check_pointer("grad", g.data, r.es, dev);
    }
    PreferenceArgs a;
    a.weight = p->weight;
    a.ref_logp = p->ref_logp;
    a.beta = p->beta;
    a.smoothing = p->smoothing;
    launched(preference_loss(r.t, r.x, labels, a, loss, margins, logp, g, workspace, (cudaStream_t)stream));
  });
}

RGC_EXPORT int rgc_distillation_loss(const rgc_logits* logits, const rgc_distillation* p, void* loss, void* terms, const rgc_gradient* grad, void* stream) {
  return entry("rgc_distillation_loss", [&] {
    const Rows r = check_logits(logits);
    if (!p) refuse("null argument");
    if (p->entries < 1 || p->entries > (int64_t)rg::OBJECTIVE_MAX_ENTRIES) refuse("teacher entries per row must be between 1 and " + std::to_string(rg::OBJECTIVE_MAX_ENTRIES));
    if (!(p->temperature >= 0x1p-60 && p->temperature <= 0x1p60)) refuse("temperature must be between 2^-60 and 2^60");  // 1 / T and T^2 in a float
    const RowOut g = check_gradient(*logits, r, grad);
    const int dev = device_of(r);
    check_pointer("loss", loss, r.es, dev);
    if (r.x.rows() > 0) {
      check_pointer("logits", logits->data, r.es, dev);
      check_pointer("index", p->index, 4, dev);
      check_pointer("teacher", p->teacher, r.es, dev);
      check_pointer("weight", p->weight, r.es, dev);
      check_pointer("terms", terms, r.es, dev);
      if (g.data) check_pointer("grad", g.data, r.es, dev);
    }
    DistillArgs a;
    a.index = p->index;
    a.teacher = p->teacher;
    a.weight = p->weight;
    a.k = p->entries;
    a.temperature = p->temperature;
    launched(distill_loss(r.t, r.x, a, loss, terms, g, (cudaStream_t)stream));
  });
}
