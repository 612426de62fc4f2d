// Kernels of the objectives over logits (objectives.cuh has the formulas).
//
// One block computes one row: a pass over the row for (m, s), the row's scalars, and, where a gradient
// is asked for, a second pass that writes it. Sums run in a fixed order, so every call gives the same
// bits. Row statistics and sums are held in the logits' type (32 bits at least); per-sequence and
// per-batch sums in 64 bits.
#include "objectives.cuh"

#include <algorithm>
#include <cmath>

namespace rgc {

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;

__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

__device__ __forceinline__ float ex(float v) { return expf(v); }
__device__ __forceinline__ double ex(double v) { return exp(v); }
__device__ __forceinline__ float ln(float v) { return logf(v); }
__device__ __forceinline__ double ln(double v) { return log(v); }

// ---- row statistics ----

// (max, sum of exp(x - max)) of a part of a row. A part without a finite maximum (no elements yet, or
// only -inf ones) has m = -inf and s = 0; NaN and +inf elements make s NaN, as the formulas do.
template <typename T> struct Stat {
  T m = -(T)INFINITY, s = (T)0;
  static __device__ T base(T m) { return m == -(T)INFINITY ? (T)0 : m; }
  __device__ void join(T m2, T s2) {
    const T n = m > m2 ? m : m2, b = base(n);
    s = s * ex(m - b) + s2 * ex(m2 - b);
    m = n;
  }
};

template <typename T> __device__ Stat<T> warp_join(Stat<T> a) {
  for (int d = 16; d; d >>= 1) {
    const T m = __shfl_xor_sync(~0u, a.m, d), s = __shfl_xor_sync(~0u, a.s, d);
    a.join(m, s);
  }
  return a;
}

// Row-wide (m, s), the same bits in every thread. `sh`: 2 * WARPS values.
template <typename T> __device__ Stat<T> block_join(Stat<T> a, T* sh) {
  a = warp_join(a);
  __syncthreads();
  if (threadIdx.x % 32 == 0) {
    sh[threadIdx.x / 32] = a.m;
    sh[WARPS + threadIdx.x / 32] = a.s;
  }
  __syncthreads();
  Stat<T> r;
  for (int w = 0; w < WARPS; ++w) r.join(sh[w], sh[WARPS + w]);
  return r;
}

// (m, s) of scale * row: a running maximum and sum per thread. NaN elements reach s through ex().
template <typename T> __device__ Stat<T> row_stats(const T* row, long long v, T scale, T* sh) {
  Stat<T> a;
  for (long long j = threadIdx.x; j < v; j += THREADS) {
    const T x = row[j] * scale;
    if (x > a.m) {
      a.s = a.s * ex(a.m - x) + (T)1;
      a.m = x;
      if (x == (T)INFINITY) a.s = (T)NAN;
    } else {
      a.s += ex(x - Stat<T>::base(a.m));
    }
  }
  return block_join(a, sh);
}

template <typename T> struct View {
  const T* data;
  long long inner, v, so, si;
  __device__ const T* row(long long r) const { return data + (r / inner) * so + (r % inner) * si; }
};
template <typename T> struct Out {
  T* data;
  long long inner, so, si;
  __device__ T* row(long long r) const { return data + (r / inner) * so + (r % inner) * si; }
};
template <typename T> View<T> view(const RowView& x) { return {(const T*)x.data, std::max<long long>(x.inner, 1), x.vocab, x.so, x.si}; }
template <typename T> Out<T> out(const RowView& x, const RowOut& g) { return {(T*)g.data, std::max<long long>(x.inner, 1), g.so, g.si}; }

__device__ __forceinline__ long long clamp_label(int l, long long v) { return l < 0 ? 0 : l >= v ? v - 1 : l; }

// ---- objectives with one target per row ----
//
// `row` gives a row's coefficient c of (onehot - p) from its log-probability and writes what the row
// reports (by one thread).

template <typename T> struct LogProbRow {
  static constexpr bool MASKED = false;
  T *logp, *stats;
  __device__ bool live(long long) const { return true; }
  __device__ void skip(long long) const {}
  __device__ T row(long long r, T lp, T m, T s, bool first) const {
    if (first) {
      if (logp) logp[r] = lp;
      if (stats) {
        stats[2 * r] = m;
        stats[2 * r + 1] = s;
      }
    }
    return (T)0;
  }
};

template <typename T> struct PolicyRow {
  const T *old_logp, *ref_logp, *advantage, *weight;
  T low, high, kl;  // the ratio's bounds 1 - clip_low and 1 + clip_high
  T *terms, *logp;
  __device__ bool live(long long r) const { return weight[r] != (T)0; }
  __device__ void skip(long long r) const {
    terms[r] = (T)0;
    if (logp) logp[r] = (T)0;
  }
  __device__ T row(long long r, T lp, T, T, bool first) const {
    const T a = advantage[r], w = weight[r], ratio = ex(lp - old_logp[r]);
    const T held = ratio < low ? low : ratio > high ? high : ratio;
    const T free_term = ratio * a, held_term = held * a;
    // A NaN ratio or advantage stays NaN through both comparisons.
    T term = free_term > held_term ? -held_term : -free_term;
    T c = (a >= (T)0 ? ratio <= high : ratio >= low) ? -free_term : (T)0;
    if (kl != (T)0) {
      const T d = ref_logp[r] - lp, e = ex(d);
      term += kl * (e - d - (T)1);
      c += kl * ((T)1 - e);
    }
    if (first) {
      terms[r] = w * term;
      if (logp) logp[r] = lp;
    }
    return w * c;
  }
};

template <typename T, class Obj, bool GRAD>
__global__ void __launch_bounds__(THREADS) k_target_rows(View<T> x, const int32_t* __restrict__ labels, long long rows, Obj obj, Out<T> g) {
  pdl_wait();
  __shared__ T sh[2 * WARPS];
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    T* gr = GRAD ? g.row(r) : nullptr;
    if (!obj.live(r)) {
      if (threadIdx.x == 0) obj.skip(r);
      if (GRAD)
        for (long long j = threadIdx.x; j < x.v; j += THREADS) gr[j] = (T)0;
      continue;
    }
    const T* xr = x.row(r);
    const long long l = clamp_label(labels[r], x.v);
    const T xl = xr[l];
    const Stat<T> st = row_stats(xr, x.v, (T)1, sh);
    const T lp = (xl - st.m) - ln(st.s);
    const T c = obj.row(r, lp, st.m, st.s, threadIdx.x == 0);
    if (GRAD)
      for (long long j = threadIdx.x; j < x.v; j += THREADS) {
        const T p = ex(xr[j] - st.m) / st.s;
        gr[j] = c * ((j == l ? (T)1 : (T)0) - p);
      }
  }
}

// ---- gradients whose coefficient needs more than the row ----

template <typename T> struct TokenCoef {
  const T* dlogp;
  __device__ T operator()(long long r) const { return dlogp[r]; }
};
template <typename T> struct PairCoef {
  const T *seq, *weight;  // per sequence, per token
  long long length;
  __device__ T operator()(long long r) const { return weight[r] == (T)0 ? (T)0 : seq[r / length] * weight[r]; }
};

template <typename T, class Coef>
__global__ void __launch_bounds__(THREADS) k_target_grad(View<T> x, const int32_t* __restrict__ labels, long long rows, const T* __restrict__ stats,
                                                         Coef coef, Out<T> g) {
  pdl_wait();
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T c = coef(r);
    T* gr = g.row(r);
    if (c == (T)0) {
      for (long long j = threadIdx.x; j < x.v; j += THREADS) gr[j] = (T)0;
      continue;
    }
    const T* xr = x.row(r);
    const long long l = clamp_label(labels[r], x.v);
    const T m = stats[2 * r], s = stats[2 * r + 1];
    for (long long j = threadIdx.x; j < x.v; j += THREADS) {
      const T p = ex(xr[j] - m) / s;
      gr[j] = c * ((j == l ? (T)1 : (T)0) - p);
    }
  }
}

// ---- sums in a fixed order ----

__device__ double block_sum(double v, double* sh) {
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  __syncthreads();
  if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
  __syncthreads();
  double r = 0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) r += sh[w];
  return r;
}

template <typename T> __global__ void __launch_bounds__(1024) k_sum_terms(const T* __restrict__ terms, long long n, T* loss, double scale) {
  pdl_wait();
  __shared__ double sh[32];
  double v = 0;
  for (long long i = threadIdx.x; i < n; i += blockDim.x) v += (double)terms[i];
  v = block_sum(v, sh);
  if (threadIdx.x == 0) *loss = (T)(v * scale);
}

// Block k: pair k's sequence sums, margin, loss term and the coefficients of its two sequences.
template <typename T>
__global__ void __launch_bounds__(THREADS) k_pairs(const T* __restrict__ token_logp, const T* __restrict__ weight, const T* __restrict__ ref, long long pairs,
                                                   long long length, double beta, double smoothing, T* terms, T* coef, T* margins, T* logp) {
  pdl_wait();
  __shared__ double sh[WARPS];
  const long long k = blockIdx.x;
  double total[2];
  for (int side = 0; side < 2; ++side) {
    const long long at = (k + side * pairs) * length;
    double v = 0;
    for (long long t = threadIdx.x; t < length; t += THREADS)
      if (weight[at + t] != (T)0) v += (double)weight[at + t] * (double)token_logp[at + t];
    total[side] = block_sum(v, sh);
  }
  if (threadIdx.x) return;
  const double h = beta * ((total[0] - (double)ref[k]) - (total[1] - (double)ref[pairs + k]));
  const double e = exp(-fabs(h)), up = h >= 0 ? 1 / (1 + e) : e / (1 + e), down = h >= 0 ? e / (1 + e) : 1 / (1 + e);
  const double tail = log1p(e);
  // -log sigma(h) = tail + max(-h, 0), -log sigma(-h) = tail + max(h, 0)
  terms[k] = (T)((1 - smoothing) * (tail + (h < 0 ? -h : 0)) + smoothing * (tail + (h > 0 ? h : 0)));
  if (h != h) terms[k] = (T)h;
  const double dh = beta * (smoothing * up - (1 - smoothing) * down) / (double)pairs;
  coef[k] = (T)dh;
  coef[pairs + k] = (T)-dh;
  if (margins) margins[k] = (T)h;
  if (logp) {
    logp[k] = (T)total[0];
    logp[pairs + k] = (T)total[1];
  }
}

// ---- distillation ----

template <typename T> struct Targets {
  const int32_t* index;
  const T *teacher, *weight;
  long long k;
  T temperature, inverse;
  T* terms;
};

// Dynamic shared memory: k probabilities, k logits at their indices and k indices.
template <typename T, bool GRAD> __global__ void __launch_bounds__(THREADS) k_distill_rows(View<T> x, long long rows, Targets<T> a, Out<T> g) {
  pdl_wait();
  extern __shared__ __align__(16) unsigned char dyn[];
  T* q = (T*)dyn;
  T* xk = q + a.k;
  int* at = (int*)(xk + a.k);
  __shared__ T sh[2 * WARPS];
  __shared__ double shd[WARPS];
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T w = a.weight[r];
    T* gr = GRAD ? g.row(r) : nullptr;
    Stat<T> tq;
    if (w != (T)0) {
      for (long long i = threadIdx.x; i < a.k; i += THREADS) tq.join(a.teacher[r * a.k + i] * a.inverse, (T)1);
      tq = block_join(tq, sh);
    }
    if (w == (T)0 || tq.s == (T)0) {  // no weight, or no entries
      if (threadIdx.x == 0) a.terms[r] = (T)0;
      if (GRAD)
        for (long long j = threadIdx.x; j < x.v; j += THREADS) gr[j] = (T)0;
      continue;
    }
    const T* xr = x.row(r);
    for (long long i = threadIdx.x; i < a.k; i += THREADS) {
      const long long l = clamp_label(a.index[r * a.k + i], x.v);
      at[i] = (int)l;
      q[i] = ex(a.teacher[r * a.k + i] * a.inverse - tq.m) / tq.s;
      xk[i] = xr[l] * a.inverse;
    }
    const Stat<T> st = row_stats(xr, x.v, a.inverse, sh);
    const T logs = ln(st.s);
    double kl = 0;
    for (long long i = threadIdx.x; i < a.k; i += THREADS) {
      const T qi = q[i];
      if (qi != (T)0) kl += (double)(qi * (ln(qi) - ((xk[i] - st.m) - logs)));
    }
    kl = block_sum(kl, shd);
    if (threadIdx.x == 0) a.terms[r] = w * a.temperature * a.temperature * (T)kl;
    if (GRAD) {
      const T c = w * a.temperature;
      for (long long j = threadIdx.x; j < x.v; j += THREADS) gr[j] = c * (ex(xr[j] * a.inverse - st.m) / st.s);
      __syncthreads();
      // An index's first entry writes its element, with the probabilities of all its entries in order.
      for (long long i = threadIdx.x; i < a.k; i += THREADS) {
        T sum = (T)0;
        bool first = true;
        for (long long o = 0; o < a.k; ++o) {
          if (at[o] != at[i]) continue;
          if (o < i) first = false;
          sum += q[o];
        }
        if (first) gr[at[i]] = c * (ex(xk[i] - st.m) / st.s - sum);
      }
    }
    __syncthreads();
  }
}

unsigned row_blocks(long long rows) { return (unsigned)std::min<long long>(std::max<long long>(rows, 1), 148 * 8); }

template <typename T> cudaError_t t_log_prob(const RowView& x, const int32_t* labels, void* logp, void* stats, cudaStream_t s) {
  if (x.rows() == 0) return cudaSuccess;
  return launch(k_target_rows<T, LogProbRow<T>, false>, row_blocks(x.rows()), THREADS, 0, s, view<T>(x), labels, x.rows(),
                LogProbRow<T>{(T*)logp, (T*)stats}, Out<T>{});
}

template <typename T, class Coef>
cudaError_t t_grad(const RowView& x, const int32_t* labels, const void* stats, Coef coef, const RowOut& g, cudaStream_t s) {
  if (x.rows() == 0) return cudaSuccess;
  return launch(k_target_grad<T, Coef>, row_blocks(x.rows()), THREADS, 0, s, view<T>(x), labels, x.rows(), (const T*)stats, coef, out<T>(x, g));
}

template <typename T> cudaError_t sum_terms(const void* terms, long long n, void* loss, double scale, cudaStream_t s) {
  return launch(k_sum_terms<T>, 1, 1024, 0, s, (const T*)terms, n, (T*)loss, scale);
}

template <typename T>
cudaError_t t_policy(const RowView& x, const int32_t* labels, const PolicyArgs& a, void* loss, void* terms, void* logp, const RowOut& g, cudaStream_t s) {
  PolicyRow<T> row{(const T*)a.old_logp, (const T*)a.ref_logp, (const T*)a.advantage, (const T*)a.weight,
                   (T)(1 - a.clip_low),  (T)(1 + a.clip_high),  (T)a.kl,                (T*)terms, (T*)logp};
  cudaError_t e = cudaSuccess;
  if (x.rows() > 0)
    e = g.data ? launch(k_target_rows<T, PolicyRow<T>, true>, row_blocks(x.rows()), THREADS, 0, s, view<T>(x), labels, x.rows(), row, out<T>(x, g))
               : launch(k_target_rows<T, PolicyRow<T>, false>, row_blocks(x.rows()), THREADS, 0, s, view<T>(x), labels, x.rows(), row, Out<T>{});
  if (e != cudaSuccess || !loss) return e;
  return sum_terms<T>(terms, x.rows(), loss, 1.0, s);
}

template <typename T>
cudaError_t t_preference(const RowView& x, const int32_t* labels, const PreferenceArgs& a, void* loss, void* margins, void* logp, const RowOut& g,
                         void* workspace, cudaStream_t s) {
  const long long rows = x.rows(), pairs = x.outer / 2;
  T* token = (T*)workspace;       // rows
  T* stats = token + rows;        // 2 * rows
  T* terms = stats + 2 * rows;    // pairs
  T* coef = terms + pairs;        // 2 * pairs
  cudaError_t e = t_log_prob<T>(x, labels, token, stats, s);
  if (e == cudaSuccess && pairs > 0)
    e = launch(k_pairs<T>, (unsigned)pairs, THREADS, 0, s, (const T*)token, (const T*)a.weight, (const T*)a.ref_logp, pairs, x.inner, a.beta, a.smoothing,
               terms, coef, (T*)margins, (T*)logp);
  if (e == cudaSuccess && loss) e = sum_terms<T>(terms, pairs, loss, pairs ? 1.0 / (double)pairs : 0.0, s);
  if (e == cudaSuccess && g.data) e = t_grad<T>(x, labels, stats, PairCoef<T>{coef, (const T*)a.weight, std::max<long long>(x.inner, 1)}, g, s);
  return e;
}

template <typename T> cudaError_t t_distill(const RowView& x, const DistillArgs& a, void* loss, void* terms, const RowOut& g, cudaStream_t s) {
  Targets<T> tg{a.index, (const T*)a.teacher, (const T*)a.weight, a.k, (T)a.temperature, (T)(1 / a.temperature), (T*)terms};
  const size_t smem = (size_t)a.k * (2 * sizeof(T) + sizeof(int));
  cudaError_t e = cudaSuccess;
  if (x.rows() > 0)
    e = g.data ? launch(k_distill_rows<T, true>, row_blocks(x.rows()), THREADS, smem, s, view<T>(x), x.rows(), tg, out<T>(x, g))
               : launch(k_distill_rows<T, false>, row_blocks(x.rows()), THREADS, smem, s, view<T>(x), x.rows(), tg, Out<T>{});
  if (e != cudaSuccess || !loss) return e;
  return sum_terms<T>(terms, x.rows(), loss, 1.0, s);
}

}  // namespace

cudaError_t token_log_prob(EType t, const RowView& x, const int32_t* labels, void* logp, void* stats, cudaStream_t s) {
  return t == EType::F64 ? t_log_prob<double>(x, labels, logp, stats, s) : t_log_prob<float>(x, labels, logp, stats, s);
}

cudaError_t token_log_prob_grad(EType t, const RowView& x, const int32_t* labels, const void* stats, const void* dlogp, const RowOut& grad,
                                cudaStream_t s) {
  return t == EType::F64 ? t_grad<double>(x, labels, stats, TokenCoef<double>{(const double*)dlogp}, grad, s)
                         : t_grad<float>(x, labels, stats, TokenCoef<float>{(const float*)dlogp}, grad, s);
}

cudaError_t policy_loss(EType t, const RowView& x, const int32_t* labels, const PolicyArgs& a, void* loss, void* terms, void* logp,
                        const RowOut& grad, cudaStream_t s) {
  return t == EType::F64 ? t_policy<double>(x, labels, a, loss, terms, logp, grad, s) : t_policy<float>(x, labels, a, loss, terms, logp, grad, s);
}

size_t preference_workspace_bytes(EType t, long long sequences, long long length) {
  return (size_t)(3 * sequences * length + 3 * (sequences / 2)) * esize(t);
}

cudaError_t preference_loss(EType t, const RowView& x, const int32_t* labels, const PreferenceArgs& a, void* loss, void* margins, void* logp,
                            const RowOut& grad, void* workspace, cudaStream_t s) {
  return t == EType::F64 ? t_preference<double>(x, labels, a, loss, margins, logp, grad, workspace, s)
                         : t_preference<float>(x, labels, a, loss, margins, logp, grad, workspace, s);
}

cudaError_t distill_loss(EType t, const RowView& x, const DistillArgs& a, void* loss, void* terms, const RowOut& grad, cudaStream_t s) {
  return t == EType::F64 ? t_distill<double>(x, a, loss, terms, grad, s) : t_distill<float>(x, a, loss, terms, grad, s);
}

}  // namespace rgc
