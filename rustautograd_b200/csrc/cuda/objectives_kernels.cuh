// Kernels of the objectives over logits (objectives.cuh has the formulas).
//
// All of them are bound by memory: a row is V logits to read and, with a gradient, V values to write, against
// one exponential per logit. So each row is read from memory once and kept on chip until its gradient is
// written:
//  - k_group (rows up to 1024 floats): a group of 8, 16 or 32 lanes holds a row in registers;
//  - k_block (longer rows, with a gradient): a block, or the blocks of a cluster, hold a row in registers,
//    16-byte pieces arriving through shared memory (cp.async) while the row before is computed;
//  - k_stream (longer rows, no gradient): a running maximum and sum, nothing is held;
//  - k_two_pass (rows longer than a cluster holds): reads the row twice;
//  - k_grad: gradients whose coefficients need more than their row (token_log_prob_grad, preferences).
//
// Numbers. Row statistics are held in the logits' type. For float, exp(x - m) is computed as
// 2^((x - m) * log2 e) with the hardware's ex2: the difference and the product are rounded, 2.3 u |x - m|
// relatively (log2 e as a float is 0.22 u off), and ex2 is within 2 ulp; against expf that halves the
// instructions per logit. What a row reports (its log-probability's terms) is computed from the statistics
// in double by one lane, and sums over rows are double: a loss is a sum of terms of both signs.
// Everything is summed in a fixed order: the same inputs give the same bits on every call. The bits of a row do
// depend on how it is split over lanes and blocks, which goes by the vocabulary and the row count.
#pragma once
#include "objectives.cuh"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <map>
#include <mutex>
#include <tuple>
#include <type_traits>

namespace rgc {

namespace {

__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, unsigned cluster, cudaStream_t s, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

// ---- numbers ----

template <typename T> struct Num;
template <> struct Num<float> {
  static constexpr int VEC = 4;  // elements of a 16-byte vector
  using Vec = float4;
  // exp(d * scale), given scale * log2 e
  static __device__ __forceinline__ float exps(float d, float k) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * k));
    return r;
  }
  static __device__ __forceinline__ float most(float a, float b) { return fmaxf(a, b); }  // a NaN gives the other
  static float factor(double scale) { return (float)(scale * 1.4426950408889634074); }
};
template <> struct Num<double> {
  static constexpr int VEC = 2;
  using Vec = double2;
  static __device__ __forceinline__ double exps(double d, double k) { return exp(d * k); }
  static __device__ __forceinline__ double most(double a, double b) { return fmax(a, b); }
  static double factor(double scale) { return scale; }
};

template <typename T> __device__ __forceinline__ T neg_inf() { return -(T)INFINITY; }
// What exponentials are taken relative to: the maximum, or 0 where there is no finite one yet.
template <typename T> __device__ __forceinline__ T base(T m) { return m == neg_inf<T>() ? (T)0 : m; }

// (max, sum of exp((x - max) * scale)) of a part of a row. A part without a finite maximum has m = -inf and
// s = 0; NaN and +inf elements make s NaN, as the formulas do.
template <typename T> struct Stat {
  T m = -(T)INFINITY, s = (T)0;
};

template <typename T> struct alignas(2 * sizeof(T)) Pair {
  T m, s;
};

template <int G, typename T> __device__ __forceinline__ Stat<T> join(Stat<T> a, T k) {
  T m = a.m;
#pragma unroll
  for (int d = G / 2; d; d >>= 1) {
    m = Num<T>::most(m, __shfl_xor_sync(~0u, m, d));
  }
  T s = a.s * Num<T>::exps(a.m - base(m), k);
#pragma unroll
  for (int d = G / 2; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
  return {m, s};
}

// ---- rows in memory ----

// Quotients of row numbers (below 2^31) by run-time divisors: a multiplication and a shift (FDiv).
__device__ __forceinline__ unsigned quotient(unsigned n, const FDiv& f) { return (unsigned)(((unsigned long long)__umulhi(n, f.m) + n) >> f.s); }

template <typename T> struct View {
  const T* data;
  FDiv inner;
  long long v, so, si;
  __device__ __forceinline__ const T* row(long long r) const {
    const unsigned a = quotient((unsigned)r, inner);
    return data + a * so + ((unsigned)r - a * inner.d) * si;
  }
};
template <typename T> struct Out {
  T* data;
  FDiv inner;
  long long so, si;
  __device__ __forceinline__ T* row(long long r) const {
    const unsigned a = quotient((unsigned)r, inner);
    return data + a * so + ((unsigned)r - a * inner.d) * si;
  }
};

// A row as 16-byte vectors from an aligned address: element j is element (j + off) % VEC of vector
// (j + off) / VEC. The first and the last vector may hold elements that are not the row's: those
// are neither read nor written. A part of a row is the same with narrower bounds.
template <typename T> struct Span {
  static constexpr int VEC = Num<T>::VEC;
  T* base;
  int off, lo, hi;  // the elements are lo .. hi - 1, counted from `base`
  template <typename P> __device__ __forceinline__ Span(P* row, long long vocab) {
    off = (int)(((unsigned long long)row / sizeof(T)) % VEC);
    base = const_cast<T*>(row) - off;
    lo = off;
    hi = (int)vocab + off;
  }
  // Only vectors first .. end - 1.
  __device__ __forceinline__ void clip(int first, int end) {
    lo = max(lo, first * VEC);
    hi = min(hi, end * VEC);
  }
  // The 16 bytes from element j on are all the row's.
  __device__ __forceinline__ bool whole(int j) const { return j >= lo && j <= hi - VEC; }
  __device__ __forceinline__ bool has(int j) const { return j >= lo && j < hi; }
  // Vector i, or -inf for elements that are not the row's.
  __device__ __forceinline__ void load(int i, T* x) const {
    if (whole(i * VEC)) {
      const typename Num<T>::Vec t = *reinterpret_cast<const typename Num<T>::Vec*>(base + (long long)i * VEC);
      memcpy(x, &t, 16);
    } else {
#pragma unroll
      for (int c = 0; c < VEC; ++c) x[c] = has(i * VEC + c) ? base[(long long)i * VEC + c] : neg_inf<T>();
    }
  }
};

// Stores the vectors first + lane + G * e (e < E, values y) of a row whose logits span `x` to the row at
// `row`, G lanes together. Where that row is aligned to 16 bytes as the logits are, a logits vector is an
// output vector; where it is not, an output vector begins SH elements into a logits vector and ends in
// the next one, which the right neighbour holds (lane 0's next vector for the last lane). The elements
// before the group's first whole output vector and behind its last go one by one.
// (A slice of positions of logits with an odd vocabulary has every alignment.)
// INSIDE: all of the group's vectors are the row's.
template <typename T, int G, int E, int SH, bool INSIDE>
__device__ __forceinline__ void store_shifted(T* at0, const Span<T>& x, int first, int lane, const T* y) {
  constexpr int VEC = Num<T>::VEC;
  const int end = min(x.hi, (first + G * E) * VEC);  // what the group holds
#pragma unroll
  for (int e = 0; e < E; ++e) {
    T o[VEC];
#pragma unroll
    for (int c = 0; c < VEC - SH; ++c) o[c] = y[e * VEC + SH + c];
#pragma unroll
    for (int c = 0; c < SH; ++c) {
      const T ahead = e + 1 < E ? y[(e + 1 < E ? e + 1 : e) * VEC + c] : y[e * VEC + c];
      o[VEC - SH + c] = __shfl_sync(~0u, lane == 0 ? ahead : y[e * VEC + c], (lane + 1) % G, G);
    }
    const int j = (first + lane + G * e) * VEC + SH;
    T* at = at0 + j;
    if (INSIDE ? SH == 0 || e < E - 1 || lane < G - 1 : j >= x.lo && j <= end - VEC) {
      typename Num<T>::Vec t;
      memcpy(&t, o, 16);
      *reinterpret_cast<typename Num<T>::Vec*>(at) = t;
    } else {
#pragma unroll
      for (int c = 0; c < VEC; ++c)
        if (INSIDE ? c < VEC - SH : j + c >= x.lo && j + c < end) at[c] = o[c];
    }
    if (SH > 0 && e == 0 && lane == 0) {
#pragma unroll
      for (int c = 0; c < SH; ++c)
        if (INSIDE || x.has(j - SH + c)) at[c - SH] = y[c];
    }
  }
}
template <typename T, int G, int E, bool INSIDE> __device__ __forceinline__ void store(T* row, const Span<T>& x, int first, int lane, const T* y) {
  constexpr int VEC = Num<T>::VEC;
  const int goff = (int)(((unsigned long long)row / sizeof(T)) % VEC), sh = (x.off - goff + VEC) % VEC;
  T* at0 = row - x.off;  // where element 0 of `x` would go
  if (sh == 0) store_shifted<T, G, E, 0, INSIDE>(at0, x, first, lane, y);
  else if (sh == 1) store_shifted<T, G, E, 1, INSIDE>(at0, x, first, lane, y);
  if constexpr (VEC == 4) {
    if (sh == 2) store_shifted<T, G, E, 2, INSIDE>(at0, x, first, lane, y);
    else if (sh == 3) store_shifted<T, G, E, 3, INSIDE>(at0, x, first, lane, y);
  }
}

// The same for the groups of a warp, each with a row of its own (and an alignment of its own).
template <typename T, int G, int E> __device__ __forceinline__ void store_group(T* row, const Span<T>& x, int lane, const T* y) {
  constexpr int VEC = Num<T>::VEC;
  if constexpr (G == 32) {
    store<T, G, E, false>(row, x, 0, lane, y);
  } else {
    const int goff = (int)(((unsigned long long)row / sizeof(T)) % VEC), sh = (x.off - goff + VEC) % VEC;
    T* at0 = row - x.off;
    if (__all_sync(~0u, sh == 0)) {
      store_shifted<T, G, E, 0, false>(at0, x, 0, lane, y);
      return;
    }
    // Some of the warp's rows are shifted: element by element.
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        const int j = (lane + G * e) * VEC + c;
        if (x.has(j)) at0[j] = y[e * VEC + c];
      }
    }
  }
}

__device__ __forceinline__ long long clamp_label(int l, long long v) { return l < 0 ? 0 : l >= v ? v - 1 : l; }

// ---- objectives ----
//
// With one target per row: Meta is what a row needs besides its logits. `coef` gives the coefficient c of
// (onehot - p) from the label's logit and the row's statistics; `report` (one lane) writes what the row
// reports. `skip` is `report` for a row that is not live.

template <typename T> struct LogProbRow {
  static constexpr bool TARGETS = false, GIVEN = false;
  const int32_t* labels;
  T *logp, *stats;
  struct Meta {
    int label;
    T w;
    __device__ __forceinline__ bool live() const { return w != (T)0; }
  };
  __device__ __forceinline__ Meta meta(long long r) const { return {labels[r], (T)1}; }
  __device__ void skip(long long) const {}
  __device__ __forceinline__ T coef(const Meta&, T, Stat<T>) const { return (T)0; }
  __device__ __forceinline__ void report(long long r, const Meta&, T xl, Stat<T> st) const {
    if (logp) logp[r] = (T)(((double)xl - (double)st.m) - log((double)st.s));
    if (stats) {
      stats[2 * r] = st.m;
      stats[2 * r + 1] = st.s;
    }
  }
};

template <typename T> struct PolicyRow {
  static constexpr bool TARGETS = false, GIVEN = false;
  const int32_t* labels;
  const T *old_logp, *ref_logp, *advantage, *weight;
  T low, high, kl;  // the ratio's bounds 1 - clip_low and 1 + clip_high
  T *terms, *logp;
  struct Meta {
    int label;
    T w, a, old, ref;
    __device__ __forceinline__ bool live() const { return w != (T)0; }
  };
  __device__ __forceinline__ Meta meta(long long r) const {
    Meta m;
    m.w = weight[r];
    m.label = labels[r];
    m.a = advantage[r];
    m.old = old_logp[r];
    m.ref = kl != (T)0 ? ref_logp[r] : (T)0;
    return m;
  }
  // The same from one value per lane of a warp.
  __device__ __forceinline__ T field(long long r, int lane) const {
    return lane == 0 ? weight[r] : lane == 1 ? advantage[r] : lane == 2 ? old_logp[r] : lane == 3 && kl != (T)0 ? ref_logp[r] : (T)0;
  }
  __device__ __forceinline__ Meta gather(int label, T f) const {
    return {label, __shfl_sync(~0u, f, 0), __shfl_sync(~0u, f, 1), __shfl_sync(~0u, f, 2), __shfl_sync(~0u, f, 3)};
  }
  __device__ void skip(long long r) const {
    terms[r] = (T)0;
    if (logp) logp[r] = (T)0;
  }
  __device__ __forceinline__ T coef(const Meta& m, T xl, Stat<T> st) const {
    const T lp = (xl - st.m) - ln(st.s), ratio = ex(lp - m.old);
    T c = (m.a >= (T)0 ? ratio <= high : ratio >= low) ? -(ratio * m.a) : (T)0;
    if (kl != (T)0) c += kl * ((T)1 - ex(m.ref - lp));
    return m.w * c;
  }
  __device__ __forceinline__ void report(long long r, const Meta& m, T xl, Stat<T> st) const {
    const double lp = ((double)xl - (double)st.m) - log((double)st.s), ratio = exp(lp - (double)m.old), a = m.a;
    const double held = ratio < (double)low ? (double)low : ratio > (double)high ? (double)high : ratio;
    // A NaN ratio or advantage stays NaN through both comparisons.
    double term = ratio * a > held * a ? -(held * a) : -(ratio * a);
    if (kl != (T)0) {
      const double d = (double)m.ref - lp;
      term += (double)kl * (exp(d) - d - 1);
    }
    terms[r] = (T)((double)m.w * term);
    if (logp) logp[r] = (T)lp;
  }
  static __device__ __forceinline__ float ex(float v) { return expf(v); }
  static __device__ __forceinline__ double ex(double v) { return exp(v); }
  static __device__ __forceinline__ float ln(float v) { return logf(v); }
  static __device__ __forceinline__ double ln(double v) { return log(v); }
};

// Coefficients that need more than the row: the statistics are those of an earlier pass. c = by_row[r], or
// by_sequence[r / length] * weight[r].
template <typename T> struct GivenRow {
  static constexpr bool TARGETS = false, GIVEN = true;
  const int32_t* labels;
  const T *stats, *by_row, *by_sequence, *weight;
  FDiv length;
  struct Meta {
    int label;
    T w, c, m, s;
    __device__ __forceinline__ bool live() const { return w != (T)0; }
  };
  __device__ __forceinline__ Meta meta(long long r) const {
    Meta q;
    if (by_row) {
      q.w = q.c = by_row[r];
    } else {
      q.w = weight[r];
      q.c = q.live() ? by_sequence[quotient((unsigned)r, length)] * q.w : (T)0;
    }
    q.label = labels[r];
    q.m = stats[2 * r];
    q.s = stats[2 * r + 1];
    return q;
  }
  __device__ void skip(long long) const {}
  __device__ __forceinline__ T coef(const Meta& q, T, Stat<T>) const { return q.c; }
  __device__ __forceinline__ void report(long long, const Meta&, T, Stat<T>) const {}
};

struct EntriesPart {
  double a, q;
  bool some;  // the row has entries
};

// The distillation: a row's targets are its teacher entries. `prepare` (one warp) gives q at shared arrays
// and the part of the term that does not need the row's statistics:
// sum q (log q - log p_i) = sum q (log q - x_i / T) + (m / T + log s) sum q.
template <typename T> struct DistillRow {
  static constexpr bool TARGETS = true, GIVEN = false;
  const int32_t* index;
  const T *teacher, *weight;
  long long k;
  double inverse;  // 1 / T
  T tk;            // Num<T>::factor(1 / T)
  T wt;            // T
  T* terms;
  struct Meta {
    T w;
    __device__ __forceinline__ bool live() const { return w != (T)0; }
  };
  using Part = EntriesPart;
  __device__ __forceinline__ Meta meta(long long r) const {
    return {weight[r]};
  }
  __device__ void skip(long long r) const { terms[r] = (T)0; }
  __device__ __forceinline__ void report(long long r, const Meta& m, Part p, Stat<T> st) const {
    const double lse = (double)st.m * inverse + log((double)st.s);
    terms[r] = p.some ? (T)((double)m.w * (double)wt * (double)wt * (p.a + lse * p.q)) : (T)0;
  }
  // One warp; x: the row's logits. Keeps q, the index and its logit of each entry when `at` is given.
  __device__ Part prepare(long long r, const T* x, long long v, int lane, int* at, T* q, T* xk) const {
    const T* t = teacher + r * k;
    const int32_t* ix = index + r * k;
    Stat<T> st;
    for (long long i = lane; i < k; i += 32) {
      const T z = t[i], m = z > st.m ? z : st.m;
      st.s = st.s * Num<T>::exps(st.m - base(m), tk) + Num<T>::exps(z - base(m), tk);
      st.m = m;
    }
    st = join<32>(st, tk);
    Part p{0, 0, false};
    p.some = st.s != (T)0;  // all entries -inf: none
    const T inv = (T)1 / st.s;
    const double logs = log((double)st.s);
    for (long long i = lane; i < k; i += 32) {
      const long long l = clamp_label(ix[i], v);
      const T d = t[i] - base(st.m), qi = p.some ? Num<T>::exps(d, tk) * inv : (T)0, xi = x[l];
      if (at) {
        at[i] = (int)l;
        q[i] = qi;
        xk[i] = xi;
      }
      if (qi != (T)0) {
        p.a += (double)qi * (((double)d - (double)xi) * inverse - logs);
        p.q += (double)qi;
      }
    }
    for (int d = 16; d; d >>= 1) {
      p.a += __shfl_xor_sync(~0u, p.a, d);
      p.q += __shfl_xor_sync(~0u, p.q, d);
    }
    return p;
  }
};

// ---- short rows: a group of G lanes per row ----

constexpr int GROUP_THREADS = 256;

// The maximum of a thread's N logits, their exponentials in place and the sum of these.
template <typename T, int N> __device__ __forceinline__ Stat<T> exponentials(T* x, T k) {
  Stat<T> a;
#pragma unroll
  for (int i = 0; i < N; ++i) a.m = Num<T>::most(x[i], a.m);
  const T b = base(a.m);
  // Two sums: half the rounding of one long chain, and half its latency.
  T s0 = (T)0, s1 = (T)0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = Num<T>::exps(x[i] - b, k);
    if (i % 2) s1 += x[i];
    else s0 += x[i];
  }
  a.s = s0 + s1;
  return a;
}

// The same of the first `turns` of E vectors.
template <typename T, int E, int VEC> __device__ __forceinline__ Stat<T> exponentials(T* x, T k, int turns) {
  Stat<T> a;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < turns) {
#pragma unroll
      for (int c = 0; c < VEC; ++c) a.m = Num<T>::most(x[e * VEC + c], a.m);
    }
  const T b = base(a.m);
  T s0 = (T)0, s1 = (T)0;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < turns) {
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        T& z = x[e * VEC + c];
        z = Num<T>::exps(z - b, k);
        if (c % 2) s1 += z;
        else s0 += z;
      }
    }
  a.s = s0 + s1;
  return a;
}

// What this thread's exponentials are multiplied by to give scale * p.
template <typename T> __device__ __forceinline__ T share(T m, Stat<T> st, T k, T scale) {
  return (m == neg_inf<T>() ? (T)0 : Num<T>::exps(m - base(st.m), k)) * (scale / st.s);
}

template <typename T, int G, int E, class Obj, bool GRAD>
__global__ void __launch_bounds__(GROUP_THREADS) k_group(View<T> x, long long rows, Obj obj, T k, Out<T> g) {
  constexpr int VEC = Num<T>::VEC, PER_WARP = 32 / G;
  pdl_wait();
  extern __shared__ __align__(16) unsigned char dyn[];
  const int lane = threadIdx.x % G;
  const long long warps = (long long)gridDim.x * (GROUP_THREADS / 32);
  // All groups of a warp take the same number of turns: shuffles name the whole warp.
  for (long long w = (long long)blockIdx.x * (GROUP_THREADS / 32) + threadIdx.x / 32; w * PER_WARP < rows; w += warps) {
    const long long r = w * PER_WARP + (threadIdx.x % 32) / G;
    const bool in = r < rows;
    typename Obj::Meta meta{};
    if (in) meta = obj.meta(r);
    const bool live = in && meta.live();
    const Span<T> row(x.row(in ? r : 0), in ? x.v : 0);
    T y[E * VEC];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (live) {
        row.load(lane + G * e, y + e * VEC);
      } else {
#pragma unroll
        for (int c = 0; c < VEC; ++c) y[e * VEC + c] = neg_inf<T>();
      }
    }
    if constexpr (!Obj::TARGETS) {
      const int l = live ? (int)clamp_label(meta.label, x.v) + row.off : 0;
      T xl = (T)0;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (lane + G * e == l / VEC) {
#pragma unroll
          for (int c = 0; c < VEC; ++c)
            if (l % VEC == c) xl = y[e * VEC + c];
        }
      Stat<T> st;
      T c, f;
      if constexpr (Obj::GIVEN) {
        st = {meta.m, meta.s};
        c = meta.c;
        f = -c / st.s;
#pragma unroll
        for (int q = 0; q < E * VEC; ++q) y[q] = Num<T>::exps(y[q] - st.m, k);
      } else {
        xl = __shfl_sync(~0u, xl, (l / VEC) % G, G);
        const Stat<T> own = exponentials<T, E * VEC>(y, k);
        st = join<G>(own, k);
        c = live ? obj.coef(meta, xl, st) : (T)0;
        f = share(own.m, st, k, -c);
      }
      if (GRAD) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
#pragma unroll
          for (int q = 0; q < VEC; ++q) y[e * VEC + q] = live ? y[e * VEC + q] * f : (T)0;
          if (live && lane + G * e == l / VEC) {
#pragma unroll
            for (int q = 0; q < VEC; ++q)
              if (l % VEC == q) y[e * VEC + q] += c;
          }
        }
        store_group<T, G, E>(g.row(in ? r : 0), row, lane, y);
      }
      if (lane == 0 && in) {
        if (live) obj.report(r, meta, xl, st);
        else obj.skip(r);
      }
    } else {
      // Per warp: the targets' total probability at each of the row's elements, and the entries.
      T* hit = (T*)dyn + (threadIdx.x / 32) * (E * 32 * VEC + 2 * obj.k);
      T* q = hit + E * 32 * VEC;
      T* xk = q + obj.k;
      int* at = (int*)((T*)dyn + (GROUP_THREADS / 32) * (E * 32 * VEC + 2 * obj.k)) + (threadIdx.x / 32) * obj.k;
      typename Obj::Part part{0, 0, false};
      if (live) part = obj.prepare(r, x.row(r), x.v, lane, GRAD ? at : nullptr, q, xk);
      const bool some = live && part.some;
      if (GRAD && some) {
#pragma unroll
        for (int e = 0; e < E * VEC; ++e) hit[lane + 32 * e] = (T)0;
        __syncwarp();
        // 32 entries at a time: the first lane of those with the same index adds them up in order.
        for (long long i0 = 0; i0 < obj.k; i0 += 32) {
          const long long i = i0 + lane;
          const bool on = i < obj.k;
          const int l = on ? at[i] : -1 - lane;
          unsigned same = __match_any_sync(~0u, l);
          const bool first = (same & ((1u << lane) - 1)) == 0;
          if (on && first) {
            T sum = hit[l + row.off];
            for (; same; same &= same - 1) sum += q[i0 + __ffs(same) - 1];
            hit[l + row.off] = sum;
          }
          __syncwarp();
        }
      }
      const Stat<T> own = exponentials<T, E * VEC>(y, k);
      const Stat<T> st = join<G>(own, k);
      if (GRAD) {
        const T c = meta.w * obj.wt, f = some ? share(own.m, st, k, c) : (T)0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
#pragma unroll
          for (int z = 0; z < VEC; ++z) y[e * VEC + z] = some ? y[e * VEC + z] * f - c * hit[(lane + 32 * e) * VEC + z] : (T)0;
        }
        store_group<T, G, E>(g.row(in ? r : 0), row, lane, y);
        __syncwarp();
      }
      if (lane == 0 && in) {
        if (live) obj.report(r, meta, part, st);
        else obj.skip(r);
      }
    }
  }
}

// ---- longer rows: a block, or a cluster of blocks, per row ----

__device__ __forceinline__ unsigned smem_addr(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned cluster_size() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Writes (m, s) to the shared memory of block `rank` of the cluster, at the place `p` has in this one's.
template <typename T> __device__ __forceinline__ void put_remote(Pair<T>* p, unsigned rank, Pair<T> v) {
  unsigned a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
  if constexpr (sizeof(T) == 4)
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(v.m), "f"(v.s) : "memory");
  else
    asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(a), "d"(v.m), "d"(v.s) : "memory");
}
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
// With constant distances (bytes) from both addresses.
template <int TO, int FROM> __device__ __forceinline__ void copy16_at(unsigned dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(dst), "l"(src), "n"(TO), "n"(FROM) : "memory");
}
template <int BYTES> __device__ __forceinline__ void copy_element(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_addr(dst)), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_done_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

constexpr int MAX_CLUSTER = 8;

// Row statistics over all warps of a block (CLUSTER: of the cluster's blocks): every warp's (m, s) goes to a
// table that is written in turn to one of two halves, so one barrier per row is enough. Every thread gets
// the result.
template <typename T, int NW, bool CLUSTER> struct Table {
  static constexpr int SLOTS = NW * (CLUSTER ? MAX_CLUSTER : 1);
  Pair<T> slot[2][SLOTS];
  Pair<T> extra[2];  // one more value for every block
  __device__ __forceinline__ void write(int half, Stat<T> st, unsigned rank, unsigned blocks) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    if constexpr (CLUSTER) {
      if (lane < (int)blocks) put_remote(&slot[half][rank * NW + warp], (unsigned)lane, Pair<T>{st.m, st.s});
    } else {
      if (lane == 0) slot[half][warp] = {st.m, st.s};
    }
  }
  __device__ __forceinline__ Stat<T> read(int half, unsigned blocks, T k) const {
    const int n = CLUSTER ? NW * (int)blocks : NW;
    Stat<T> a;
    for (int i = threadIdx.x % 32; i < n; i += 32) {
      const Pair<T> b = slot[half][i];
      const T m = b.m > a.m ? b.m : a.m;
      a.s = a.s * Num<T>::exps(a.m - base(m), k) + b.s * Num<T>::exps(b.m - base(m), k);
      a.m = m;
    }
    return join<32>(a, k);
  }
};

// Entries of a row's distillation targets, kept until its gradient has been written.
template <typename T> struct Kept {
  long long row = -1;
  T c = 0, scale = 0, m = 0;  // the gradient at an entry: exp((x - m) k) scale - c sum q
};

// f(0) .. f(N - 1) with compile-time numbers.
template <int N, int I = 0, typename F> __device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<N, I + 1>(f);
  }
}

// What a row's gradient needs, from one warp to all.
template <typename T> struct Scalars {
  T c, scale, m;  // c; the factor of exp((x - m) k); m
  int at;         // the label's element, counted as a Span's; or whether the row has entries
};

// Calls, not inlined: one warp makes them while every warp's registers hold a row.
template <typename T, class Obj> __device__ __noinline__ T coef_of(const Obj& obj, int label, T fields, T xl, Stat<T> st) {
  return obj.coef(obj.gather(label, fields), xl, st);
}
template <typename T, class Obj> __device__ __noinline__ void report_of(const Obj& obj, long long r, int label, T fields, T xl, Stat<T> st) {
  const typename Obj::Meta m = obj.gather(label, fields);
  if (threadIdx.x % 32 == 0) obj.report(r, m, xl, st);
}
template <typename T, class Obj>
__device__ __noinline__ void entries_of(const Obj& obj, long long r, const T* x, long long v, int* at, T* q, T* xk, typename Obj::Part* part) {
  const typename Obj::Part p = obj.prepare(r, x, v, threadIdx.x % 32, at, q, xk);
  if (threadIdx.x % 32 == 0) *part = p;
}
template <typename T, class Obj> __device__ __noinline__ void report_entries(const Obj& obj, long long r, const typename Obj::Part& part, Stat<T> st) {
  if (threadIdx.x % 32 == 0) obj.report(r, obj.meta(r), part, st);
}

// A block of NT threads (or a cluster of such blocks, `slice` vectors each) per row. A warp holds 32 * turns
// adjacent vectors of its block's slice in registers (turns <= E), as vectors of the gradient, which are stored
// whole; the logits they need come through the warp's own piece of shared memory, where an offset between the
// alignments of the two (a slice of positions of logits with an odd vocabulary has every one) costs element-wise
// reads and nothing else. The copies of the next STAGES rows are under way meanwhile: a warp copies what it
// will read itself, so no block-wide barrier stands between copy and use.
// Issue slots are what is scarce (45 per logit and lane at the copy rate), so warps whose vectors are all inside
// the row take a path without bounds, and what a row needs once is computed by one warp.
template <typename T, int NT, int E, int STAGES, bool CLUSTER, class Obj>
__global__ void __launch_bounds__(NT, 512 / NT)
    k_block(const View<T> x, const long long rows, const __grid_constant__ Obj obj, const T k, const Out<T> g, const int slice, const int turns) {
  constexpr int VEC = Num<T>::VEC, NW = NT / 32, PIECE = 32 * E + 1;  // a piece has one vector more for the offset
  using Vec = typename Num<T>::Vec;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Table<T, NW, CLUSTER> table;
  __shared__ Scalars<T> scalars;
  const unsigned rank = CLUSTER ? cluster_rank() : 0, blocks = CLUSTER ? cluster_size() : 1;
  const long long step = gridDim.x / blocks, first = blockIdx.x / blocks;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  Vec* ring = (Vec*)dyn + warp * STAGES * PIECE;
  // This warp's first vector; this thread's are warp0 + lane + 32 * e.
  const int begin = (int)rank * slice, warp0 = begin + warp * 32 * turns;
  pdl_wait();
  if constexpr (CLUSTER) cluster_sync();  // every block's shared memory is there before another writes to it

  // Row r, elements counted from the gradient's 16-byte boundary before it: element u is logit u - off. The
  // warp's piece begins `shift` elements before its first element.
  struct Place {
    const T* from;  // the piece's first logit, 16-byte aligned
    T* to;          // the gradient's element 0
    int off, lo, hi, shift;
  };
  auto place = [&](long long r) {
    Place q;
    T* gr = g.row(r);
    q.off = (int)(((unsigned long long)gr / sizeof(T)) % VEC);
    q.to = gr - q.off;
    q.lo = max(q.off, begin * VEC);
    q.hi = min(q.off + (int)x.v, (begin + slice) * VEC);
    const T* at = x.row(r) + ((long long)warp0 * VEC - q.off);
    q.shift = (int)(((unsigned long long)at / sizeof(T)) % VEC);
    q.from = at - q.shift;
    return q;
  };
  const int last = warp0 + 32 * turns;
  auto inside = [&](const Place& q) { return warp0 * VEC >= q.lo && last * VEC <= q.hi; };
  auto fetch = [&](long long r, int stage) {
    const Place q = place(r);
    Vec* to = ring + stage * PIECE;
    // The row's elements in the piece: from_lo .. from_hi - 1 of it.
    const int from_lo = q.off - (warp0 * VEC - q.shift), from_hi = from_lo + (int)x.v, need = min(q.hi - warp0 * VEC, 32 * turns * VEC) + q.shift;
    if (from_lo <= 0 && from_hi >= (32 * turns + 1) * VEC && need > 0) {
      const unsigned d = smem_addr(to + lane);
      const T* from = q.from + lane * VEC;
      each<E>([&](auto e) {
        if (e < turns) copy16_at<e * 512, e * 512>(d, from);
      });
      if (q.shift && lane == 0) copy16(to + 32 * turns, q.from + 32 * turns * VEC);
    } else if (need > 0) {
#pragma unroll 1
      for (int i = lane; i * VEC < need; i += 32) {
        const int j = i * VEC;
        if (j >= from_lo && j + VEC <= from_hi) {
          copy16(to + i, q.from + j);
        } else {
#pragma unroll 1
          for (int c = 0; c < VEC; ++c)
            if (j + c >= from_lo && j + c < from_hi) copy_element<sizeof(T)>((T*)(to + i) + c, q.from + j + c);
        }
      }
    }
  };
  // Distillation: two halves of k entries each, the row they belong to, and what its gradient needs.
  T* tq = (T*)((Vec*)dyn + NW * STAGES * PIECE);
  T* tx = nullptr;
  int* ti = nullptr;
  Kept<T> kept;
  if constexpr (Obj::TARGETS) {
    tx = tq + 2 * obj.k;
    ti = (int*)(tx + 2 * obj.k);
  }
  __shared__ typename std::conditional<Obj::TARGETS, EntriesPart, int>::type part;
  // After a barrier that orders the row's gradient before it: the entries of the row. The first entry
  // of an index writes its element, with the probabilities of all entries of that index in order.
  auto finish = [&](int half) {
    if constexpr (Obj::TARGETS) {
      if (rank != 0 || kept.row < 0) return;
      T* gr = g.row(kept.row);
      const int* ix = ti + half * obj.k;
      const T* q = tq + half * obj.k;
#pragma unroll 1
      for (int i = threadIdx.x; i < (int)obj.k; i += NT) {
        const int l = ix[i];
        T sum = (T)0;
        bool leads = true;
#pragma unroll 1
        for (int o = 0; o < (int)obj.k; ++o) {
          if (ix[o] != l) continue;
          leads = leads && o >= i;
          sum += q[o];
        }
        if (leads) gr[l] = Num<T>::exps(tx[half * obj.k + i] - kept.m, k) * kept.scale - kept.c * sum;
      }
    }
  };

  // Row r's operands are read a turn before they are used: the weights by everyone, the rest by the first
  // warp, whose lanes hold one value each.
  T weight[STAGES + 1], fields = (T)0, target = (T)0;
  int label = 0;
#pragma unroll
  for (int a = 0; a <= STAGES; ++a) weight[a] = first + a * step < rows ? obj.weight[first + a * step] : (T)0;
#pragma unroll
  for (int a = 0; a < STAGES; ++a) {
    if (weight[a] != (T)0) fetch(first + a * step, a);
    copies_done_group();
  }
  if constexpr (!Obj::TARGETS)
    if (warp == 0 && weight[0] != (T)0) {
      label = obj.labels[first];
      fields = obj.field(first, lane);
      target = x.row(first)[clamp_label(label, x.v)];
    }
  int stage = 0, half = 0;
  for (long long r = first; r < rows; r += step) {
    const bool live = weight[0] != (T)0;
    const T now_weight = weight[0], now_fields = fields, xl = target;
    const int now_label = label;
#pragma unroll
    for (int a = 0; a < STAGES; ++a) weight[a] = weight[a + 1];
    weight[STAGES] = r + (STAGES + 1) * step < rows ? obj.weight[r + (STAGES + 1) * step] : (T)0;
    if constexpr (Obj::TARGETS) {
      // The first warp of the cluster's first block: the row's entries (before any of its gradient is
      // written, which may be in the logits' place).
      if (live && rank == 0 && warp == 0) {
        entries_of<T, Obj>(obj, r, x.row(r), x.v, ti + half * obj.k, tq + half * obj.k, tx + half * obj.k, &part);
        __syncwarp();
        const Pair<T> some{part.some ? (T)1 : (T)0, (T)0};
        if constexpr (CLUSTER) {
          if (lane < (int)blocks) put_remote(&table.extra[half], (unsigned)lane, some);
        } else {
          if (lane == 0) table.extra[half] = some;
        }
      }
    } else if (warp == 0 && weight[0] != (T)0) {
      label = obj.labels[r + step];
      fields = obj.field(r + step, lane);
    }
    const Place row = place(r);
    const bool fast = inside(row);
    T y[E * VEC];
    Stat<T> own;
    copies_wait<STAGES - 1>();
    __syncwarp();
    if (live) {
      const Vec* from = ring + stage * PIECE + lane;
      if (row.shift == 0) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e < turns) {
            const Vec t = from[32 * e];
            memcpy(y + e * VEC, &t, 16);
          }
      } else {
        const T* el = (const T*)from + row.shift;
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e < turns) {
#pragma unroll
            for (int c = 0; c < VEC; ++c) y[e * VEC + c] = el[32 * VEC * e + c];
          }
      }
      if (!fast) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e < turns) {
            const int u = (warp0 + lane + 32 * e) * VEC;
            if (u < row.lo || u + VEC > row.hi) {
#pragma unroll
              for (int c = 0; c < VEC; ++c)
                if (u + c < row.lo || u + c >= row.hi) y[e * VEC + c] = neg_inf<T>();
            }
          }
      }
      own = exponentials<T, E, VEC>(y, k, turns);
    }
    // All that was copied has been used: the next row into its place.
    __syncwarp();
    if (weight[STAGES - 1] != (T)0) fetch(r + STAGES * step, stage);
    copies_done_group();
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    if constexpr (!Obj::TARGETS)
      if (warp == 0 && weight[0] != (T)0) target = x.row(r + step)[clamp_label(label, x.v)];
    if (!live) {
      if (rank == 0 && threadIdx.x == 0) obj.skip(r);
#pragma unroll
      for (int q = 0; q < E * VEC; ++q) y[q] = (T)0;
    } else {
      table.write(half, join<32>(own, k), rank, blocks);
      if constexpr (CLUSTER) cluster_sync();
      else __syncthreads();
      Stat<T> st;
      if (warp == 0) {
        st = table.read(half, blocks, k);
        Scalars<T> s;
        s.m = st.m;
        if constexpr (Obj::TARGETS) {
          // A row without entries counts nothing.
          s.at = table.extra[half].m != (T)0;
          s.c = now_weight * obj.wt;
          s.scale = s.c / st.s;
        } else {
          s.at = (int)clamp_label(now_label, x.v);
          s.c = coef_of<T, Obj>(obj, now_label, now_fields, xl, st);
          s.scale = -s.c / st.s;
        }
        if (lane == 0) scalars = s;
      }
      finish(half ^ 1);  // of the row before
      __syncthreads();
      const Scalars<T> s = scalars;
      const T fs = own.m == neg_inf<T>() ? (T)0 * s.scale : Num<T>::exps(own.m - base(s.m), k) * s.scale;
      if constexpr (Obj::TARGETS) {
        kept.row = s.at ? r : -1;
        kept.c = s.c;
        kept.scale = s.scale;
        kept.m = s.m;
#pragma unroll
        for (int q = 0; q < E * VEC; ++q) y[q] = s.at ? y[q] * fs : (T)0;
        if (rank == 0 && warp == 0) report_entries<T, Obj>(obj, r, part, st);
      } else {
#pragma unroll
        for (int q = 0; q < E * VEC; ++q) y[q] *= fs;
        const int l = s.at + row.off - warp0 * VEC;  // within the warp's vectors
        if (l >= 0 && l < 32 * turns * VEC && (l / VEC) % 32 == lane) {
#pragma unroll
          for (int q = 0; q < E * VEC; ++q)
            if (q == l / (32 * VEC) * VEC + l % VEC) y[q] += s.c;
        }
        if (rank == 0 && warp == 0) report_of<T, Obj>(obj, r, now_label, now_fields, xl, st);
      }
      half ^= 1;
    }
    T* to = row.to + (long long)(warp0 + lane) * VEC;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < turns) {
        const int u = (warp0 + lane + 32 * e) * VEC;
        if (fast || (u >= row.lo && u + VEC <= row.hi)) {
          Vec t;
          memcpy(&t, y + e * VEC, 16);
          *reinterpret_cast<Vec*>(to + 32 * VEC * e) = t;
        } else {
#pragma unroll
          for (int c = 0; c < VEC; ++c)
            if (u + c >= row.lo && u + c < row.hi) to[32 * VEC * e + c] = y[e * VEC + c];
        }
      }
  }
  if constexpr (Obj::TARGETS) {
    if constexpr (CLUSTER) cluster_sync();
    else __syncthreads();
    finish(half ^ 1);
  }
  if constexpr (CLUSTER) cluster_sync();  // no block leaves while another may still write to it
}

// ---- longer rows without a gradient ----

constexpr int STREAM_THREADS = 256, STREAM_UNROLL = 4;

// A block, or a cluster of blocks, per row: a running maximum and sum per thread, four vectors at a time.
template <typename T, bool CLUSTER, class Obj>
__global__ void __launch_bounds__(STREAM_THREADS) k_stream(View<T> x, long long rows, Obj obj, T k, int slice) {
  constexpr int VEC = Num<T>::VEC, NT = STREAM_THREADS, U = STREAM_UNROLL;
  __shared__ Table<T, NT / 32, CLUSTER> table;
  const unsigned rank = CLUSTER ? cluster_rank() : 0, blocks = CLUSTER ? cluster_size() : 1;
  const long long step = gridDim.x / blocks;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, begin = (int)rank * slice;
  const bool reports = rank == 0 && warp == 0;
  pdl_wait();
  if constexpr (CLUSTER) cluster_sync();
  int half = 0;
  long long r = blockIdx.x / blocks;
  typename Obj::Meta next{};
  if (r < rows) next = obj.meta(r);
  for (; r < rows; r += step) {
    const typename Obj::Meta now = next;
    if (r + step < rows) next = obj.meta(r + step);
    if (!now.live()) {
      if (rank == 0 && threadIdx.x == 0) obj.skip(r);
      continue;
    }
    Span<T> row(x.row(r), x.v);
    row.clip(begin, begin + slice);
    T xl = (T)0;
    typename std::conditional<Obj::TARGETS, EntriesPart, int>::type part{};
    if constexpr (Obj::TARGETS) {
      if (reports) part = obj.prepare(r, x.row(r), x.v, lane, nullptr, nullptr, nullptr);
    } else {
      if (reports && lane == 0) xl = x.row(r)[clamp_label(now.label, x.v)];
    }
    Stat<T> a;
    for (int i = begin + (int)threadIdx.x; i * VEC < row.hi; i += NT * U) {
      T y[U * VEC];
#pragma unroll
      for (int u = 0; u < U; ++u) row.load(i + NT * u, y + u * VEC);
      const Stat<T> b = exponentials<T, U * VEC>(y, k);
      const T m = b.m > a.m ? b.m : a.m;
      a.s = a.s * Num<T>::exps(a.m - base(m), k) + b.s * Num<T>::exps(base(b.m) - base(m), k);
      a.m = m;
    }
    table.write(half, join<32>(a, k), rank, blocks);
    if constexpr (CLUSTER) cluster_sync();
    else __syncthreads();
    if (reports) {
      const Stat<T> st = table.read(half, blocks, k);
      if (lane == 0) {
        if constexpr (Obj::TARGETS) obj.report(r, now, part, st);
        else obj.report(r, now, xl, st);
      }
    }
    half ^= 1;
  }
  if constexpr (CLUSTER) cluster_sync();
}

// ---- gradients from the statistics of an earlier pass ----

// A block computes a piece of NT * U vectors of a row.
constexpr int GRAD_THREADS = 256;
template <typename T, int U>
__global__ void __launch_bounds__(GRAD_THREADS) k_grad(View<T> x, long long rows, GivenRow<T> obj, T k, Out<T> g, int pieces) {
  constexpr int VEC = Num<T>::VEC, NT = GRAD_THREADS;
  pdl_wait();
  const int lane = threadIdx.x % 32;
  // Piece p of row r; then gridDim.x pieces on.
  const long long step_r = gridDim.x / (unsigned)pieces;
  const int step_p = (int)(gridDim.x % (unsigned)pieces);
  long long r = blockIdx.x / (unsigned)pieces;
  for (int p = (int)(blockIdx.x % (unsigned)pieces); r < rows; r += step_r + (p + step_p >= pieces), p = p + step_p >= pieces ? p + step_p - pieces : p + step_p) {
    const int first = p * NT * U;
    const typename GivenRow<T>::Meta q = obj.meta(r);
    Span<T> row(x.row(r), x.v);
    row.clip(first, first + NT * U);
    const int warp0 = first + (int)threadIdx.x / 32 * 32 * U;  // this warp's vectors: warp0 + lane + 32 * u
    T y[U * VEC];
    const bool inside = warp0 * VEC >= row.lo && (warp0 + 32 * U) * VEC <= row.hi;
    if (q.live()) {
      const T* from = row.base + (long long)(warp0 + lane) * VEC;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (inside) {
          const typename Num<T>::Vec t = *reinterpret_cast<const typename Num<T>::Vec*>(from + u * 32 * VEC);
          memcpy(y + u * VEC, &t, 16);
        } else {
          row.load(warp0 + lane + 32 * u, y + u * VEC);
        }
      }
    }
    const T f = -q.c / q.s;
    const int l = (int)clamp_label(q.label, x.v) + row.off;
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int c = 0; c < VEC; ++c) y[u * VEC + c] = q.live() ? Num<T>::exps(y[u * VEC + c] - q.m, k) * f : (T)0;
      if (q.live() && warp0 + lane + 32 * u == l / VEC) {
#pragma unroll
        for (int c = 0; c < VEC; ++c)
          if (l % VEC == c) y[u * VEC + c] += q.c;
      }
    }
    if (inside) store<T, 32, U, true>(g.row(r), row, warp0, lane, y);
    else store<T, 32, U, false>(g.row(r), row, warp0, lane, y);
  }
}

// ---- rows longer than a cluster holds ----

// A block per row reads it twice.
constexpr int LONG_THREADS = 1024;
template <typename T, class Obj> __global__ void __launch_bounds__(LONG_THREADS) k_two_pass(View<T> x, long long rows, Obj obj, T k, Out<T> g) {
  constexpr int VEC = Num<T>::VEC, NT = LONG_THREADS, U = 2;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Table<T, NT / 32, false> table;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  T *tq = (T*)dyn, *tx = nullptr;
  int* ti = nullptr;
  if constexpr (Obj::TARGETS) {
    tx = tq + obj.k;
    ti = (int*)(tx + obj.k);
  }
  pdl_wait();
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const typename Obj::Meta now = obj.meta(r);
    const Span<T> row(x.row(r), x.v);
    // Whole warps take each turn.
    const int vectors = (row.hi + VEC - 1) / VEC, turns = (vectors + NT - 1) / NT;
    T xl = (T)0, c = (T)0, f = (T)0;
    int l = -1;
    Stat<T> a, st;
    typename std::conditional<Obj::TARGETS, EntriesPart, int>::type part{};
    bool zero = !now.live();
    if (now.live()) {
      if constexpr (Obj::TARGETS) {
        if (warp == 0) {
          part = obj.prepare(r, x.row(r), x.v, lane, ti, tq, tx);
          if (lane == 0) table.extra[0].m = part.some ? (T)1 : (T)0;
        }
      } else {
        l = (int)clamp_label(now.label, x.v);
        xl = x.row(r)[l];
        l += row.off;
      }
      for (int i = (int)threadIdx.x; i < vectors; i += NT * U) {
        T y[U * VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) row.load(i + NT * u, y + u * VEC);
        const Stat<T> b = exponentials<T, U * VEC>(y, k);
        const T m = b.m > a.m ? b.m : a.m;
        a.s = a.s * Num<T>::exps(a.m - base(m), k) + b.s * Num<T>::exps(base(b.m) - base(m), k);
        a.m = m;
      }
      table.write(0, join<32>(a, k), 0, 1);
      __syncthreads();
      st = table.read(0, 1, k);
      if constexpr (Obj::TARGETS) {
        zero = table.extra[0].m == (T)0;
        c = now.w * obj.wt;
        f = c / st.s;
      } else {
        c = obj.coef(now, xl, st);
        f = -c / st.s;
      }
    }
    for (int e = 0; e < turns; ++e) {
      const int i = (int)threadIdx.x + NT * e;
      T y[VEC];
      if (!zero) row.load(i, y);
#pragma unroll
      for (int q = 0; q < VEC; ++q) {
        y[q] = zero ? (T)0 : Num<T>::exps(y[q] - st.m, k) * f;
        if (!zero && i * VEC + q == l) y[q] += c;
      }
      store<T, 32, 1, false>(g.row(r), row, i - lane, lane, y);
    }
    __syncthreads();
    if constexpr (Obj::TARGETS) {
      if (!zero) {
        T* gr = g.row(r);
        for (long long i = threadIdx.x; i < obj.k; i += NT) {
          T sum = (T)0;
          bool leads = true;
          for (long long o = 0; o < obj.k; ++o) {
            if (ti[o] != ti[i]) continue;
            leads = leads && o >= i;
            sum += tq[o];
          }
          if (leads) gr[ti[i]] = c * (Num<T>::exps(tx[i] - st.m, k) / st.s - sum);
        }
      }
      if (warp == 0 && lane == 0) {
        if (now.live()) obj.report(r, now, part, st);
        else obj.skip(r);
      }
      __syncthreads();
    } else if (threadIdx.x == 0) {
      if (now.live()) obj.report(r, now, xl, st);
      else obj.skip(r);
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
constexpr int PAIR_THREADS = 256;
template <typename T>
__global__ void __launch_bounds__(PAIR_THREADS) k_pairs(const T* __restrict__ token_logp, const T* __restrict__ weight, const T* __restrict__ ref,
                                                        long long pairs, long long length, double beta, double smoothing, T* terms, T* coef, T* margins,
                                                        T* logp) {
  pdl_wait();
  __shared__ double sh[PAIR_THREADS / 32];
  const long long k = blockIdx.x;
  double total[2];
  for (int side = 0; side < 2; ++side) {
    const long long at = (k + side * pairs) * length;
    double v = 0;
    for (long long t = threadIdx.x; t < length; t += PAIR_THREADS)
      if (weight[at + t] != (T)0) v += (double)weight[at + t] * (double)token_logp[at + t];
    total[side] = block_sum(v, sh);
  }
  if (threadIdx.x) return;
  const double h = beta * ((total[0] - (double)ref[k]) - (total[1] - (double)ref[pairs + k]));
  const double e = exp(-fabs(h)), up = h >= 0 ? 1 / (1 + e) : e / (1 + e), down = h >= 0 ? e / (1 + e) : 1 / (1 + e);
  const double tail = log1p(e);
  // -log sigma(h) = tail + max(-h, 0), -log sigma(-h) = tail + max(h, 0)
  terms[k] = h != h ? (T)h : (T)((1 - smoothing) * (tail + (h < 0 ? -h : 0)) + smoothing * (tail + (h > 0 ? h : 0)));
  const double dh = beta * (smoothing * up - (1 - smoothing) * down) / (double)pairs;
  coef[k] = (T)dh;
  coef[pairs + k] = (T)-dh;
  if (margins) margins[k] = (T)h;
  if (logp) {
    logp[k] = (T)total[0];
    logp[pairs + k] = (T)total[1];
  }
}

// ---- host side ----

template <typename T> View<T> view(const RowView& x) { return {(const T*)x.data, make_fdiv((unsigned long long)std::max<long long>(x.inner, 1)), x.vocab, x.so, x.si}; }
template <typename T> Out<T> out(const RowView& x, const RowOut& g) { return {(T*)g.data, make_fdiv((unsigned long long)std::max<long long>(x.inner, 1)), g.so, g.si}; }

// Vectors of the longest row, from the alignments that rows have.
template <typename T> long long most_vectors(const RowView& x, const void* data, long long so, long long si) {
  constexpr long long VEC = Num<T>::VEC;
  const bool aligned = (uintptr_t)data % 16 == 0 && (x.outer <= 1 || so % VEC == 0) && (x.inner <= 1 || si % VEC == 0);
  return (x.vocab + (aligned ? 0 : VEC - 1) + VEC - 1) / VEC;
}
template <typename T> long long most_vectors(const RowView& x) { return most_vectors<T>(x, x.data, x.so, x.si); }

int sm_count() {
  static int n = [] {
    int dev = 0, v = 0;
    cudaGetDevice(&dev);
    return cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && v > 0 ? v : 148;
  }();
  return n;
}

// Clusters of `cluster` blocks of a kernel that the GPU holds at once (1: blocks), looked up once per kernel,
// shared memory and cluster. Also lets the kernel have that much dynamic shared memory, on each device.
template <typename K> long long resident(K* kernel, int threads, size_t smem, unsigned cluster) {
  static std::mutex mu;
  static std::map<std::tuple<const void*, size_t, unsigned, int>, long long> known;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  const auto key = std::make_tuple((const void*)kernel, smem, cluster, dev);
  const auto it = known.find(key);
  if (it != known.end()) return it->second;
  if (smem > 48 * 1024) cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  int n = 0;
  if (cluster > 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster * 1024);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, (const void*)kernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = sm_count() / (int)cluster;
    }
  } else {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, (const void*)kernel, threads, smem) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = 1;
    }
    n *= sm_count();
  }
  return known[key] = n;
}

long long pieces_of(long long n, long long of) { return (n + of - 1) / of; }

// Blocks per row: the fewest that hold it (`most` vectors each), and more when the rows alone would
// leave SMs without work, down to `least` vectors each.
unsigned split(long long rows, long long vectors, long long most, long long least) {
  unsigned c = 1;
  while (c < MAX_CLUSTER && pieces_of(vectors, c) > most) c *= 2;
  while (c < MAX_CLUSTER && rows * c * 2 <= sm_count() && vectors / (2 * c) >= least) c *= 2;
  return c;
}

template <typename T, int G, int E, class Obj, bool GRAD> cudaError_t go_group(const RowView& x, const Obj& obj, T k, const RowOut& g, size_t smem, cudaStream_t s) {
  auto* kernel = k_group<T, G, E, Obj, GRAD>;
  const long long warps = pieces_of(x.rows(), 32 / G), blocks = std::min(pieces_of(warps, GROUP_THREADS / 32), resident(kernel, GROUP_THREADS, smem, 1));
  return launch(kernel, dim3((unsigned)blocks), dim3(GROUP_THREADS), smem, 1, s, view<T>(x), x.rows(), obj, k, out<T>(x, g));
}

// Rows of at most 256 vectors, by the fewest lanes that hold one in at most 8 vectors each.
constexpr long long GROUP_VECTORS = 256;
template <typename T, class Obj, bool GRAD> cudaError_t group(const RowView& x, const Obj& obj, T k, const RowOut& g, cudaStream_t s) {
  const long long v = most_vectors<T>(x);
  if constexpr (Obj::TARGETS) {
    const int e = v <= 32 ? 1 : v <= 64 ? 2 : v <= 128 ? 4 : 8;
    const size_t smem = (GROUP_THREADS / 32) * ((e * 32 * Num<T>::VEC + 2 * (size_t)obj.k) * sizeof(T) + (size_t)obj.k * sizeof(int));
    switch (e) {
      case 1: return go_group<T, 32, 1, Obj, GRAD>(x, obj, k, g, smem, s);
      case 2: return go_group<T, 32, 2, Obj, GRAD>(x, obj, k, g, smem, s);
      case 4: return go_group<T, 32, 4, Obj, GRAD>(x, obj, k, g, smem, s);
      default: return go_group<T, 32, 8, Obj, GRAD>(x, obj, k, g, smem, s);
    }
  } else {
    if (v <= 8) return go_group<T, 8, 1, Obj, GRAD>(x, obj, k, g, 0, s);
    if (v <= 16) return go_group<T, 8, 2, Obj, GRAD>(x, obj, k, g, 0, s);
    if (v <= 32) return go_group<T, 8, 4, Obj, GRAD>(x, obj, k, g, 0, s);
    if (v <= 64) return go_group<T, 8, 8, Obj, GRAD>(x, obj, k, g, 0, s);
    if (v <= 128) return go_group<T, 16, 8, Obj, GRAD>(x, obj, k, g, 0, s);
    return go_group<T, 32, 8, Obj, GRAD>(x, obj, k, g, 0, s);
  }
}

template <class Obj> size_t target_bytes(const Obj& obj, size_t es, int halves) {
  if constexpr (Obj::TARGETS) return halves * (size_t)obj.k * (2 * es + sizeof(int));
  else return 0;
}

template <typename T, int NT, int E, int STAGES, bool CLUSTER, class Obj>
cudaError_t go_block(const RowView& x, const Obj& obj, T k, const RowOut& g, long long slice, unsigned cluster, cudaStream_t s) {
  auto* kernel = k_block<T, NT, E, STAGES, CLUSTER, Obj>;
  const size_t smem = (size_t)STAGES * (NT / 32) * (32 * E + 1) * 16 + target_bytes(obj, sizeof(T), 2);
  const long long clusters = std::min(x.rows(), resident(kernel, NT, smem, cluster));
  return launch(kernel, dim3((unsigned)(clusters * cluster)), dim3(NT), smem, cluster, s, view<T>(x), x.rows(), obj, k, out<T>(x, g), (int)slice,
                (int)pieces_of(slice, NT));
}

// Rows with a gradient that no group holds.
constexpr long long BLOCK_VECTORS = 4096;
template <typename T, class Obj> cudaError_t block(const RowView& x, const Obj& obj, T k, const RowOut& g, cudaStream_t s) {
  const long long v = most_vectors<T>(x, g.data, g.so, g.si);
  const unsigned c = split(x.rows(), v, BLOCK_VECTORS, 512);
  const long long slice = pieces_of(pieces_of(v, c), 32) * 32;
  if (slice > BLOCK_VECTORS) {
    auto* kernel = k_two_pass<T, Obj>;
    const size_t smem = target_bytes(obj, sizeof(T), 1);
    return launch(kernel, dim3((unsigned)std::min(x.rows(), resident(kernel, LONG_THREADS, smem, 1))), dim3(LONG_THREADS), smem, 1, s, view<T>(x), x.rows(),
                  obj, k, out<T>(x, g));
  }
  if (c == 1) {
    if (slice <= 512) return go_block<T, 64, 8, 2, false>(x, obj, k, g, slice, 1, s);
    if (slice <= 1024) return go_block<T, 64, 16, 1, false>(x, obj, k, g, slice, 1, s);
    if (slice <= 2048) return go_block<T, 128, 16, 1, false>(x, obj, k, g, slice, 1, s);
    return go_block<T, 256, 16, 1, false>(x, obj, k, g, slice, 1, s);
  }
  if (slice <= 1024) return go_block<T, 64, 16, 1, true>(x, obj, k, g, slice, c, s);
  if (slice <= 2048) return go_block<T, 128, 16, 1, true>(x, obj, k, g, slice, c, s);
  return go_block<T, 256, 16, 1, true>(x, obj, k, g, slice, c, s);
}

template <typename T, class Obj> cudaError_t stream(const RowView& x, const Obj& obj, T k, cudaStream_t s) {
  const long long v = most_vectors<T>(x);
  const unsigned c = split(x.rows(), v, v, 512);
  const long long slice = pieces_of(v, c);
  if (c == 1) {
    auto* kernel = k_stream<T, false, Obj>;
    return launch(kernel, dim3((unsigned)std::min(x.rows(), resident(kernel, STREAM_THREADS, 0, 1))), dim3(STREAM_THREADS), 0, 1, s, view<T>(x), x.rows(), obj,
                  k, (int)slice);
  }
  auto* kernel = k_stream<T, true, Obj>;
  return launch(kernel, dim3((unsigned)(std::min(x.rows(), resident(kernel, STREAM_THREADS, 0, c)) * c)), dim3(STREAM_THREADS), 0, c, s, view<T>(x), x.rows(),
                obj, k, (int)slice);
}

// An objective's rows, with or without their gradient. scale: what the logits are multiplied by.
template <typename T, class Obj> cudaError_t rows_of(const RowView& x, const Obj& obj, double scale, const RowOut& g, cudaStream_t s) {
  if (x.rows() == 0) return cudaSuccess;
  const T k = Num<T>::factor(scale);
  if (most_vectors<T>(x) <= GROUP_VECTORS) return g.data ? group<T, Obj, true>(x, obj, k, g, s) : group<T, Obj, false>(x, obj, k, g, s);
  return g.data ? block<T, Obj>(x, obj, k, g, s) : stream<T, Obj>(x, obj, k, s);
}

template <typename T> cudaError_t given_grad(const RowView& x, const GivenRow<T>& obj, const RowOut& g, cudaStream_t s) {
  if (x.rows() == 0) return cudaSuccess;
  const T k = Num<T>::factor(1.0);
  const long long v = most_vectors<T>(x);
  if (v <= GROUP_VECTORS) return group<T, GivenRow<T>, true>(x, obj, k, g, s);
  auto go = [&](auto* kernel, int u) {
    const long long pieces = pieces_of(v, GRAD_THREADS * u);
    return launch(kernel, dim3((unsigned)std::min(x.rows() * pieces, resident(kernel, GRAD_THREADS, 0, 1))), dim3(GRAD_THREADS), 0, 1, s, view<T>(x), x.rows(),
                  obj, k, out<T>(x, g), (int)pieces);
  };
  return v <= 2 * GRAD_THREADS ? go(k_grad<T, 2>, 2) : go(k_grad<T, 4>, 4);
}

template <typename T> cudaError_t sum_terms(const void* terms, long long n, void* loss, double scale, cudaStream_t s) {
  return launch(k_sum_terms<T>, 1, 1024, 0, 1, s, (const T*)terms, n, (T*)loss, scale);
}

}  // namespace

template <typename T> cudaError_t Objectives<T>::log_prob(const RowView& x, const int32_t* labels, void* logp, void* stats, cudaStream_t s) {
  const LogProbRow<T> obj{labels, (T*)logp, (T*)stats};
  if (x.rows() == 0) return cudaSuccess;
  const T k = Num<T>::factor(1.0);
  return most_vectors<T>(x) <= GROUP_VECTORS ? group<T, LogProbRow<T>, false>(x, obj, k, RowOut{}, s) : stream<T, LogProbRow<T>>(x, obj, k, s);
}

template <typename T>
cudaError_t Objectives<T>::log_prob_grad(const RowView& x, const int32_t* labels, const void* stats, const void* dlogp, const RowOut& grad, cudaStream_t s) {
  return given_grad<T>(x, GivenRow<T>{labels, (const T*)stats, (const T*)dlogp, nullptr, nullptr, FDiv{}}, grad, s);
}

template <typename T>
cudaError_t Objectives<T>::policy(const RowView& x, const int32_t* labels, const PolicyArgs& a, void* loss, void* terms, void* logp, const RowOut& g, cudaStream_t s) {
  const PolicyRow<T> obj{labels,
                         (const T*)a.old_logp,
                         (const T*)a.ref_logp,
                         (const T*)a.advantage,
                         (const T*)a.weight,
                         (T)(1 - a.clip_low),
                         (T)(1 + a.clip_high),
                         (T)a.kl,
                         (T*)terms,
                         (T*)logp};
  const cudaError_t e = rows_of<T>(x, obj, 1.0, g, s);
  if (e != cudaSuccess || !loss) return e;
  return sum_terms<T>(terms, x.rows(), loss, 1.0, s);
}

template <typename T>
cudaError_t Objectives<T>::preference(const RowView& x, const int32_t* labels, const PreferenceArgs& a, void* loss, void* margins, void* logp, const RowOut& g,
                         void* workspace, cudaStream_t s) {
  const long long rows = x.rows(), pairs = x.outer / 2;
  T* token = (T*)workspace;     // rows
  T* stats = token + rows;      // 2 * rows
  T* terms = stats + 2 * rows;  // pairs
  T* coef = terms + pairs;      // 2 * pairs
  cudaError_t e = log_prob(x, labels, token, stats, s);
  if (e == cudaSuccess && pairs > 0)
    e = launch(k_pairs<T>, dim3((unsigned)pairs), dim3(PAIR_THREADS), 0, 1, s, (const T*)token, (const T*)a.weight, (const T*)a.ref_logp, pairs, x.inner,
               a.beta, a.smoothing, terms, coef, (T*)margins, (T*)logp);
  if (e == cudaSuccess && loss) e = sum_terms<T>(terms, pairs, loss, pairs ? 1.0 / (double)pairs : 0.0, s);
  if (e == cudaSuccess && g.data)
    e = given_grad<T>(x, GivenRow<T>{labels, stats, nullptr, coef, (const T*)a.weight, make_fdiv((unsigned long long)std::max<long long>(x.inner, 1))}, g, s);
  return e;
}

template <typename T> cudaError_t Objectives<T>::distill(const RowView& x, const DistillArgs& a, void* loss, void* terms, const RowOut& g, cudaStream_t s) {
  const double inverse = 1 / a.temperature;
  const DistillRow<T> obj{a.index, (const T*)a.teacher, (const T*)a.weight, a.k, inverse, Num<T>::factor(inverse), (T)a.temperature, (T*)terms};
  const cudaError_t e = rows_of<T>(x, obj, inverse, g, s);
  if (e != cudaSuccess || !loss) return e;
  return sum_terms<T>(terms, x.rows(), loss, 1.0, s);
}

}  // namespace rgc
