// Kernels of the objectives over logits (objectives.cuh has the formulas).
//
// All of them are bound by memory: a row is V logits to read and, with a gradient, V values to write, against
// one exponential per logit (two with a gradient).
//  - k_group, k_group_targets (rows up to 640 vectors of 16 bytes): groups of 8, 16 or 32 lanes hold rows in registers
//    from the loads to the gradient;
//  - k_rows (longer rows, with a gradient): a block, or a cluster of blocks, reads a row twice, the second time from
//    the L2;
//  - k_stream (longer rows, no gradient): a running maximum and sum, nothing is held;
//  - k_grad (longer rows): gradients whose coefficients need more than their row (token_log_prob_grad, preferences).
// Of the rate of a plain copy (6563 GB/s) they reach, in floats: k_stream 90 % (8192 logits), 96 % (32000), 98 % (50257), k_grad 96 %,
// k_rows 87 % (4096, 8192), 91 % (16384), 87 % (32000), 82 % (50257, 131072), k_group with 1000 logits 81 % (policy), 74 % (without
// a gradient), 92 % (with statistics given), and 61 % at 96.
//
// Numbers. Row statistics are held in the logits' type. For float, exp(x - m) is computed as
// 2^((x - m) * log2 e) with the hardware's ex2: the difference and the product are rounded, 2 u |x - m|
// relatively, and ex2 is within 2 ulp; against expf that halves the instructions per logit. What does not average out over
// a row's logits is taken out, since it is the same in every row of a batch and a loss is a sum of terms of both
// signs: log2 e has two parts (as one float it is 1.3e-8 too small), ex2's mean error is put into its argument, and
// the factors between parts of a row are a polynomial's (Num<float>::share). Row sums of normal logits, deviation 1 and 2.5, are then
// off by 3e-9 to 9e-9 on average (8192 to 50257 logits; 7e-9 at 96; without all that -2e-8 to -9e-8), with a spread of 4.5e-8. Two
// floats to an instruction, this costs 1 to 4 % of the time of k_stream, 2 % of that of k_group and k_rows (5 % more by single
// ones in k_stream; from 131072 logits on k_rows gains 4 %, k_grad up to 10 %). For double it is a polynomial (Num<double>).
// What a row reports (a log-probability, a term of a loss) is computed from its statistics in double by one lane, and sums
// over rows are double. A gradient's coefficient is computed in the logits' type, but a clipped ratio next to its bound in
// double too, so that the gradient is that of the term.
// Everything is summed in a fixed order: the same call gives the same bits. What a row's bits depend on beside its values is how it
// is split over lanes and blocks: by the vocabulary, the row count, the alignment of base and strides to 16 bytes, the SM count and
// what the call computes (k_rows with a gradient, k_stream without).
#pragma once
#include "objectives.cuh"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <map>
#include <mutex>
#include <tuple>
#include <type_traits>
#include <utility>

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
  // scale * log2 e in two parts. hi is rounded towards 0 and lo is above 0, so both products have d's sign (-inf stays -inf).
  struct Scale {
    float hi, lo;
    float far;  // the difference at which the exponent is -126
  };
  // ex2 is on average 5.0e-8 too small (measured: 5.0e-8 to 5.2e-8 for t from -1 to -120, 2e-8 to 3e-8 above -1): t is raised
  // by log2(1 + 5.0e-8), before it is rounded. At d = 0 the result is 1.
  static constexpr float RAISE = 7.2e-8f;
  static __device__ __forceinline__ float ex2(float t) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
    return r;
  }
  // exp(d * scale)
  static __device__ __forceinline__ float exps(float d, Scale k) { return ex2(__fmaf_rn(d, k.hi, __fmaf_rn(d, k.lo, RAISE))); }
  // The same for differences of about 1, without lo and with half the raise: on average off by 2.5e-8 at most on either side of -1, and 1
  // at d = 0. For a thread's running sum, at each of its turns over a row (by share instead 16 x 511 x 50257 takes 1.4 % longer).
  static __device__ __forceinline__ float near(float d, Scale k) { return ex2(__fmaf_rn(d, k.hi, RAISE / 2)); }
  // The same for d <= 0 without ex2's share, for the factors between parts of a row (each element meets several): 2^t with
  // t = n + f, n whole and |f| <= 1/2; 2^f by the polynomial of degree 6 that equals it at 7 Chebyshev nodes (with Horner's
  // roundings off by 1.4 u at most, 1e-9 on average). At d = 0 it is 1; below 2^-126 it is 2^-126.
  static __device__ __forceinline__ float share(float d, Scale k) {
    constexpr float C[7] = {0x1.0p+0f, 0x1.62e43p-1f, 0x1.ebfbep-3f, 0x1.c6aeccp-5f, 0x1.3b2a1cp-7f, 0x1.5f48cp-10f, 0x1.444p-13f};
    constexpr float WHOLE = 12582912.0f;  // 3 * 2^22: adding it rounds to a whole number, in the low bits
    d = fmaxf(d, k.far);
    const float w = __fmaf_rn(d, k.hi, WHOLE), f = __fmaf_rn(d, k.lo, __fmaf_rn(d, k.hi, WHOLE - w));
    float r = C[6];
#pragma unroll
    for (int i = 5; i >= 0; --i) r = __fmaf_rn(r, f, C[i]);
    return r * __int_as_float((__float_as_int(w) + 127) << 23);
  }
  // Two floats to an instruction: three additions and products for two logits' exponentials and one for their sum.
  using Two = unsigned long long;
  static __device__ __forceinline__ Two two(float a, float b) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
  }
  static __device__ __forceinline__ void split(Two t, float* a, float* b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(t)); }
  static __device__ __forceinline__ Two add(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
  }
  static __device__ __forceinline__ Two mul(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
  }
  static __device__ __forceinline__ Two fma(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
  }
  // x[i] = exps(x[i] - b, k)
  template <int N> static __device__ __forceinline__ void exps_of(float* x, float b, Scale k) {
    const Two minus = two(-b, -b), hi = two(k.hi, k.hi), lo = two(k.lo, k.lo), raise = two(RAISE, RAISE);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const Two d = add(two(x[i], x[i + 1]), minus);
      float t0, t1;
      split(fma(d, hi, fma(d, lo, raise)), &t0, &t1);
      x[i] = ex2(t0);
      x[i + 1] = ex2(t1);
    }
  }
  // Two chains, of the even and the odd elements: half the rounding of one long chain, and half its latency.
  template <int N> static __device__ __forceinline__ float sum(const float* x) {
    Two s = two(x[0], x[1]);
#pragma unroll
    for (int i = 2; i < N; i += 2) s = add(s, two(x[i], x[i + 1]));
    float s0, s1;
    split(s, &s0, &s1);
    return s0 + s1;
  }
  template <int N> static __device__ __forceinline__ void times(float* x, float f) {
    const Two both = two(f, f);
#pragma unroll
    for (int i = 0; i < N; i += 2) split(mul(two(x[i], x[i + 1]), both), &x[i], &x[i + 1]);
  }
  static __device__ __forceinline__ float ex(float v) { return expf(v); }
  static __device__ __forceinline__ float exm1(float v) { return expm1f(v); }
  static __device__ __forceinline__ float ln(float v) { return logf(v); }
  static __device__ __forceinline__ float most(float a, float b) { return fmaxf(a, b); }  // a NaN gives the other
  static Scale factor(double scale) {
    const double k = scale * 1.4426950408889634074;
    float hi = (float)k;
    if ((double)hi >= k) hi = std::nextafter(hi, 0.0f);
    return {hi, (float)(k - (double)hi), -126.0f / hi};
  }
};
template <> struct Num<double> {
  static constexpr int VEC = 2;
  using Vec = double2;
  // exp(d * scale) for d <= 0: 2^t with t = d * scale * log2 e = n + f, n whole and |f| <= 1/2; 2^f by the polynomial of
  // degree 11 that equals it at 12 Chebyshev nodes (off by 2.0e-17 relatively with its coefficients as doubles; 1.2 u with
  // Horner's roundings).
  // Below 2^-1022 it is 0. (7 x 129 x 10007 without gradient: 28.6 us, with exp() 32.6. The power of two put in by integer
  // operations, 14 instead of 17 double ones: 8192 x 8192 in 190 instead of 165 us, so not those alone bound it.)
  struct Scale {
    double k;
  };
  static __device__ __forceinline__ double exps(double d, Scale k) {
    constexpr double C[12] = {0x1.0000000000000p+0,  0x1.62e42fefa39efp-1,  0x1.ebfbdff82c5aep-3,  0x1.c6b08d704a0c6p-5,
                              0x1.3b2ab6fb9f1a5p-7,  0x1.5d87fe78a3f9cp-10, 0x1.430913112c61bp-13, 0x1.ffcbfc6da6ed1p-17,
                              0x1.62bfc2c86d700p-20, 0x1.b524ebd13a55fp-24, 0x1.e6228acd1c6e5p-28, 0x1.e9ec1fcb69a7fp-32};
    constexpr double WHOLE = 6755399441055744.0;  // 3 * 2^51: adding it rounds to a whole number, in the low bits
    const double t = d * k.k, w = t + WHOLE, f = t - (w - WHOLE);
    double r = C[11];
#pragma unroll
    for (int i = 10; i >= 0; --i) r = __fma_rn(r, f, C[i]);
    // Beyond 2^1024, which only wrong statistics of a caller's give, it is infinity; NaN stays NaN in r.
    const double two_n = __hiloint2double(__double2hiint(t) >= 0x40900000 ? 0x7ff00000 : (__double2loint(w) + 1023) << 20, 0);
    return t < -1022.0 ? 0.0 : r * two_n;
  }
  static __device__ __forceinline__ double near(double d, Scale k) { return exps(d, k); }
  static __device__ __forceinline__ double share(double d, Scale k) { return exps(d, k); }
  template <int N> static __device__ __forceinline__ void exps_of(double* x, double b, Scale k) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = exps(x[i] - b, k);
  }
  template <int N> static __device__ __forceinline__ double sum(const double* x) {
    double s0 = 0, s1 = 0;
#pragma unroll
    for (int i = 0; i < N; i += 2) s0 += x[i], s1 += x[i + 1];
    return s0 + s1;
  }
  template <int N> static __device__ __forceinline__ void times(double* x, double f) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= f;
  }
  static __device__ __forceinline__ double ex(double v) { return exp(v); }
  static __device__ __forceinline__ double exm1(double v) { return expm1(v); }
  static __device__ __forceinline__ double ln(double v) { return log(v); }
  static __device__ __forceinline__ double most(double a, double b) { return fmax(a, b); }
  static Scale factor(double scale) { return {scale * 1.4426950408889634074}; }
};

template <typename T> using Scale = typename Num<T>::Scale;

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

template <int G, bool LONG = false, typename T> __device__ __forceinline__ Stat<T> join(Stat<T> a, Scale<T> k) {
  T m = a.m;
#pragma unroll
  for (int d = G / 2; d; d >>= 1) {
    m = Num<T>::most(m, __shfl_xor_sync(~0u, m, d));
  }
  const T d = a.m - base(m);
  T s = a.s * (LONG ? Num<T>::share(d, k) : Num<T>::exps(d, k));
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
      __stcs(reinterpret_cast<typename Num<T>::Vec*>(at), t);
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

// The same for the groups of a warp, each with a row of its own (and an alignment of its own); with many vectors a lane
// the registers do not hold the shifted ones too.
template <typename T, int G, int E> __device__ __forceinline__ void store_group(T* row, const Span<T>& x, int lane, const T* y) {
  constexpr int VEC = Num<T>::VEC;
  if constexpr (G == 32 && E <= 8) {
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
  const T* weight;  // null: every row counts
  T *logp, *stats;
  struct Meta {
    int label;
    T w;
    __device__ __forceinline__ bool live() const { return w != (T)0; }
  };
  __device__ __forceinline__ Meta meta(long long r) const { return {labels[r], weight ? weight[r] : (T)1}; }
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
  double low, high, kl;  // the ratio's bounds 1 - clip_low and 1 + clip_high: as floats, 1.28 and 0.8 are 2e-8 off in every clipped token
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
    m.ref = kl != 0 ? ref_logp[r] : (T)0;
    return m;
  }
  __device__ void skip(long long r) const {
    terms[r] = (T)0;
    if (logp) logp[r] = (T)0;
  }
  __device__ __forceinline__ double log_prob(T xl, Stat<T> st) const { return ((double)xl - (double)st.m) - log((double)st.s); }
  // Whether the bound counts in the ratio's place. A NaN ratio or advantage is not clipped: the term and the gradient are NaN.
  template <typename F> __device__ __forceinline__ bool clipped(F ratio, F a) const { return a >= 0 ? ratio > (F)high : a < 0 && ratio < (F)low; }
  __device__ __forceinline__ T coef(const Meta& m, T xl, Stat<T> st) const {
    const T ls = Num<T>::ln(st.s), lp = (xl - st.m) - ls, d = lp - m.old, ratio = Num<T>::ex(d);
    bool bound = clipped(ratio, m.a);
    if constexpr (sizeof(T) == 4) {
      // The term's ratio is the double one, and the gradient is the term's: a ratio so close to its bound that the roundings decide is
      // computed again. With u = 2^-24: x - m, lp and d are off by u of themselves, the logarithm and the exponential by 2 u and
      // 4 u, the bound by u; |x - m| is at most |lp| + log s.
      const T edge = (T)(m.a >= (T)0 ? high : low);
      if (fabsf(ratio - edge) <= edge * 0x1p-22f * (fabsf(lp) + ls + fabsf(d) + 2.0f)) bound = clipped(exp(log_prob(xl, st) - (double)m.old), (double)m.a);
    }
    T c = bound ? (T)0 : -(ratio * m.a);
    if (kl != 0) c -= (T)kl * Num<T>::exm1(m.ref - lp);
    return m.w * c;
  }
  __device__ __forceinline__ void report(long long r, const Meta& m, T xl, Stat<T> st) const {
    const double lp = log_prob(xl, st), ratio = exp(lp - (double)m.old), a = m.a;
    double term = clipped(ratio, a) ? -((a >= 0 ? high : low) * a) : -(ratio * a);
    if (kl != 0) {
      const double d = (double)m.ref - lp;
      term += kl * (expm1(d) - d);
    }
    terms[r] = (T)((double)m.w * term);
    if (logp) logp[r] = (T)lp;
  }
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
      const T c = by_sequence[quotient((unsigned)r, length)];
      q.c = q.live() ? c * q.w : (T)0;
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

// Some of a row's teacher entries: the largest teacher logit m and the largest logit `from` of the row at them, with
// e = exp((t - m) / T) the sum s of e and the sum a of e ((t - m) - (x - from)). Without any entry s is 0.
template <typename T> struct EntriesPart {
  T m = -(T)INFINITY, from = (T)0;
  double s = 0, a = 0;
};

// The distillation: a row's targets are its teacher entries. With q = e / s the term is
// sum q (log q - log p_i) = a / (s T) - log s + (row's m - from) / T + log(row's s).
// Taken relative to `from`, the logits' own size does not count in the difference of the two sums.
template <typename T> struct DistillRow {
  static constexpr bool TARGETS = true, GIVEN = false;
  const int32_t* index;
  const T *teacher, *weight;
  long long k;
  double inverse;  // 1 / T
  Scale<T> tk;     // of 1 / T
  T wt;            // T
  T* terms;
  struct Meta {
    T w;
    __device__ __forceinline__ bool live() const { return w != (T)0; }
  };
  using Part = EntriesPart<T>;
  __device__ __forceinline__ Meta meta(long long r) const { return {weight[r]}; }
  __device__ void skip(long long r) const { terms[r] = (T)0; }
  struct Entry {
    T t, x;
    int at;
    __device__ __forceinline__ Part part() const {
      Part p;
      if (t != neg_inf<T>()) p.m = t, p.from = x, p.s = 1;
      return p;
    }
  };
  // Entry i of row r, without its logit: that is element `at` of the row.
  __device__ __forceinline__ Entry entry(long long r, long long v, int i) const {
    Entry e;
    e.t = teacher[r * k + i];
    e.at = (int)clamp_label(index[r * k + i], v);
    return e;
  }
  // What the n parts of WIDTH neighbouring lanes are together, each lane's own every WIDTH-th of them from `first` on.
  template <int WIDTH, typename F> __device__ __forceinline__ Part join(int first, int n, F part) const {
    T top = neg_inf<T>(), far = neg_inf<T>();
    for (int i = first; i < n; i += WIDTH) {
      const Part p = part(i);
      if (p.s == 0) continue;
      top = Num<T>::most(top, p.m);
      far = Num<T>::most(far, p.from);
    }
#pragma unroll
    for (int d = WIDTH / 2; d; d >>= 1) {
      top = Num<T>::most(top, __shfl_xor_sync(~0u, top, d));
      far = Num<T>::most(far, __shfl_xor_sync(~0u, far, d));
    }
    if (!(far > neg_inf<T>() && far < -neg_inf<T>())) far = (T)0;
    Part all{top, far, 0, 0};
    for (int i = first; i < n; i += WIDTH) {
      const Part p = part(i);
      const T f = Num<T>::exps(p.m - base(top), tk);
      if (p.s != p.s || (p.s != 0 && f != (T)0)) {  // a NaN stays, whatever its weight
        all.s += (double)f * p.s;
        all.a += (double)f * (p.a + p.s * (((double)p.m - (double)top) - ((double)p.from - (double)far)));
      }
    }
#pragma unroll
    for (int d = WIDTH / 2; d; d >>= 1) {
      all.s += __shfl_xor_sync(~0u, all.s, d);
      all.a += __shfl_xor_sync(~0u, all.a, d);
    }
    return all;
  }
  // By a warp: the largest of the k teacher logits at t and the sum of their exponentials.
  __device__ __forceinline__ Stat<T> total(const T* t) const {
    const int lane = (int)threadIdx.x % 32;
    Stat<T> st;
    for (int i = lane; i < (int)k; i += 32) st.m = Num<T>::most(st.m, t[i]);
#pragma unroll
    for (int d = 16; d; d >>= 1) st.m = Num<T>::most(st.m, __shfl_xor_sync(~0u, st.m, d));
    for (int i = lane; i < (int)k; i += 32) st.s += Num<T>::exps(t[i] - base(st.m), tk);
#pragma unroll
    for (int d = 16; d; d >>= 1) st.s += __shfl_xor_sync(~0u, st.s, d);
    return st;
  }
  // q of an entry with teacher logit t, of all entries' part.
  __device__ __forceinline__ T share(T t, T m, T inverse_s) const { return Num<T>::exps(t - base(m), tk) * inverse_s; }
  __device__ __forceinline__ void report(long long r, const Meta& m, const Part& p, Stat<T> st) const {
    const double term = (p.a / p.s + ((double)st.m - (double)p.from)) * inverse + log((double)st.s / p.s);
    terms[r] = p.s != 0 ? (T)((double)m.w * (double)wt * (double)wt * term) : (T)0;
  }
};

// A row's entries in shared memory: the indices (whole vectors of four, what is not an entry negative), the teacher's
// logits, the row's.
template <typename T> struct Kept {
  int* at;
  T *t, *x;
  __device__ __forceinline__ Kept(unsigned char* p, int slots) {  // slots: a multiple of four
    at = (int*)p;
    t = (T*)(p + slots * sizeof(int));
    x = t + slots;
  }
  // Whether entry i of k is the first with its index; *sum: share(t) of all of them, in order.
  template <typename F> __device__ __forceinline__ bool leads(int i, int k, T* sum, F share) const {
    const int mine = at[i];
    *sum = (T)0;
#pragma unroll 4
    for (int o = 0; o < k; o += 4) {
      const int4 z = *reinterpret_cast<const int4*>(at + o);
      if (z.x != mine && z.y != mine && z.z != mine && z.w != mine) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if ((c == 0 ? z.x : c == 1 ? z.y : c == 2 ? z.z : z.w) != mine) continue;
        if (o + c < i) return false;
        *sum += share(t[o + c]);
      }
    }
    return true;
  }
};
template <typename T> size_t kept_bytes(size_t slots) { return slots * (sizeof(int) + 2 * sizeof(T)); }

__device__ __forceinline__ unsigned smem_addr(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
// One number from global to shared memory, there for this thread after copies_wait().
template <typename T> __device__ __forceinline__ void copy_ahead(T* to, const T* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_addr(to)), "l"(from), "n"((int)sizeof(T)) : "memory");
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ---- short rows: a group of G lanes per row ----

constexpr int GROUP_THREADS = 256;

// The maximum of a thread's N logits, their exponentials in place and the sum of these.
template <typename T, int N> __device__ __forceinline__ Stat<T> exponentials(T* x, Scale<T> k) {
  Stat<T> a;
#pragma unroll
  for (int i = 0; i < N; ++i) a.m = Num<T>::most(x[i], a.m);
  Num<T>::template exps_of<N>(x, base(a.m), k);
  a.s = Num<T>::template sum<N>(x);
  return a;
}

// The same for N more logits of a thread's running maximum and sum: relative to the maximum of both, so one of the two sums
// needs no factor. (8192 x 8192 doubles 165 us, 180 with two sums joined.)
template <typename T, int N> __device__ __forceinline__ void extend(Stat<T>& a, T* x, Scale<T> k) {
  T m = a.m;
#pragma unroll
  for (int i = 0; i < N; ++i) m = Num<T>::most(x[i], m);
  const T b = base(m);
  Num<T>::template exps_of<N>(x, b, k);
  a.s = a.s * Num<T>::near(a.m - b, k) + Num<T>::template sum<N>(x);
  a.m = m;
}

// A warp computes B times 32 / G rows together (G lanes each, E vectors a lane): all loads first, then the sums, then what
// the rows need once, a lane per row, then the gradients. The label's element is stored a second time by
// its row's lane, so no lane looks for it.
// What a row needs once is some 400 instructions: with a lane of every group doing it per row, 131072 x 96 took 62 us.
template <typename T, int G, int E, int B, class Obj, bool GRAD>
__global__ void __launch_bounds__(GROUP_THREADS, B == 1 && E <= 12 ? 3 : 2) k_group(const View<T> x, const long long rows, const Obj obj, const Scale<T> k, const Out<T> g) {
  constexpr int VEC = Num<T>::VEC, R = 32 / G, ROWS = B * R;
  static_assert(ROWS <= 32, "a lane per row");
  pdl_wait();
  const int lane = threadIdx.x % 32, in_group = lane % G, group = lane / G;
  const long long warps = (long long)gridDim.x * (GROUP_THREADS / 32);
  for (long long w = (long long)blockIdx.x * (GROUP_THREADS / 32) + threadIdx.x / 32; w * ROWS < rows; w += warps) {
    const long long row0 = w * ROWS, mine = row0 + lane;
    const bool in = lane < ROWS && mine < rows;
    typename Obj::Meta meta{};
    if (in) meta = obj.meta(mine);
    const bool live = in && meta.live();
    const unsigned lives = __ballot_sync(~0u, live);
    const T xl = live ? x.row(mine)[clamp_label(meta.label, x.v)] : (T)0;
    T y[B][E * VEC], most[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int at = b * R + group;
      if (lives >> at & 1) {
        const Span<T> row(x.row(row0 + at), x.v);
#pragma unroll
        for (int e = 0; e < E; ++e) row.load(in_group + G * e, y[b] + e * VEC);
      } else {
#pragma unroll
        for (int q = 0; q < E * VEC; ++q) y[b][q] = neg_inf<T>();
      }
    }
    Stat<T> st;
    if constexpr (Obj::GIVEN) {
      st = {meta.m, meta.s};
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const T m = __shfl_sync(~0u, st.m, (b * R + group) % 32);
        Num<T>::template exps_of<E * VEC>(y[b], m, k);
      }
    } else {
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const Stat<T> own = exponentials<T, E * VEC>(y[b], k);
        most[b] = own.m;
        const Stat<T> all = join<G>(own, k);
        const T m = __shfl_sync(~0u, all.m, lane % R * G), s = __shfl_sync(~0u, all.s, lane % R * G);
        if (lane / R == b) st = {m, s};
      }
    }
    T c = (T)0, scale = (T)0;
    if (live) {
      c = obj.coef(meta, xl, st);
      scale = -c / st.s;
    }
    if constexpr (GRAD) {
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const int at = (b * R + group) % 32;
        const T sc = __shfl_sync(~0u, scale, at);
        T f = sc;
        if constexpr (!Obj::GIVEN) {
          const T m = __shfl_sync(~0u, st.m, at);
          f = most[b] == neg_inf<T>() ? (T)0 * sc : Num<T>::exps(most[b] - base(m), k) * sc;
        }
        const bool zero = !(lives >> at & 1), have = row0 + b * R + group < rows;
#pragma unroll
        for (int q = 0; q < E * VEC; ++q) y[b][q] = zero ? (T)0 : y[b][q] * f;
        const long long r = have ? row0 + b * R + group : row0;
        store_group<T, G, E>(g.row(r), Span<T>(x.row(r), have ? x.v : 0), in_group, y[b]);
      }
      __syncwarp();  // the label's element over what its group has stored
      if (live) g.row(mine)[clamp_label(meta.label, x.v)] = c + Num<T>::exps(xl - st.m, k) * scale;
    }
    if (in) {
      if (live) obj.report(mine, meta, xl, st);
      else obj.skip(mine);
    }
  }
}

// The same for the distillation: 32 / ROWS lanes take a row's entries, one after the other, and what they come to goes to the
// row's lane. The entries reach shared memory while the logits are under way. (With a lane for every entry and 5 steps
// between lanes for each row, 131072 x 96 with 32 entries took 142 us.)
// The gradients at the entries are written a second time, over what the row's lanes have stored; the first entry of an
// index writes its element, with the probabilities of all of that index.
template <typename T, int G, int E, int B, class Obj, bool GRAD>
__global__ void __launch_bounds__(GROUP_THREADS, E * B <= 8 ? 4 : E * B <= 10 ? 3 : 2) k_group_targets(const View<T> x, const long long rows, const Obj obj, const Scale<T> k, const Out<T> g, const int slots) {
  constexpr int VEC = Num<T>::VEC, R = 32 / G, ROWS = B * R, TEAM = 32 / ROWS;
  static_assert(ROWS <= 32, "a lane per row");
  extern __shared__ __align__(16) unsigned char dyn[];
  pdl_wait();
  const int lane = threadIdx.x % 32, in_group = lane % G, group = lane / G, mate = lane % TEAM, of = lane / TEAM, entries = (int)obj.k;
  // Of this lane's row of entries.
  const Kept<T> kept(dyn + (threadIdx.x / 32 * ROWS + of) * slots * (sizeof(int) + 2 * sizeof(T)), slots);
  if (mate == 0) *reinterpret_cast<int4*>(kept.at + (entries - 1) / 4 * 4) = make_int4(-1, -1, -1, -1);  // behind the entries
  __syncwarp();
  const long long warps = (long long)gridDim.x * (GROUP_THREADS / 32);
  for (long long w = (long long)blockIdx.x * (GROUP_THREADS / 32) + threadIdx.x / 32; w * ROWS < rows; w += warps) {
    const long long row0 = w * ROWS, mine = row0 + lane;
    const bool in = lane < ROWS && mine < rows;
    typename Obj::Meta meta{};
    if (in) meta = obj.meta(mine);
    const bool live = in && meta.live();
    const unsigned lives = __ballot_sync(~0u, live);
    const bool fed = lives >> of & 1;
    for (int i = mate; fed && i < entries; i += TEAM) {
      copy_ahead(kept.t + i, obj.teacher + (row0 + of) * obj.k + i);
      copy_ahead(kept.at + i, obj.index + (row0 + of) * obj.k + i);
    }
    T y[B][E * VEC], most[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int at = b * R + group;
      if (lives >> at & 1) {
        const Span<T> row(x.row(row0 + at), x.v);
#pragma unroll
        for (int e = 0; e < E; ++e) row.load(in_group + G * e, y[b] + e * VEC);
      } else {
#pragma unroll
        for (int q = 0; q < E * VEC; ++q) y[b][q] = neg_inf<T>();
      }
    }
    copies_wait();
    for (int i = mate; fed && i < entries; i += TEAM) {
      const int at = (int)clamp_label(kept.at[i], x.v);
      kept.at[i] = at;
      copy_ahead(kept.x + i, x.row(row0 + of) + at);
    }
    Stat<T> st;
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const Stat<T> own = exponentials<T, E * VEC>(y[b], k);
      most[b] = own.m;
      const Stat<T> all = join<G>(own, k);
      const T m = __shfl_sync(~0u, all.m, lane % R * G), s = __shfl_sync(~0u, all.s, lane % R * G);
      if (lane / R == b) st = {m, s};
    }
    copies_wait();
    typename Obj::Part part = obj.template join<TEAM>(mate, fed ? entries : 0, [&](int i) { return typename Obj::Entry{kept.t[i], kept.x[i], 0}.part(); });
    const int src = lane % ROWS * TEAM;
    part = {__shfl_sync(~0u, part.m, src), __shfl_sync(~0u, part.from, src), __shfl_sync(~0u, part.s, src), __shfl_sync(~0u, part.a, src)};
    const bool some = live && part.s != 0;
    if constexpr (GRAD) {
      const unsigned somes = __ballot_sync(~0u, some);
      const T c = some ? meta.w * obj.wt : (T)0, scale = some ? c / st.s : (T)0, inverse_s = (T)1 / (T)part.s;
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const int at = (b * R + group) % 32;
        const T sc = __shfl_sync(~0u, scale, at), m = __shfl_sync(~0u, st.m, at);
        const T f = most[b] == neg_inf<T>() ? (T)0 * sc : Num<T>::exps(most[b] - base(m), k) * sc;
        const bool zero = !(somes >> at & 1), have = row0 + b * R + group < rows;
#pragma unroll
        for (int q = 0; q < E * VEC; ++q) y[b][q] = zero ? (T)0 : y[b][q] * f;
        const long long r = have ? row0 + b * R + group : row0;
        store_group<T, G, E>(g.row(r), Span<T>(x.row(r), have ? x.v : 0), in_group, y[b]);
      }
      __syncwarp();
      const T sc = __shfl_sync(~0u, scale, of), cj = __shfl_sync(~0u, c, of), m = __shfl_sync(~0u, st.m, of);
      const T top = __shfl_sync(~0u, part.m, of), inv = __shfl_sync(~0u, inverse_s, of);
      if (somes >> of & 1) {
        T* gr = g.row(row0 + of);
        for (int i = mate; i < entries; i += TEAM) {
          T sum;
          if (kept.leads(i, entries, &sum, [&](T z) { return obj.share(z, top, inv); })) gr[kept.at[i]] = Num<T>::exps(kept.x[i] - m, k) * sc - cj * sum;
        }
      }
    }
    __syncwarp();  // the kept entries are read before the next rows'
    if (in) {
      if (live) obj.report(mine, meta, part, st);
      else obj.skip(mine);
    }
  }
}

// ---- longer rows: a block, or a cluster of blocks, per row ----

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
// The cluster's barrier, by whole warps.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Without ordering: for warps that have written nothing another block reads.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
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
constexpr int MAX_CLUSTER = 8;

// (m, s) of every warp of a block, or of every block of a cluster, in turn in one of two halves.
template <typename T, int N> struct Table {
  Pair<T> slot[2][N];
  // By a warp: what the first n of N slots hold together.
  __device__ __forceinline__ Stat<T> read(int half, int n, Scale<T> k) const {
    Stat<T> a;
    const int lane = threadIdx.x % 32;
    if (lane < n) a = {slot[half][lane].m, slot[half][lane].s};
    return join<32, true>(a, k);
  }
};
template <typename T> __device__ __forceinline__ Pair<T> pair(Stat<T> a) { return {a.m, a.s}; }

constexpr int MANY_ENTRIES = 64;  // 4096 x 50257: 338 us with 64, a barrier a row (65) 349

// A row's entries, if the objective has any, by the threads of a block: entry threadIdx.x of the first NT is loaded before the
// row's logits, and its own logit after the first of them, when the index is there.
template <typename T, int NT, class Obj, bool TARGETS = Obj::TARGETS> struct Entries {
  __device__ __forceinline__ Entries(const Obj&, long long, const T*, long long, bool) {}
  __device__ __forceinline__ void gather() {}
  static __device__ __forceinline__ int slots(const Obj&) { return 0; }
};
template <typename T, int NT, class Obj> struct Entries<T, NT, Obj, true> {
  const Obj& obj;
  const long long r, v;
  const T* x;
  const bool on;
  typename Obj::Entry first{neg_inf<T>(), (T)0, -1};
  __device__ __forceinline__ Entries(const Obj& o, long long row, const T* logits, long long vocab, bool live) : obj(o), r(row), v(vocab), x(logits), on(live) {
    if (on && (int)threadIdx.x < (int)obj.k) first = obj.entry(r, v, (int)threadIdx.x);
  }
  __device__ __forceinline__ void gather() {
    if (on && (int)threadIdx.x < (int)obj.k) first.x = x[first.at];
  }
  static __device__ __forceinline__ int slots(const Obj& obj) { return ((int)obj.k + 3) / 4 * 4; }
  // Leaves the entries in `kept`. Whether this thread has any that is not absent.
  __device__ __forceinline__ bool keep(const Kept<T>& kept) {
    bool some = false;
    for (int i = (int)threadIdx.x; i < slots(obj); i += NT) {
      typename Obj::Entry n{neg_inf<T>(), (T)0, -1};
      if (i < NT) {
        n = first;
      } else if (i < (int)obj.k) {
        n = obj.entry(r, v, i);
        n.x = x[n.at];
      }
      kept.at[i] = n.at;
      kept.t[i] = n.t;
      kept.x[i] = n.x;
      some = some || n.t != neg_inf<T>();
    }
    return some;
  }
};
// By a warp: what the kept entries are together.
template <typename T, class Obj> __device__ __forceinline__ typename Obj::Part together(const Obj& obj, const Kept<T>& kept) {
  return obj.template join<32>((int)threadIdx.x % 32, (int)obj.k, [&](int i) { return typename Obj::Entry{kept.t[i], kept.x[i], 0}.part(); });
}

// ---- longer rows without a gradient ----

// Sixteen logits a thread at a time. (8192 x 8192 doubles: 153 us, with eight 165.)
template <typename T> constexpr int STREAM_UNROLL = 16 / Num<T>::VEC;

// A block, or a cluster of blocks, per row: a running maximum and sum per thread.
template <typename T, int NT, bool CLUSTER, class Obj>
__global__ void __launch_bounds__(NT) k_stream(View<T> x, long long rows, Obj obj, Scale<T> k, int slice) {
  constexpr int VEC = Num<T>::VEC, U = STREAM_UNROLL<T>;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Table<T, NT / 32> table;
  __shared__ Table<T, CLUSTER ? MAX_CLUSTER : 1> shares;
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
    Entries<T, NT, Obj> entries(obj, r, x.row(r), x.v, rank == 0);
    if constexpr (!Obj::TARGETS) {
      if (reports && lane == 0) xl = x.row(r)[clamp_label(now.label, x.v)];
    }
    Stat<T> a;
    for (int i = begin + (int)threadIdx.x; i * VEC < row.hi; i += NT * U) {
      T y[U * VEC];
#pragma unroll
      for (int u = 0; u < U; ++u) row.load(i + NT * u, y + u * VEC);
      if (i < begin + NT * U) entries.gather();
      extend<T, U * VEC>(a, y, k);
    }
    const Kept<T> kept(dyn + half * Entries<T, NT, Obj>::slots(obj) * (sizeof(int) + 2 * sizeof(T)), Entries<T, NT, Obj>::slots(obj));
    if constexpr (Obj::TARGETS) {
      if (rank == 0) {
        if ((begin + (int)threadIdx.x) * VEC >= row.hi) entries.gather();  // no logits for this thread
        entries.keep(kept);
      }
    }
    const Stat<T> of_warp = join<32, true>(a, k);
    if (lane == 0) table.slot[half][warp] = pair(of_warp);
    __syncthreads();
    if constexpr (CLUSTER) {
      if (warp == 0) {
        const Stat<T> st = table.read(half, NT / 32, k);
        if (lane == 0) put_remote(&shares.slot[half][rank], 0u, pair(st));
        cluster_arrive();
      } else {
        cluster_arrive_relaxed();
      }
      cluster_wait();
    }
    if (reports) {
      const Stat<T> st = CLUSTER ? shares.read(half, (int)blocks, k) : table.read(half, NT / 32, k);
      if constexpr (Obj::TARGETS) {
        const auto part = together(obj, kept);
        if (lane == 0) obj.report(r, now, part, st);
      } else {
        if (lane == 0) obj.report(r, now, xl, st);
      }
    }
    half ^= 1;
  }
  if constexpr (CLUSTER) cluster_sync();
}

// ---- gradients from the statistics of an earlier pass ----

// A warp computes a piece of 64 vectors of a row at a time. Many warps with two vectors a lane under way: with four, 32 instead
// of 48 warps fit an SM, and 8192 x 8192 took 100 instead of 83 us.
constexpr int GRAD_THREADS = 256, GRAD_UNROLL = 2, GRAD_VECTORS = 32 * GRAD_UNROLL;
template <typename T>
__global__ void __launch_bounds__(GRAD_THREADS, 6) k_grad(View<T> x, long long rows, GivenRow<T> obj, Scale<T> k, Out<T> g, int pieces) {
  constexpr int VEC = Num<T>::VEC, U = GRAD_UNROLL;
  pdl_wait();
  const int lane = threadIdx.x % 32;
  // Piece p of row r; then as many pieces on as there are warps.
  const unsigned warps = gridDim.x * (GRAD_THREADS / 32), warp = blockIdx.x * (GRAD_THREADS / 32) + threadIdx.x / 32;
  const long long step_r = warps / (unsigned)pieces;
  const int step_p = (int)(warps % (unsigned)pieces);
  long long r = warp / (unsigned)pieces;
  for (int p = (int)(warp % (unsigned)pieces); r < rows; r += step_r + (p + step_p >= pieces), p = p + step_p >= pieces ? p + step_p - pieces : p + step_p) {
    const int warp0 = p * GRAD_VECTORS;  // this warp's vectors: warp0 + lane + 32 * u
    const typename GivenRow<T>::Meta q = obj.meta(r);
    Span<T> row(x.row(r), x.v);
    row.clip(warp0, warp0 + GRAD_VECTORS);
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
    if (q.live()) {
      Num<T>::template exps_of<U * VEC>(y, q.m, k);
      Num<T>::template times<U * VEC>(y, -q.c / q.s);
    } else {
#pragma unroll
      for (int c = 0; c < U * VEC; ++c) y[c] = (T)0;
    }
    const int l = (int)clamp_label(q.label, x.v) + row.off;
#pragma unroll
    for (int u = 0; u < U; ++u) {
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

// ---- longer rows with a gradient ----

// A block of NT threads, or a cluster of such blocks (`slice` vectors each), per row: one pass for the statistics and
// one, backwards, that reads the logits again and writes the gradient. The second pass finds them in the L2 (or the
// L1), as long as the rows under way fit there, so memory sees each logit once.
// Measured against keeping a row on chip between the passes (in registers and shared memory, copies of the next row under
// way): 83 against 57 % of the copy rate at 50257 logits and 88 against 69 % at 32000, where a row needs a cluster of
// blocks and each waits for the slowest; 91 against 85 % at 16384, where one block holds it.
// 32 warps to an SM with 4 vectors a lane under way: with 48 and 2 16384 logits run at 75 %, with 24 and 8 at 84 %. Doubles:
// 24 warps and 4 vectors, 8192 x 8192 in 290 us; with 32 and 2 341. The first pass asks the L2 for nothing special: lines marked to
// be evicted last gain 2 of 183 us at 4096 x 32000, nothing at 16384 x 50257, and stay behind: two sums over the same 64 MB
// after the loss then take 53 us instead of 46.
template <typename T, int NT, bool CLUSTER, class Obj>
__global__ void __launch_bounds__(NT, (sizeof(T) == 4 ? 1024 : 768) / NT) k_rows(const View<T> x, const long long rows, const __grid_constant__ Obj obj, const Scale<T> k, const Out<T> g, const int slice) {
  constexpr int VEC = Num<T>::VEC, NW = NT / 32, U = 4;
  using Vec = typename Num<T>::Vec;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Table<T, NW> table;                          // of the block's warps
  __shared__ Table<T, CLUSTER ? MAX_CLUSTER : 1> shares;  // of the cluster's blocks
  const unsigned rank = CLUSTER ? cluster_rank() : 0, blocks = CLUSTER ? cluster_size() : 1;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, begin = (int)rank * slice, first = begin + warp * 32 * U;
  const int slots = Entries<T, NT, Obj>::slots(obj);
  pdl_wait();
  if constexpr (CLUSTER) cluster_sync();  // every block's shared memory is there before another writes to it
  const long long step = gridDim.x / blocks;
  long long r = blockIdx.x / blocks;
  int half = 0;
  for (; r < rows; r += step) {
    const typename Obj::Meta now = obj.meta(r);
    const T* xr = x.row(r);
    Span<T> row(xr, x.v);
    row.clip(begin, begin + slice);
    // Turn e: a warp's 32 * U adjacent vectors of the block's NT * U.
    const int turns = max(0, (row.hi + VEC - 1) / VEC - begin + NT * U - 1) / (NT * U);
    auto inside = [&](int i) { return i * VEC >= row.lo && (i + 32 * U) * VEC <= row.hi; };
    auto load = [&](int i, T* y, auto last) {  // vectors i + lane + 32 * u
      if (inside(i)) {
        const Vec* from = reinterpret_cast<const Vec*>(row.base) + (i + lane);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const Vec z = last ? __ldcs(from + 32 * u) : from[32 * u];
          memcpy(y + u * VEC, &z, 16);
        }
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) row.load(i + lane + 32 * u, y + u * VEC);
      }
    };
    // Two rows' entries: the block's other warps are in the next row when the entries' gradients are written.
    const Kept<T> kept(dyn + half * slots * (sizeof(int) + 2 * sizeof(T)), slots);
    T xl = (T)0, c = (T)0, f = (T)0, m_all = (T)0;
    int l = -1;
    Stat<T> st;
    bool zero = !now.live();
    if (now.live()) {
      Entries<T, NT, Obj> entries(obj, r, xr, x.v, true);
      if constexpr (!Obj::TARGETS) {
        l = (int)clamp_label(now.label, x.v);
        xl = xr[l];
        l += row.off;
      }
      Stat<T> a;
      for (int e = 0; e < turns; ++e) {
        if ((first + NT * U * e) * VEC >= row.hi) break;  // nothing of the row for this warp
        T y[U * VEC];
        load(first + NT * U * e, y, std::false_type{});
        if (e == 0) entries.gather();
        extend<T, U * VEC>(a, y, k);
      }
      bool some = false;
      if constexpr (Obj::TARGETS) {
        // Before any of the gradient is written, which may be in the logits' place.
        if (first * VEC >= row.hi) entries.gather();
        some = entries.keep(kept);
      }
      const Stat<T> of_warp = join<32, true>(a, k);
      if (lane == 0) table.slot[half][warp] = pair(of_warp);
      if constexpr (Obj::TARGETS) zero = !__syncthreads_or(some);  // a row without entries counts nothing
      else __syncthreads();
      st = table.read(half, NW, k);
      if constexpr (CLUSTER) {
        if (warp == 0 && lane < (int)blocks) put_remote(&shares.slot[half][rank], (unsigned)lane, pair(st));
        cluster_sync();
        st = shares.read(half, (int)blocks, k);
      }
      if constexpr (Obj::TARGETS) {
        c = zero ? (T)0 : now.w * obj.wt;
        f = zero ? (T)0 : c / st.s;
      } else {
        c = obj.coef(now, xl, st);
        f = -c / st.s;
      }
      m_all = zero ? (T)0 : st.m;
      half ^= 1;
    }
    T* gr = g.row(r);
    for (int e = turns - 1; e >= 0; --e) {
      const int i = first + NT * U * e;
      if (i * VEC >= row.hi) continue;
      T y[U * VEC];
      if (!zero) {
        load(i, y, std::true_type{});
      } else {
#pragma unroll
        for (int q = 0; q < U * VEC; ++q) y[q] = (T)0;
      }
      Num<T>::template exps_of<U * VEC>(y, m_all, k);
      Num<T>::template times<U * VEC>(y, f);
      if (!zero && l >= i * VEC && l < (i + 32 * U) * VEC) {
#pragma unroll
        for (int q = 0; q < U * VEC; ++q)
          if ((i + lane + 32 * (q / VEC)) * VEC + q % VEC == l) y[q] += c;
      }
      if (inside(i)) store<T, 32, U, true>(gr, row, i, lane, y);
      else store<T, 32, U, false>(gr, row, i, lane, y);
    }
    if constexpr (Obj::TARGETS) {
      // The entries' elements, over what has been stored. Few entries: every warp those among its own vectors, so no warp waits
      // for another and the next row's loads begin (a barrier here: 32000 logits with 32 entries 224 us). Many: a thread
      // each, after a barrier.
      if (!zero) {
        const bool many = obj.k > MANY_ENTRIES;
        if (many) __syncthreads();
        else __syncwarp();
        const Stat<T> all = obj.total(kept.t);
        const T inverse_s = (T)1 / all.s;
        const int lo = begin * VEC - row.off, hi = (begin + slice) * VEC - row.off;
        for (int i = many ? (int)threadIdx.x : lane; i < (int)obj.k; i += many ? NT : 32) {
          const int at = kept.at[i];
          T sum;
          if (at < lo || at >= hi || !(many || ((at + row.off) / VEC - begin) / (32 * U) % NW == warp)) continue;
          if (kept.leads(i, (int)obj.k, &sum, [&](T t) { return obj.share(t, all.m, inverse_s); })) gr[at] = Num<T>::exps(kept.x[i] - m_all, k) * f - c * sum;
        }
        if (rank == 0 && warp == NW - 1) {
          const auto part = together(obj, kept);
          if (lane == 0) obj.report(r, now, part, st);
        }
      } else if (rank == 0 && threadIdx.x == 0) {
        obj.skip(r);
      }
    } else if (rank == 0 && threadIdx.x == 0) {
      if (now.live()) obj.report(r, now, xl, st);
      else obj.skip(r);
    }
  }
  if constexpr (CLUSTER) cluster_sync();  // no block leaves while another may still write to it
}

// ---- sums in a fixed order ----

// sh: one of each of the block's warps.
__device__ double block_sum(double v, double* sh) {
  const int lane = threadIdx.x % 32;
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  __syncthreads();
  if (lane == 0) sh[threadIdx.x / 32] = v;
  __syncthreads();
  v = lane < (int)blockDim.x / 32 ? sh[lane] : 0.0;
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}

// A cluster's blocks, or one block, add up the terms: eight of a thread at a time, then threads, warps and blocks in order.
// (131072 terms: 6 us; sixteen at a time with a bound on each load 11.)
constexpr int SUM_THREADS = 512, SUM_CLUSTER = 8, SUM_AHEAD = 8;
template <typename T> __global__ void __launch_bounds__(SUM_THREADS) k_sum_terms(const T* __restrict__ terms, long long n, T* loss) {
  pdl_wait();
  __shared__ double sh[SUM_THREADS / 32];
  __shared__ Pair<double> of_block[SUM_CLUSTER];
  const unsigned rank = cluster_rank(), blocks = cluster_size();
  if (blocks > 1) cluster_sync();
  double v = 0;
  const long long step = (long long)blocks * SUM_THREADS;
  long long i = (long long)rank * SUM_THREADS + threadIdx.x;
  for (; i + (SUM_AHEAD - 1) * step < n; i += SUM_AHEAD * step) {
    T z[SUM_AHEAD];
#pragma unroll
    for (int q = 0; q < SUM_AHEAD; ++q) z[q] = terms[i + q * step];
    double part[4] = {0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < SUM_AHEAD; ++q) part[q % 4] += (double)z[q];
    v += (part[0] + part[1]) + (part[2] + part[3]);
  }
  for (; i < n; i += step) v += (double)terms[i];
  v = block_sum(v, sh);
  if (blocks > 1) {
    if (threadIdx.x == 0) put_remote(&of_block[rank], 0u, Pair<double>{v, 0.0});
    cluster_sync();
    if (rank != 0) return;
    v = 0;
    for (unsigned b = 0; b < blocks; ++b) v += of_block[b].m;
  }
  if (rank == 0 && threadIdx.x == 0) *loss = (T)v;
}

// The pairs, a warp for each (or a block, LONG), over the warps (blocks) of a cluster or one block: both sequences' sums, the margin, the
// loss term and the coefficients of the two sequences; then the mean of the terms.
constexpr int PAIR_THREADS = 512;
template <typename T, bool LONG>
__global__ void __launch_bounds__(PAIR_THREADS) k_pairs(const T* __restrict__ token_logp, const T* __restrict__ weight, const T* __restrict__ ref,
                                                        long long pairs, long long length, double beta, double smoothing, T* coef, T* margins, T* logp,
                                                        T* loss) {
  pdl_wait();
  __shared__ double sh[PAIR_THREADS / 32];
  __shared__ Pair<double> of_block[SUM_CLUSTER];
  const unsigned rank = cluster_rank(), blocks = cluster_size();
  if (blocks > 1) cluster_sync();
  constexpr int TEAM = LONG ? PAIR_THREADS : 32, TEAMS = PAIR_THREADS / TEAM;
  const int lane = threadIdx.x % TEAM;
  double terms = 0;
  for (long long k = (long long)rank * TEAMS + threadIdx.x / TEAM; k < pairs; k += (long long)blocks * TEAMS) {
    double total[2] = {0, 0};
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const long long at = (k + side * pairs) * length;
#pragma unroll 4
      for (long long t = lane; t < length; t += TEAM) {
        const T w = weight[at + t], lp = w != (T)0 ? token_logp[at + t] : (T)0;
        total[side] += (double)w * (double)lp;
      }
      if constexpr (LONG) {
        total[side] = block_sum(total[side], sh);
      } else {
        for (int d = 16; d; d >>= 1) total[side] += __shfl_xor_sync(~0u, total[side], d);
      }
    }
    const double h = beta * ((total[0] - (double)ref[k]) - (total[1] - (double)ref[pairs + k]));
    const double e = exp(-fabs(h)), up = h >= 0 ? 1 / (1 + e) : e / (1 + e), down = h >= 0 ? e / (1 + e) : 1 / (1 + e);
    const double tail = log1p(e);
    // -log sigma(h) = tail + max(-h, 0), -log sigma(-h) = tail + max(h, 0)
    // (A side without weight counts nothing, however far its answer is out of reach: 0 times infinity would be NaN.)
    const double chosen = smoothing < 1 ? (1 - smoothing) * (tail + (h < 0 ? -h : 0)) : 0, other = smoothing > 0 ? smoothing * (tail + (h > 0 ? h : 0)) : 0;
    if (lane == 0) terms += h != h ? h : chosen + other;
    const double dh = beta * (smoothing * up - (1 - smoothing) * down) / (double)pairs;
    if (lane < 2) {
      coef[k + lane * pairs] = (T)(lane ? -dh : dh);
      if (logp) logp[k + lane * pairs] = (T)total[lane];
      if (margins && lane == 0) margins[k] = (T)h;
    }
  }
  terms = block_sum(terms, sh);
  if (blocks > 1) {
    if (threadIdx.x == 0) put_remote(&of_block[rank], 0u, Pair<double>{terms, 0.0});
    cluster_sync();
    if (rank != 0) return;
    terms = 0;
    for (unsigned b = 0; b < blocks; ++b) terms += of_block[b].m;
  }
  if (loss && rank == 0 && threadIdx.x == 0) *loss = (T)(terms / (double)pairs);
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
// shared memory and cluster. Also lets the kernel have that much dynamic shared memory, on each device: never less than it has
// been given before, which another call may be counting on.
template <typename K> long long resident(K* kernel, int threads, size_t smem, unsigned cluster) {
  static std::mutex mu;
  static std::map<std::tuple<const void*, size_t, unsigned, int>, long long> known;
  static std::map<std::pair<const void*, int>, size_t> given;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  const auto key = std::make_tuple((const void*)kernel, smem, cluster, dev);
  const auto it = known.find(key);
  if (it != known.end()) return it->second;
  size_t& most = given[{(const void*)kernel, dev}];
  if (smem > 48 * 1024 && smem > most) {
    const cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) most = smem;
    else cudaGetLastError();  // the launch says so
  }
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

// Blocks per row: more than one when the rows alone would leave SMs without work, down to 512 vectors each. (48 rows of
// 50257: 11.5 us with 8 blocks each, 17.3 with 2.)
unsigned split(long long rows, long long vectors) {
  unsigned c = 1;
  while (c < MAX_CLUSTER && rows * c * 2 <= 4 * sm_count() && vectors / (2 * c) >= 512) c *= 2;
  return c;
}

template <typename K, typename... A> cudaError_t go_group(K* kernel, long long rows_per_warp, size_t smem, const RowView& x, cudaStream_t s, A... args) {
  const long long warps = pieces_of(x.rows(), rows_per_warp), blocks = std::min(pieces_of(warps, GROUP_THREADS / 32), resident(kernel, GROUP_THREADS, smem, 1));
  return launch(kernel, dim3((unsigned)blocks), dim3(GROUP_THREADS), smem, 1, s, args...);
}

// Rows of at most 640 vectors, by the fewest lanes that hold one; some 16 vectors a lane in all, or one row. (516 vectors,
// 65536 x 2064: 184 us here, 260 by a block per row; with 24 vectors a lane for 750, 65536 x 3000: 273 us here, 269.)
constexpr long long GROUP_VECTORS = 640;
template <typename T, class Obj, bool GRAD> cudaError_t group(const RowView& x, const Obj& obj, Scale<T> k, const RowOut& g, cudaStream_t s) {
  const long long v = most_vectors<T>(x);
  if constexpr (Obj::TARGETS) {
    // Slots for a row's entries: vectors of four, an odd number of them, so that rows begin in different banks.
    const int slots = ((int)pieces_of(obj.k, 4) | 1) * 4;
    auto go = [&](auto* kernel, int rows) {
      return go_group(kernel, rows, GROUP_THREADS / 32 * rows * kept_bytes<T>((size_t)slots), x, s, view<T>(x), x.rows(), obj, k, out<T>(x, g), slots);
    };
    // Up to 128 vectors: four vectors a lane, two rows to a group of lanes (8, 4 or 2 rows to a warp, whose entries 4, 8 or 16 lanes
    // take). 131072 x 96 with 8 entries: 44 us, 49 with one row to a group, 45 with four (32 entries: 110, 112 and 155), 147 with
    // one row to a warp; 32768 x 500 with 8: 42, 49 and 41. With more entries than 64 one row to a warp: at 65 that is slower (131072 x 96
    // 453 us, 294 by eight rows to a warp), at 128 faster (914 and 1184), and the entries of a double row leave room for two blocks.
    // Wider rows: the fewest vectors a lane that hold one.
    if (obj.k <= 64) {
      if (v <= 8) return go(k_group_targets<T, 8, 1, 2, Obj, GRAD>, 8);
      if (v <= 16) return go(k_group_targets<T, 8, 2, 2, Obj, GRAD>, 8);
      if (v <= 32) return go(k_group_targets<T, 8, 4, 2, Obj, GRAD>, 8);
      if (v <= 64) return go(k_group_targets<T, 16, 4, 2, Obj, GRAD>, 4);
      if (v <= 128) return go(k_group_targets<T, 32, 4, 2, Obj, GRAD>, 2);
    }
    if (v <= 32) return go(k_group_targets<T, 32, 1, 1, Obj, GRAD>, 1);
    if (v <= 128) return go(k_group_targets<T, 32, 4, 1, Obj, GRAD>, 1);
    if (v <= 256) return go(k_group_targets<T, 32, 8, 1, Obj, GRAD>, 1);
    if (v <= 320) return go(k_group_targets<T, 32, 10, 1, Obj, GRAD>, 1);
    if (v <= 512) return go(k_group_targets<T, 32, 16, 1, Obj, GRAD>, 1);
    return go(k_group_targets<T, 32, 20, 1, Obj, GRAD>, 1);
  } else {
    auto go = [&](auto* kernel, int rows) { return go_group(kernel, rows, 0, x, s, view<T>(x), x.rows(), obj, k, out<T>(x, g)); };
    if (v <= 8) return go(k_group<T, 8, 1, 8, Obj, GRAD>, 32);
    if (v <= 16) return go(k_group<T, 8, 2, 8, Obj, GRAD>, 32);
    if (v <= 24) return go(k_group<T, 8, 3, 5, Obj, GRAD>, 20);
    if (v <= 32) return go(k_group<T, 8, 4, 4, Obj, GRAD>, 16);
    if (v <= 64) return go(k_group<T, 16, 4, 4, Obj, GRAD>, 8);
    if (v <= 128) return go(k_group<T, 32, 4, 4, Obj, GRAD>, 4);
    if (v <= 192) return go(k_group<T, 32, 6, 3, Obj, GRAD>, 3);
    if (v <= 256) return go(k_group<T, 32, 8, 2, Obj, GRAD>, 2);
    if (v <= 320) return go(k_group<T, 32, 10, 1, Obj, GRAD>, 1);
    if (v <= 384) return go(k_group<T, 32, 12, 1, Obj, GRAD>, 1);
    if (v <= 512) return go(k_group<T, 32, 16, 1, Obj, GRAD>, 1);
    return go(k_group<T, 32, 20, 1, Obj, GRAD>, 1);
  }
}

template <typename T, class Obj> size_t target_bytes(const Obj& obj) {
  if constexpr (Obj::TARGETS) return 2 * kept_bytes<T>(((size_t)obj.k + 3) / 4 * 4);
  else return 0;
}

template <typename T, int NT, bool CLUSTER, class Obj>
cudaError_t go_rows(const RowView& x, const Obj& obj, Scale<T> k, const RowOut& g, long long slice, unsigned cluster, cudaStream_t s) {
  auto* kernel = k_rows<T, NT, CLUSTER, Obj>;
  const size_t smem = target_bytes<T>(obj);
  const long long clusters = std::min(x.rows(), resident(kernel, NT, smem, cluster));
  return launch(kernel, dim3((unsigned)(clusters * cluster)), dim3(NT), smem, cluster, s, view<T>(x), x.rows(), obj, k, out<T>(x, g), (int)slice);
}

constexpr long long L2_ROWS_BYTES = 80ll << 20;
// Rows with a gradient that no group holds.
template <typename T, class Obj> cudaError_t block(const RowView& x, const Obj& obj, Scale<T> k, const RowOut& g, cudaStream_t s) {
  const long long v = most_vectors<T>(x);
  unsigned c = split(x.rows(), v);
  // Rows under way at once that do not fit the L2 (its two halves hold copies of what the other half's SMs read):
  // fewer, each by a cluster. (4096 x 50257, 60 MB under way: 300 us, by clusters of two 385. 4096 x 65536: clusters
  // of two, 78 MB, 396 us, of four 409.)
  if (c == 1 && v * 16 * 2 * sm_count() > L2_ROWS_BYTES)
    for (c = 2; c < MAX_CLUSTER && v * 16 * 4 * sm_count() / c > L2_ROWS_BYTES; c *= 2) {
    }
  const long long slice = pieces_of(v, c);
  if (c > 1) return go_rows<T, 256, true>(x, obj, k, g, slice, c, s);
  // About four turns of a block over the row: 8192 floats (2048 vectors) at 78, 91, 84 and 65 % of the copy rate with 64, 128,
  // 256 and 512 threads, 16384 at 68, 78, 90 and 81 %, 4096 at 88, 84, 68 and 33 %.
  if (v <= 1448) return go_rows<T, 64, false>(x, obj, k, g, slice, 1, s);
  if (v <= 2896) return go_rows<T, 128, false>(x, obj, k, g, slice, 1, s);
  if (v <= 5792) return go_rows<T, 256, false>(x, obj, k, g, slice, 1, s);
  return go_rows<T, 512, false>(x, obj, k, g, slice, 1, s);
}

template <typename T, int NT, bool CLUSTER, class Obj>
cudaError_t go_stream(const RowView& x, const Obj& obj, Scale<T> k, long long slice, unsigned cluster, cudaStream_t s) {
  auto* kernel = k_stream<T, NT, CLUSTER, Obj>;
  const size_t smem = target_bytes<T>(obj);
  const long long clusters = std::min(x.rows(), resident(kernel, NT, smem, cluster));
  return launch(kernel, dim3((unsigned)(clusters * cluster)), dim3(NT), smem, cluster, s, view<T>(x), x.rows(), obj, k, (int)slice);
}

// Rows without a gradient that no group holds.
template <typename T, class Obj> cudaError_t stream(const RowView& x, const Obj& obj, Scale<T> k, cudaStream_t s) {
  const long long v = most_vectors<T>(x);
  const unsigned c = split(x.rows(), v);
  if (c > 1) return go_stream<T, 256, true>(x, obj, k, pieces_of(v, c), c, s);
  // Some three turns of a block over the row: 2800 floats (700 vectors, 64 threads) 121 us against 226 with 256; 5400 (1350) 62
  // and 60 with 64 and 128; 11000 (2750) 110 and 115 with 128 and 256; 32000 (8000) 325 and 301.
  if (v <= 1024 / 4 * STREAM_UNROLL<T>) return go_stream<T, 64, false>(x, obj, k, v, 1, s);
  if (v <= 2896 / 4 * STREAM_UNROLL<T>) return go_stream<T, 128, false>(x, obj, k, v, 1, s);
  return go_stream<T, 256, false>(x, obj, k, v, 1, s);
}

// An objective's rows, with or without their gradient. scale: what the logits are multiplied by.
template <typename T, class Obj> cudaError_t rows_of(const RowView& x, const Obj& obj, double scale, const RowOut& g, cudaStream_t s) {
  if (x.rows() == 0) return cudaSuccess;
  const Scale<T> k = Num<T>::factor(scale);
  if (most_vectors<T>(x) <= GROUP_VECTORS) return g.data ? group<T, Obj, true>(x, obj, k, g, s) : group<T, Obj, false>(x, obj, k, g, s);
  return g.data ? block<T, Obj>(x, obj, k, g, s) : stream<T, Obj>(x, obj, k, s);
}

template <typename T> cudaError_t given_grad(const RowView& x, const GivenRow<T>& obj, const RowOut& g, cudaStream_t s) {
  if (x.rows() == 0) return cudaSuccess;
  const Scale<T> k = Num<T>::factor(1.0);
  const long long v = most_vectors<T>(x);
  if (v <= GROUP_VECTORS) return group<T, GivenRow<T>, true>(x, obj, k, g, s);
  const long long pieces = pieces_of(v, GRAD_VECTORS), blocks = pieces_of(x.rows() * pieces, GRAD_THREADS / 32);
  return launch(k_grad<T>, dim3((unsigned)std::min(blocks, resident(k_grad<T>, GRAD_THREADS, 0, 1))), dim3(GRAD_THREADS), 0, 1, s, view<T>(x), x.rows(), obj, k,
                out<T>(x, g), (int)pieces);
}

template <typename T> cudaError_t sum_terms(const void* terms, long long n, void* loss, cudaStream_t s) {
  const unsigned blocks = n > SUM_AHEAD * SUM_THREADS ? SUM_CLUSTER : 1;
  return launch(k_sum_terms<T>, dim3(blocks), dim3(SUM_THREADS), 0, blocks, s, (const T*)terms, n, (T*)loss);
}

// weight: null, or rows with weight 0 are not read and give nothing.
template <typename T> cudaError_t log_prob_rows(const RowView& x, const int32_t* labels, const T* weight, T* logp, T* stats, cudaStream_t s) {
  const LogProbRow<T> obj{labels, weight, logp, stats};
  if (x.rows() == 0) return cudaSuccess;
  const Scale<T> k = Num<T>::factor(1.0);
  return most_vectors<T>(x) <= GROUP_VECTORS ? group<T, LogProbRow<T>, false>(x, obj, k, RowOut{}, s) : stream<T, LogProbRow<T>>(x, obj, k, s);
}

}  // namespace

template <typename T> cudaError_t Objectives<T>::log_prob(const RowView& x, const int32_t* labels, void* logp, void* stats, cudaStream_t s) {
  return log_prob_rows<T>(x, labels, nullptr, (T*)logp, (T*)stats, s);
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
                         1 - a.clip_low,
                         1 + a.clip_high,
                         a.kl,
                         (T*)terms,
                         (T*)logp};
  const cudaError_t e = rows_of<T>(x, obj, 1.0, g, s);
  if (e != cudaSuccess || !loss) return e;
  return sum_terms<T>(terms, x.rows(), loss, s);
}

template <typename T>
cudaError_t Objectives<T>::preference(const RowView& x, const int32_t* labels, const PreferenceArgs& a, void* loss, void* margins, void* logp, const RowOut& g,
                         void* workspace, cudaStream_t s) {
  const long long rows = x.rows(), pairs = x.outer / 2;
  T* token = (T*)workspace;    // rows
  T* stats = token + rows;     // 2 * rows
  T* coef = stats + 2 * rows;  // 2 * pairs
  const T* weight = (const T*)a.weight;
  cudaError_t e = log_prob_rows<T>(x, labels, weight, token, stats, s);
  if (e == cudaSuccess) {
    auto go = [&](auto* kernel, long long at_once) {
      return launch(kernel, dim3(pairs > at_once ? SUM_CLUSTER : 1), dim3(PAIR_THREADS), 0, pairs > at_once ? SUM_CLUSTER : 1, s, (const T*)token, weight,
                    (const T*)a.ref_logp, pairs, x.inner, a.beta, a.smoothing, coef, (T*)margins, (T*)logp, (T*)loss);
    };
    // A warp's loads under way hold 128 tokens of a sequence.
    e = x.inner > 256 ? go(k_pairs<T, true>, 1) : go(k_pairs<T, false>, PAIR_THREADS / 32);
  }
  if (e == cudaSuccess && g.data)
    e = given_grad<T>(x, GivenRow<T>{labels, stats, nullptr, coef, weight, make_fdiv((unsigned long long)std::max<long long>(x.inner, 1))}, g, s);
  return e;
}

template <typename T> cudaError_t Objectives<T>::distill(const RowView& x, const DistillArgs& a, void* loss, void* terms, const RowOut& g, cudaStream_t s) {
  const double inverse = 1 / a.temperature;
  const DistillRow<T> obj{a.index, (const T*)a.teacher, (const T*)a.weight, a.k, inverse, Num<T>::factor(inverse), (T)a.temperature, (T*)terms};
  const cudaError_t e = rows_of<T>(x, obj, inverse, g, s);
  if (e != cudaSuccess || !loss) return e;
  return sum_terms<T>(terms, x.rows(), loss, s);
}

}  // namespace rgc
