// Losses on the log-probability of ONE label per score row, with their gradient: the
// log-probabilities themselves, the clipped policy loss with a KL term and the preference loss on
// pairs of label sequences.  Score rows S [n, m] in fp32, bf16 or fp16 with any row stride.
//
//   x = S / tau,  M_i = max_j S_ij,  Z_i = sum_j exp(x_ij - M_i / tau)
//   l_i = (S_{i, y_i} - M_i) / tau - log Z_i             (0 for y_i = -1: the row carries nothing)
//   dL/dS_ij = c_i / tau ([j = y_i] - exp(x_ij - M_i / tau) / Z_i)      with c_i = dL/dl_i
//
// so every loss is one pass over the scores for (M, Z), a few scalars per row for c, and one pass
// that writes the gradient.  HBM-bound: about 8 operations per score against 4-8 bytes.
//
//   policy:      r = exp(l - old), d = ref - l,  L = scale sum_i w_i (-min(r A, clip(r) A) + kl (e^d - d - 1))
//                c_i = scale w_i (-A r [r A <= clip(r) A] + kl (1 - e^d)).  c_i needs its own row only: rows
//                that fit a workgroup's registers are read ONCE (policy_fused_kernel).
//   preference:  pi_q = sum or mean of l over the labelled rows of sequence q, z = beta ((pi_w - ref_w) -
//                (pi_l - ref_l)), L = scale sum_pairs -((1 - e) log sigma(z) + e log sigma(-z)).  c_i needs the
//                whole pair: the gradient pass reads the scores again.
//
// Precision: the exponentials are v_exp_f32 on fp32 differences, summed in fp32 per thread and in
// fp64 across threads; the per-row scalars (log Z, ratios, coefficients) are fp64, because the
// clipped loss jumps at its borders and e^d - d - 1 cancels for small d.  Losses are summed in fp64
// in a fixed order.  A 16-bit gradient is rounded once, when it is written.
//
// A row with label -1 or coefficient 0 gets a zero gradient without being read.  A label outside
// [-1, m) poisons its row (NaN loss and gradient).  -inf scores (masked candidates) have probability 0;
// a labelled row of nothing but -inf has no distribution and gives NaN, as does a NaN score.
#include <math.h>

#include <type_traits>

#include "common.h"

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Vec;  // 16 bytes of scores
template <>
struct Vec<float> {
  static constexpr int N = 4;
  typedef f32x4 type;
};
template <>
struct Vec<__bf16> {
  static constexpr int N = 8;
  typedef bf16x8 type;
};
template <>
struct Vec<_Float16> {
  static constexpr int N = 8;
  typedef f16x8 type;
};

template <typename T>
__device__ __forceinline__ void unpack(const u32x4& r, float (&f)[Vec<T>::N]) {
  const typename Vec<T>::type v = __builtin_bit_cast(typename Vec<T>::type, r);
#pragma unroll
  for (int e = 0; e < Vec<T>::N; ++e) f[e] = (float)v[e];
}
template <typename T>
__device__ __forceinline__ u32x4 pack(const float (&f)[Vec<T>::N]) {
  typename Vec<T>::type v;
#pragma unroll
  for (int e = 0; e < Vec<T>::N; ++e) v[e] = (T)f[e];  // round to nearest even, once
  return __builtin_bit_cast(u32x4, v);
}

// A row as its elements before the first 16-byte boundary (head), whole vectors, and the rest
// (tail): rows of any alignment are read with 16-byte loads and never outside themselves.
template <typename T>
struct Row {
  const T* p;
  int m, head, nvec;
  __device__ __forceinline__ Row(const T* row, int m_) : p(row), m(m_) {
    const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    head = min(m, (Vec<T>::N - off) & (Vec<T>::N - 1));
    nvec = (m - head) / Vec<T>::N;
  }
  __device__ __forceinline__ const u32x4* vecs() const { return reinterpret_cast<const u32x4*>(p + head); }
  // The edge element of thread t (head elements: threads 0 .. 7, tail elements: 8 .. 15), or -1.
  __device__ __forceinline__ int edge(int t) const {
    if (t < 8) return t < head ? t : -1;
    const int j = head + nvec * Vec<T>::N + (t - 8);
    return t < 16 && j < m ? j : -1;
  }
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// max over the workgroup, returned to every thread (NaN dropped: it comes back through the sum)
template <int NT>
__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  if (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v = fmaxf(v, red[w]);
  return v;
}

// sum over the workgroup in fp64 and a fixed order; only wave 0 gets the result
template <int NT>
__device__ __forceinline__ double block_sum_wave0(float v, double* red) {
  double s = (double)v;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if (NT == 64) return s;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return 0.0;
  s = red[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) s += red[w];
  return s;
}

// exponent scale: exp((x - M) / tau) = exp2((x - M) * k2)
struct Temp {
  float k2;
  double inv;  // 1 / tau
};
inline Temp temp_of(double tau) { return {(float)(1.4426950408889634 / tau), 1.0 / tau}; }

// The subtrahend of the exponentials: a row (or part of one) of nothing but -inf sums to 0
// instead of NaN, which its owner tells from an empty part of a row with finite scores.
__device__ __forceinline__ float safe_max(float mx) { return mx == -INFINITY ? 0.f : mx; }

// l = log-probability of the label from (M, Z)
template <typename T>
__device__ __forceinline__ double label_logp(const T* row, int m, int64_t y, float mx, double z, double inv_tau) {
  if (y < 0 || y >= m) return NAN;  // callers skip y = -1
  return ((double)(float)row[y] - (double)mx) * inv_tau - log(z);
}

// A thread's running sum of exp2((x - ref) k2).  The reference is the maximum of the thread's first batch that
// is not all -inf, not the running maximum: while the sum stays below 2^40 a later, larger score does no harm
// (the sum just exceeds its count), and the fast path needs neither a maximum nor a rescaling.  Beyond 2^40 (or
// for NaN) the batch is summed again against its own maximum.
struct Sum {
  float ref = -INFINITY, sm = 0.f;

  __device__ __forceinline__ void rebase(float to, float k2) {  // before the first batch, or to a larger reference
    if (ref != -INFINITY) sm *= exp2_hw((ref - to) * k2);  // (a NaN met before stays)
    ref = to;
  }
  // one element
  __device__ __forceinline__ void one(float x, float k2) {
    if (x == -INFINITY) return;
    if (x == x) rebase(x, k2);
    sm += x == x && x != INFINITY ? 1.f : NAN;
  }
  // vectors v, v + stride, .. of which those below `end` count (the others repeat one that does)
  template <typename T, int U, int STRIDE>
  __device__ __forceinline__ void batch(const u32x4 (&raw)[U], int v, int end, float k2) {
    constexpr int N = Vec<T>::N;
    auto largest = [&]() {
      float bm = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[N];
        unpack<T>(raw[u], f);
#pragma unroll
        for (int e = 0; e < N; ++e) bm = fmaxf(bm, f[e]);
      }
      return bm;
    };
    auto sum = [&]() {
      float a = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[N];
        unpack<T>(raw[u], f);
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) x += exp2_hw((f[e] - ref) * k2);
        if (v + u * STRIDE < end) a += x;
      }
      return a;
    };
    if (ref == -INFINITY) {
      const float bm = largest();
      if (bm == -INFINITY) {  // nothing, or NaN beside -inf
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[N];
          unpack<T>(raw[u], f);
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (f[e] != f[e]) sm = NAN;
        }
        return;
      }
      rebase(bm, k2);
    }
    float next = sm + sum();
    if (__builtin_expect(!(next <= 1.0995116e12f), 0)) {
      const float bm = largest();
      if (bm > ref) rebase(bm, k2);
      next = sm + sum();
    }
    sm = next;
  }
};

// ---- per-row scalars of the policy loss ------------------------------------------------------
struct Policy {
  const float* adv;
  const float* old_logp;
  const float* ref_logp;  // or null: no KL term
  const float* weights;   // or null: 1
  double lo, hi, kl, scale;
};

__device__ __forceinline__ void policy_row(const Policy& p, int64_t i, double l, double& loss, double& c) {
  const double a = p.adv[i], w = (p.weights ? (double)p.weights[i] : 1.0) * p.scale;
  const double r = exp(l - (double)p.old_logp[i]);
  const double held = fmin(fmax(r, 1.0 - p.lo), 1.0 + p.hi) * a, open = r * a;
  // a NaN ratio compares false: it takes the open side, so that it reaches loss and gradient
  const bool clipped = held < open;
  loss = clipped ? -held : -open;
  c = clipped ? 0.0 : -open;
  if (p.ref_logp) {
    const double d = (double)p.ref_logp[i] - l, em = expm1(d);
    loss += p.kl * (em == INFINITY ? em : em - d);
    c -= p.kl * em;
  }
  loss *= w;
  c *= w;
}

// What a pass leaves per row.  MODE 0: logp.  1: policy (logp, coefficient, loss).  2: logp and
// coefficient 0 (the pairs write theirs afterwards).
struct Rows {
  float* stats;  // [n, 2] (M, Z) or null
  float* logp;
  float* coef;
  double* loss;
};

template <int MODE>
__device__ __forceinline__ void put_row(const Rows& o, const Policy& pol, int64_t row, float mx, double z, double l,
                                        bool labelled) {
  double loss = 0.0, c = 0.0;
  if (MODE == 1 && labelled) policy_row(pol, row, l, loss, c);
  if (o.stats) {
    o.stats[2 * row] = mx;
    o.stats[2 * row + 1] = (float)z;
  }
  o.logp[row] = (float)l;
  if (MODE == 1) {
    o.coef[row] = (float)c;
    o.loss[row] = loss;
  }
  if (MODE == 2) o.coef[row] = 0.f;
}

// ---- pass 1: (M, Z) of every row, or of every part of a row ------------------------------------
// Several parts: part_stats[2 i] = M, [2 i + 1] = Z of part i = row * parts + part (the rows' scalars
// follow in rows_kernel, or where they are needed).  One part: the row's scalars at once.
constexpr int ST = 256;  // threads
// 16-byte loads in flight per thread: as many as leave eight waves per SIMD their registers
template <typename T>
constexpr int SU = sizeof(T) == 4 ? 8 : 4;

template <typename T, int MODE>
__global__ void __launch_bounds__(ST) stats_kernel(const T* __restrict__ s, int64_t lds, int m, int parts, int per,
                                                   const int64_t* __restrict__ labels, Temp t,
                                                   float* __restrict__ part_stats, Policy pol, Rows o) {
  __shared__ float redm[ST / 64];
  __shared__ double reds[ST / 64];
  const int64_t row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - row * parts), tid = threadIdx.x;
  const int64_t y = labels[row];
  if (y == -1) {
    if (parts == 1 && tid == 0) put_row<MODE>(o, pol, row, -INFINITY, 0.0, 0.0, false);
    return;
  }
  const Row<T> r(s + row * lds, m);
  if (MODE == 1 && parts > 1 && part == 0 && tid == 0) o.stats[2 * row] = y >= 0 && y < m ? (float)r.p[y] : NAN;
  const int v0 = part * per, v1 = min(r.nvec, v0 + per);
  const int je = ((part == 0 && tid < 8) || (part == parts - 1 && tid >= 8)) ? r.edge(tid) : -1;
  Sum acc;
  if (je >= 0) acc.one((float)r.p[je], t.k2);
  const u32x4* vp = r.vecs();
  constexpr int U = SU<T>;
  for (int b = v0; b < v1; b += ST * U) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = vp[min(b + u * ST + tid, v1 - 1)];
    acc.template batch<T, U, ST>(raw, b + tid, v1, t.k2);
  }
  const float mx = acc.ref;
  float sm = acc.sm;
  const float all = block_max<ST>(mx, redm);
  sm *= exp2_hw((mx - safe_max(all)) * t.k2);
  const double z = block_sum_wave0<ST>(sm, reds);
  if (tid != 0) return;
  if (parts == 1) {
    put_row<MODE>(o, pol, row, all, z, label_logp<T>(r.p, m, y, all, z, t.inv), true);
  } else {
    part_stats[2 * (int64_t)blockIdx.x] = all;
    part_stats[2 * (int64_t)blockIdx.x + 1] = (float)z;
  }
}

// (M, Z) of a row from its parts, by one wave; every lane gets them
__device__ __forceinline__ void join_parts(const float* ps, int parts, float k2, float& mx, double& z) {
  const int lane = threadIdx.x & 63;
  mx = -INFINITY;
  z = 0.0;
  for (int k = lane; k < parts; k += 64) mx = fmaxf(mx, ps[2 * k]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
  for (int k = lane; k < parts; k += 64) z += (double)(ps[2 * k + 1] * exp2_hw((ps[2 * k] - safe_max(mx)) * k2));
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) z += __shfl_xor(z, off, 64);
}

// ---- the rows' scalars from several parts: one wave per row ----------------------------------------
template <typename T, int MODE>
__global__ void __launch_bounds__(256) rows_kernel(const T* __restrict__ s, int64_t lds, int64_t n, int m, int parts,
                                                   const int64_t* __restrict__ labels, Temp t,
                                                   const float* __restrict__ part_stats, Policy pol, Rows o) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= n) return;
  const int64_t y = labels[row];
  float mx = -INFINITY;
  double z = 0.0, l = 0.0;
  if (y != -1) {
    join_parts(part_stats + 2 * row * parts, parts, t.k2, mx, z);
    l = label_logp<T>(s + row * lds, m, y, mx, z, t.inv);
  }
  if ((threadIdx.x & 63) == 0) put_row<MODE>(o, pol, row, mx, z, l, y != -1);
}

// ---- one wave per pair of sequences ------------------------------------------------------------
struct Pairs {
  const float* logp;
  const int64_t* labels;
  int64_t n;
  const int64_t* ptr;
  const float* ref;  // or null: 0
  double beta, smooth, scale;
  int average;
  float* seq_logp;
  float* coef;
};

// The pair's loss, in every lane
__device__ __forceinline__ double one_pair(const Pairs& p, int64_t pair, int lane) {
  int64_t b[3];
  for (int q = 0; q < 3; ++q) {
    const int64_t v = p.ptr[2 * pair + q];
    b[q] = v < 0 ? 0 : (v > p.n ? p.n : v);
  }
  double pi[2], rows[2];
  for (int q = 0; q < 2; ++q) {
    double a = 0.0, k = 0.0;
    for (int64_t i = b[q] + lane; i < b[q + 1]; i += 64)
      if (p.labels[i] != -1) {
        a += (double)p.logp[i];
        k += 1.0;
      }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      a += __shfl_xor(a, off, 64);
      k += __shfl_xor(k, off, 64);
    }
    rows[q] = p.average ? fmax(k, 1.0) : 1.0;
    pi[q] = a / rows[q];
  }
  const double rw = p.ref ? (double)p.ref[2 * pair] : 0.0, rl = p.ref ? (double)p.ref[2 * pair + 1] : 0.0;
  const double z = p.beta * ((pi[0] - rw) - (pi[1] - rl));
  const double e = exp(-fabs(z)), lp = log1p(e);
  const double up = (z >= 0 ? e : 1.0) / (1.0 + e);    // sigma(-z)
  const double down = (z >= 0 ? 1.0 : e) / (1.0 + e);  // sigma(z)
  // -log sigma(z) = max(-z, 0) + log1p(e), -log sigma(-z) = max(z, 0) + log1p(e)
  const double loss = (1.0 - p.smooth) * (fmax(-z, 0.0) + lp) + p.smooth * (fmax(z, 0.0) + lp);
  const double c = z != z ? z : -p.scale * p.beta * ((1.0 - p.smooth) * up - p.smooth * down);
  if (lane == 0) {
    p.seq_logp[2 * pair] = (float)pi[0];
    p.seq_logp[2 * pair + 1] = (float)pi[1];
  }
  for (int q = 0; q < 2; ++q)
    for (int64_t i = b[q] + lane; i < b[q + 1]; i += 64)
      if (p.labels[i] != -1) p.coef[i] = (float)((q ? -c : c) / rows[q]);
  return z != z ? z : p.scale * loss;
}

__global__ void __launch_bounds__(256) pairs_kernel(Pairs p, int64_t pairs, double* __restrict__ pair_loss) {
  const int64_t pair = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (pair >= pairs) return;
  const double loss = one_pair(p, pair, threadIdx.x & 63);
  if ((threadIdx.x & 63) == 0) pair_loss[pair] = loss;
}

// few pairs: one workgroup, the total in the same launch
__global__ void __launch_bounds__(1024) pairs_few_kernel(Pairs p, int pairs, float* __restrict__ total) {
  __shared__ double sum[16];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  double a = 0.0;
  for (int k = wave; k < pairs; k += 16) a += one_pair(p, k, lane);
  if (lane == 0) sum[wave] = a;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double x = 0.0;
  for (int w = 0; w < 16; ++w) x += sum[w];
  total[0] = (float)x;
}

// total of the per-row (per-pair) losses: one workgroup, fp64, fixed order
constexpr int TT = 1024;
__global__ void __launch_bounds__(TT) total_kernel(const double* __restrict__ v, int64_t n, float* __restrict__ out) {
  __shared__ double red[TT / 64];
  double a = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 4 * TT) {
    double x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = i + u * TT < n ? v[i + u * TT] : 0.0;
    a += (x[0] + x[1]) + (x[2] + x[3]);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) a += __shfl_xor(a, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < TT / 64; ++w) s += red[w];
  out[0] = (float)s;
}

// ---- the gradient of a row (or part of one) from its scalars ------------------------------------
// g_j = c [j = y] - e_j cz,  e_j = exp2((s_j - M) k2), cz = c / Z.  g may be the score row itself:
// every element is read and written by the same thread.
template <typename T>
__device__ __forceinline__ u32x4 grad_vec(const u32x4& raw, int j0, int y, float mx, float k2, float c, float cz) {
  constexpr int N = Vec<T>::N;
  float f[N];
  unpack<T>(raw, f);
#pragma unroll
  for (int e = 0; e < N; ++e) f[e] = -exp2_hw((f[e] - mx) * k2) * cz;
  if ((unsigned)(y - j0) < (unsigned)N) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (j0 + e == y) f[e] += c;
  }
  return pack<T>(f);
}

// Gradients are stored past the caches: at 60 MB read + 60 MB written a plain copy takes 24.4 us with ordinary
// stores and 19.1 us with these, a read followed by a copy 32.4 and 28.8 (the scores of a second pass stay
// in the memory-side cache: 100 against 82 us at 168 MB).
template <typename T>
__device__ __forceinline__ void store_vec(T* g, bool vec, int j0, const u32x4& v) {
  if (vec) {
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(g + j0));
  } else {
    const typename Vec<T>::type x = __builtin_bit_cast(typename Vec<T>::type, v);
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e) g[j0 + e] = x[e];
  }
}

template <typename T>
__device__ __forceinline__ bool same_alignment(const T* a, const T* b) {
  return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15u) == 0;
}

// MODE 0: from stored (M, Z) and coefficients.  MODE 1: policy, scalars from the parts' (M, Z); the workgroup of a
// row's first part writes them out.  Rows in descending order: the last ones pass 1 read are still
// in the memory-side cache.
template <typename T, int MODE>
__global__ void __launch_bounds__(ST) grad_kernel(const T* s, int64_t lds, int64_t n, int m, int parts, int per,
                                                  const int64_t* __restrict__ labels, Temp t,
                                                  const float* __restrict__ stats, const float* __restrict__ coef,
                                                  const float* __restrict__ gscale, Policy pol, Rows o, T* g, int64_t ldg) {
  constexpr int N = Vec<T>::N;
  const int64_t back = blockIdx.x / parts, row = n - 1 - back;
  const int part = parts - 1 - (int)(blockIdx.x - back * parts), tid = threadIdx.x;
  const int64_t yl = labels[row];
  const Row<T> r(s + row * lds, m);
  T* gr = g + row * ldg;
  const int v0 = part * per, v1 = min(r.nvec, v0 + per);
  const int je = ((part == 0 && tid < 8) || (part == parts - 1 && tid >= 8)) ? r.edge(tid) : -1;
  const bool vec = same_alignment(r.p, (const T*)gr);
  const u32x4* vp = r.vecs();
  const int y = (yl >= 0 && yl < m) ? (int)yl : -1;
  float c = 0.f, mx = 0.f, z = 1.f;
  // the first loads are on their way while the row's scalars are worked out
  constexpr int U = SU<T>;
  u32x4 raw[U];
  if (yl != -1 && v0 < v1) {
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = vp[min(v0 + u * ST + tid, v1 - 1)];
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = (u32x4){0u, 0u, 0u, 0u};
  }
  if (MODE == 0) {
    if (yl != -1) {
      c = (float)((double)coef[row] * (gscale ? (double)gscale[0] : 1.0) * t.inv);
      mx = stats[2 * row];
      z = stats[2 * row + 1];
    }
  } else if (yl == -1) {
    if (part == 0 && tid == 0) {
      o.logp[row] = 0.f;
      o.loss[row] = 0.0;
    }
  } else {
    // the label's score from pass 1: another workgroup may have overwritten it (g may be s)
    double zd, loss, cd;
    join_parts(stats + 2 * row * parts, parts, t.k2, mx, zd);
    z = (float)zd;
    const double l = y < 0 ? NAN : ((double)o.stats[2 * row] - (double)mx) * t.inv - log(zd);
    policy_row(pol, row, l, loss, cd);
    c = (float)(cd * t.inv);
    if (part == 0 && tid == 0) {
      o.logp[row] = (float)l;
      o.loss[row] = loss;
    }
  }
  if (c == 0.f) {
    const u32x4 zero = {0u, 0u, 0u, 0u};
    if (je >= 0) gr[je] = (T)0.f;
    for (int v = v0 + tid; v < v1; v += ST) store_vec<T>(gr, vec, r.head + v * N, zero);
    return;
  }
  mx = safe_max(mx);
  const float cz = y < 0 ? NAN : c / z;
  if (je >= 0) {
    const float v = -exp2_hw(((float)r.p[je] - mx) * t.k2) * cz;
    gr[je] = (T)(je == y ? v + c : v);
  }
  for (int b = v0; b < v1;) {
    u32x4 out[U];
#pragma unroll
    for (int u = 0; u < U; ++u) out[u] = grad_vec<T>(raw[u], r.head + (b + u * ST + tid) * N, y, mx, t.k2, c, cz);
    const int next = b + ST * U;
    if (next < v1) {
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = vp[min(next + u * ST + tid, v1 - 1)];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = b + u * ST + tid;
      if (v < v1) store_vec<T>(gr, vec, r.head + v * N, out[u]);
    }
    b = next;
  }
}

// ---- policy loss and gradient of rows that fit a workgroup's registers: one pass ----------------------
// NT threads hold NV 16-byte vectors each; the row is read once and its gradient written from the
// registers (every read happens before the barriers, every write after: g may be s).  The row's
// scalars are wave 0's work while the other waves wait; other workgroups of the CU fill that time.
// One row by NT threads (a workgroup, or with NT = 64 a wave, which needs no barrier); the first thread gets the
// row's loss.
template <typename T, int NT, int NV>
__device__ __forceinline__ double policy_row_fused(const T* s, int64_t lds, int m, int64_t row, int tid,
                                                   const int64_t* __restrict__ labels, Temp t, const Policy& pol,
                                                   float* __restrict__ logp, T* g, int64_t ldg, float* redm, double* reds,
                                                   float* sh) {
  constexpr int N = Vec<T>::N;
  const int64_t yl = labels[row];
  const Row<T> r(s + row * lds, m);
  T* gr = g + row * ldg;
  const int je = r.edge(tid);
  const bool vec = same_alignment(r.p, (const T*)gr);
  if (yl == -1) {
    const u32x4 zero = {0u, 0u, 0u, 0u};
    if (je >= 0) gr[je] = (T)0.f;
    for (int v = tid; v < r.nvec; v += NT) store_vec<T>(gr, vec, r.head + v * N, zero);
    if (tid == 0) logp[row] = 0.f;
    return 0.0;
  }
  const int y = (yl >= 0 && yl < m) ? (int)yl : -1;
  const u32x4* vp = r.vecs();
  u32x4 raw[NV];
  if (r.nvec > 0) {
#pragma unroll
    for (int u = 0; u < NV; ++u) raw[u] = vp[min(u * NT + tid, r.nvec - 1)];
  } else {
#pragma unroll
    for (int u = 0; u < NV; ++u) raw[u] = (u32x4){0u, 0u, 0u, 0u};
  }
  const float edge = je >= 0 ? (float)r.p[je] : -INFINITY;
  const float sy = y >= 0 ? (float)r.p[y] : NAN;
  float mx = je >= 0 ? edge : -INFINITY;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    if (u * NT + tid >= r.nvec) continue;
    float f[N];
    unpack<T>(raw[u], f);
#pragma unroll
    for (int e = 0; e < N; ++e) mx = fmaxf(mx, f[e]);
  }
  mx = block_max<NT>(mx, redm);
  const float ref = safe_max(mx);
  float sm = je >= 0 ? exp2_hw((edge - ref) * t.k2) : 0.f;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    if (u * NT + tid >= r.nvec) continue;
    float f[N], a = 0.f;
    unpack<T>(raw[u], f);
#pragma unroll
    for (int e = 0; e < N; ++e) a += exp2_hw((f[e] - ref) * t.k2);
    sm += a;
  }
  const double z = block_sum_wave0<NT>(sm, reds);
  double loss = 0.0;
  float c = 0.f, cz = 0.f;
  if (tid < 64) {
    const double l = ((double)sy - (double)mx) * t.inv - log(z);
    double cd;
    policy_row(pol, row, l, loss, cd);
    c = (float)(cd * t.inv);
    cz = y < 0 ? NAN : c / (float)z;
    if (tid == 0) logp[row] = (float)l;
  }
  if (NT > 64) {
    if (tid == 0) {
      sh[0] = c;
      sh[1] = cz;
    }
    __syncthreads();
    c = sh[0];
    cz = sh[1];
  }
  const bool off = c == 0.f;  // a zero gradient, whatever the scores
  if (je >= 0) {
    const float v = -exp2_hw((edge - ref) * t.k2) * cz;
    gr[je] = (T)(off ? 0.f : je == y ? v + c : v);
  }
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int v = u * NT + tid;
    if (v < r.nvec)
      store_vec<T>(gr, vec, r.head + v * N,
                   off ? (u32x4){0u, 0u, 0u, 0u} : grad_vec<T>(raw[u], r.head + v * N, y, ref, t.k2, c, cz));
  }
  return loss;
}

template <typename T, int NT, int NV>
__global__ void __launch_bounds__(NT) policy_fused_kernel(const T* s, int64_t lds, int m, const int64_t* __restrict__ labels,
                                                          Temp t, Policy pol, Rows o, T* g, int64_t ldg) {
  __shared__ float redm[NT / 64], sh[2];
  __shared__ double reds[NT / 64];
  const double loss = policy_row_fused<T, NT, NV>(s, lds, m, blockIdx.x, threadIdx.x, labels, t, pol, o.logp, g, ldg, redm,
                                                  reds, sh);
  if (threadIdx.x == 0) o.loss[blockIdx.x] = loss;
}

// Few short rows: one workgroup, a wave per row, the total in the same launch.  A launch costs the host
// about 3.3 us, the whole call of 16 x 500 scores 20.7 us with two of them.
template <typename T>
__global__ void __launch_bounds__(1024) policy_few_kernel(const T* s, int64_t lds, int n, int m,
                                                          const int64_t* __restrict__ labels, Temp t, Policy pol,
                                                          float* __restrict__ logp, T* g, int64_t ldg,
                                                          float* __restrict__ total) {
  __shared__ double sum[16];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  double a = 0.0;
  for (int row = wave; row < n; row += 16)
    a += policy_row_fused<T, 64, 4>(s, lds, m, row, lane, labels, t, pol, logp, g, ldg, nullptr, nullptr, nullptr);
  if (lane == 0) sum[wave] = a;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double x = 0.0;
  for (int w = 0; w < 16; ++w) x += sum[w];
  total[0] = (float)x;
}

#define KGE_TRY(expr)        \
  do {                       \
    const int _r = (expr);   \
    if (_r) return _r;       \
  } while (0)

// ---- host side ------------------------------------------------------------------------------------

int elem_size(int dtype) { return dtype == KGE_DT_F32 ? 4 : 2; }

// Parts a row is cut into: enough workgroups to fill the chip when there are few rows.  Rows of up
// to 64 KiB stay whole: one workgroup's two batches of loads, and no launch to join parts.
constexpr int64_t FILL = 2048, PART_MIN = 16384, WHOLE = 65536;
struct Split {
  int parts, per;  // per: 16-byte vectors per part
};
Split split_of(int64_t n, int64_t m, int dtype) {
  const int64_t bytes = m * elem_size(dtype);
  int64_t parts = bytes <= WHOLE ? 1 : std::min<int64_t>((FILL + n - 1) / n, (bytes + PART_MIN - 1) / PART_MIN);
  const int64_t vecs = bytes / 16;
  int64_t per = (vecs + parts - 1) / parts;
  if (per < 1) per = 1;
  parts = std::max<int64_t>(1, (vecs + per - 1) / per);
  return {(int)parts, (int)per};
}

int64_t round256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// workspace: part stats | row stats | coefficients | row (pair) losses
struct Ws {
  float *part, *stats, *coef;
  double* loss;
  int64_t bytes;
};
Ws ws_of(void* base, int64_t n, int64_t m, int dtype, int64_t pairs) {
  char* b = (char*)base;
  Ws w;
  int64_t o = 0;
  w.part = (float*)(b + o);
  // ceil(FILL / k) parts of k <= n rows: below FILL + n
  if (n > 0 && m * elem_size(dtype) > WHOLE) o += round256((n + FILL) * 8);
  w.stats = (float*)(b + o);
  o += round256(n * 8);
  w.coef = (float*)(b + o);
  o += round256(n * 4);
  w.loss = (double*)(b + o);
  o += round256(std::max(n, pairs) * 8);
  w.bytes = o;
  return w;
}

bool temperature_ok(double t) { return t >= 1e-30 && t <= 1e30; }  // (1 / t is a 32-bit factor, neither 0 nor infinite)

// (a launch has at most n + FILL workgroups)
bool shape_ok(const void* s, int dtype, int64_t lds, int64_t n, int64_t m, const int64_t* labels) {
  return dtype >= KGE_DT_F32 && dtype <= KGE_DT_F16 && n >= 0 && m >= 1 && m < (int64_t)1 << 31 && lds >= (n > 1 ? m : 0) &&
         n <= (int64_t)1 << 30 && (n == 0 || (s && labels)) &&
         (reinterpret_cast<uintptr_t>(s) % elem_size(dtype)) == 0;
}

// The rows' scalars: pass 1, and the join of its parts where `join` and rows have several.
template <typename T, int MODE>
int run_rows(const T* s, int64_t lds, int64_t n, int64_t m, const Split& sp, const int64_t* labels, Temp t, float* part,
             const Policy& pol, const Rows& o, bool join, hipStream_t st) {
  stats_kernel<T, MODE><<<dim3((unsigned)(n * sp.parts)), dim3(ST), 0, st>>>(s, lds, (int)m, sp.parts, sp.per, labels, t,
                                                                             part, pol, o);
  KGE_CHECK_LAUNCH();
  if (sp.parts == 1 || !join) return 0;
  rows_kernel<T, MODE><<<dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st>>>(s, lds, n, (int)m, sp.parts, labels, t, part,
                                                                            pol, o);
  KGE_CHECK_LAUNCH();
  return 0;
}

template <typename T>
int run_grad(const T* s, int64_t lds, int64_t n, int64_t m, const Split& sp, const int64_t* labels, Temp t,
             const float* stats, const float* coef, const float* gscale, T* g, int64_t ldg, hipStream_t st) {
  grad_kernel<T, 0><<<dim3((unsigned)(n * sp.parts)), dim3(ST), 0, st>>>(
      s, lds, n, (int)m, sp.parts, sp.per, labels, t, stats, coef, gscale, Policy{}, Rows{}, g, ldg);
  KGE_CHECK_LAUNCH();
  return 0;
}

// Policy loss with its gradient.  Rows of up to 256 KiB are read once, by the smallest workgroup that
// holds them (a 1024-thread workgroup leaves no second one on its CU to fill its waits).  Longer rows are read
// twice, in groups of rows whose scores stay in the memory-side cache (256 MB) between the passes.
constexpr int64_t GROUP = 128 << 20;

template <typename T, int NT, int NV>
int launch_fused(const T* s, int64_t lds, int64_t n, int64_t m, const int64_t* labels, Temp t, const Policy& pol,
                 const Rows& o, T* g, int64_t ldg, hipStream_t st) {
  policy_fused_kernel<T, NT, NV><<<dim3((unsigned)n), dim3(NT), 0, st>>>(s, lds, (int)m, labels, t, pol, o, g, ldg);
  KGE_CHECK_LAUNCH();
  return 0;
}

template <typename T>
int run_policy_grad(const T* s, int64_t lds, int64_t n, int64_t m, int dtype, const int64_t* labels, Temp t, float* part,
                    const Policy& pol, const Rows& o, T* g, int64_t ldg, hipStream_t st) {
  const int64_t bytes = m * (int64_t)sizeof(T);
  if (bytes <= 1 << 10) return launch_fused<T, 64, 1>(s, lds, n, m, labels, t, pol, o, g, ldg, st);
  if (bytes <= 4 << 10) return launch_fused<T, 64, 4>(s, lds, n, m, labels, t, pol, o, g, ldg, st);
  if (bytes <= 16 << 10) return launch_fused<T, 256, 4>(s, lds, n, m, labels, t, pol, o, g, ldg, st);
  if (bytes <= 32 << 10) return launch_fused<T, 256, 8>(s, lds, n, m, labels, t, pol, o, g, ldg, st);
  if (bytes <= 64 << 10) return launch_fused<T, 512, 8>(s, lds, n, m, labels, t, pol, o, g, ldg, st);
  if (bytes <= 128 << 10) return launch_fused<T, 1024, 8>(s, lds, n, m, labels, t, pol, o, g, ldg, st);
  if (bytes <= 256 << 10 && n >= 64) return launch_fused<T, 1024, 16>(s, lds, n, m, labels, t, pol, o, g, ldg, st);
  const int64_t rows = std::min(n, std::max<int64_t>(1, GROUP / bytes));
  for (int64_t i = 0; i < n; i += rows) {
    const int64_t k = std::min(rows, n - i);
    const Split sp = split_of(k, m, dtype);
    Policy p = pol;
    p.adv += i;
    p.old_logp += i;
    if (p.ref_logp) p.ref_logp += i;
    if (p.weights) p.weights += i;
    const Rows r{o.stats + 2 * i, o.logp + i, o.coef + i, o.loss + i};
    KGE_TRY((run_rows<T, 1>(s + i * lds, lds, k, m, sp, labels + i, t, part, p, r, false, st)));
    grad_kernel<T, 1><<<dim3((unsigned)(k * sp.parts)), dim3(ST), 0, st>>>(
        s + i * lds, lds, k, (int)m, sp.parts, sp.per, labels + i, t, part, nullptr, nullptr, p, r, g + i * ldg, ldg);
    KGE_CHECK_LAUNCH();
  }
  return 0;
}

int run_total(const double* v, int64_t n, float* out, hipStream_t st) {
  total_kernel<<<dim3(1), dim3(TT), 0, st>>>(v, n, out);
  KGE_CHECK_LAUNCH();
  return 0;
}

// f(pointer type tag) for the element type of a dtype code
template <typename F>
int by_type(int dtype, F f) {
  if (dtype == KGE_DT_F32) return f((float*)nullptr);
  if (dtype == KGE_DT_BF16) return f((__bf16*)nullptr);
  return f((_Float16*)nullptr);
}

}  // namespace

extern "C" int64_t kge_label_ws_size(int64_t n, int64_t m, int dtype, int64_t pairs) {
  if (n < 0 || m < 1 || pairs < 0 || dtype < KGE_DT_F32 || dtype > KGE_DT_F16) return 0;
  return ws_of(nullptr, n, m, dtype, pairs).bytes;
}

extern "C" int kge_label_logprobs(const void* s, int dtype, int64_t lds, int64_t n, int64_t m, const int64_t* labels,
                                  double temperature, float* logp, float* stats, void* ws, int64_t ws_bytes,
                                  void* stream) {
  KGE_REQUIRE(shape_ok(s, dtype, lds, n, m, labels) && temperature_ok(temperature));
  if (n == 0) return 0;
  const Ws w = ws_of(ws, n, m, dtype, 0);
  KGE_REQUIRE(logp && ws && ws_bytes >= w.bytes && aligned16(ws));
  const Temp t = temp_of(temperature);
  return by_type(dtype, [&](auto* tag) -> int {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    return run_rows<T, 0>((const T*)s, lds, n, m, split_of(n, m, dtype), labels, t, w.part, Policy{},
                          Rows{stats, logp, nullptr, nullptr}, true, as_stream(stream));
  });
}

extern "C" int kge_label_grad(const void* s, int dtype, int64_t lds, int64_t n, int64_t m, const int64_t* labels,
                              double temperature, const float* stats, const float* coef, const float* gscale, void* g,
                              int64_t ldg, void* stream) {
  KGE_REQUIRE(shape_ok(s, dtype, lds, n, m, labels) && temperature_ok(temperature));
  if (n == 0) return 0;
  KGE_REQUIRE(stats && coef && g && ldg >= (n > 1 ? m : 0) && (reinterpret_cast<uintptr_t>(g) % elem_size(dtype)) == 0);
  const Temp t = temp_of(temperature);
  return by_type(dtype, [&](auto* tag) -> int {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    return run_grad<T>((const T*)s, lds, n, m, split_of(n, m, dtype), labels, t, stats, coef, gscale, (T*)g, ldg,
                       as_stream(stream));
  });
}

extern "C" int kge_policy_loss(const void* s, int dtype, int64_t lds, int64_t n, int64_t m, const int64_t* labels,
                               const float* advantages, const float* old_logp, const float* ref_logp,
                               const float* weights, double clip_low, double clip_high, double kl, double temperature,
                               double scale, float* loss, float* logp, float* stats, float* coef, void* g, int64_t ldg,
                               void* ws, int64_t ws_bytes, void* stream) {
  KGE_REQUIRE(shape_ok(s, dtype, lds, n, m, labels) && temperature_ok(temperature) && loss);
  const hipStream_t st = as_stream(stream);
  if (n == 0) return run_total(nullptr, 0, loss, st);
  const Ws w = ws_of(ws, n, m, dtype, 0);
  KGE_REQUIRE(advantages && old_logp && logp && ws && ws_bytes >= w.bytes && aligned16(ws));
  KGE_REQUIRE(!g || (!stats && !coef && ldg >= (n > 1 ? m : 0) && (reinterpret_cast<uintptr_t>(g) % elem_size(dtype)) == 0));
  const Temp t = temp_of(temperature);
  const Policy pol{advantages, old_logp, ref_logp, weights, clip_low, clip_high, kl, scale};
  if (!stats) stats = w.stats;
  if (!coef) coef = w.coef;
  return by_type(dtype, [&](auto* tag) -> int {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    const Rows o{stats, logp, coef, w.loss};
    if (g && n <= 64 && m * (int64_t)sizeof(T) <= 4096) {
      policy_few_kernel<T><<<dim3(1), dim3(1024), 0, st>>>((const T*)s, lds, (int)n, (int)m, labels, t, pol, logp, (T*)g, ldg,
                                                           loss);
      KGE_CHECK_LAUNCH();
      return 0;
    }
    if (g)
      KGE_TRY(run_policy_grad<T>((const T*)s, lds, n, m, dtype, labels, t, w.part, pol, o, (T*)g, ldg, st));
    else
      KGE_TRY((run_rows<T, 1>((const T*)s, lds, n, m, split_of(n, m, dtype), labels, t, w.part, pol, o, true, st)));
    return run_total(w.loss, n, loss, st);
  });
}

extern "C" int kge_preference_loss(const void* s, int dtype, int64_t lds, int64_t n, int64_t m, const int64_t* labels,
                                   const int64_t* seq_ptr, int64_t pairs, const float* ref_logp, double beta,
                                   double smoothing, int average, double temperature, double scale, float* loss,
                                   float* seq_logp, float* logp, float* stats, float* coef, void* g, int64_t ldg,
                                   void* ws, int64_t ws_bytes, void* stream) {
  KGE_REQUIRE(shape_ok(s, dtype, lds, n, m, labels) && temperature_ok(temperature) && loss && pairs >= 0);
  const hipStream_t st = as_stream(stream);
  const Ws w = ws_of(ws, n, m, dtype, pairs);
  KGE_REQUIRE((n == 0 && pairs == 0) || (ws && ws_bytes >= w.bytes && aligned16(ws)));
  KGE_REQUIRE(pairs == 0 || (seq_ptr && seq_logp));
  KGE_REQUIRE(n == 0 || logp);
  KGE_REQUIRE(!g || (ldg >= (n > 1 ? m : 0) && (reinterpret_cast<uintptr_t>(g) % elem_size(dtype)) == 0));
  const Temp t = temp_of(temperature);
  if (!stats) stats = w.stats;
  if (!coef) coef = w.coef;
  return by_type(dtype, [&](auto* tag) -> int {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    const Split sp = n > 0 ? split_of(n, m, dtype) : Split{1, 1};
    if (n > 0)
      KGE_TRY((run_rows<T, 2>((const T*)s, lds, n, m, sp, labels, t, w.part, Policy{}, Rows{stats, logp, coef, nullptr},
                              true, st)));
    const Pairs p{logp, labels, n, seq_ptr, ref_logp, beta, smoothing, scale, average, seq_logp, coef};
    const bool few = pairs <= 64;  // (0 too: the total of nothing)
    if (few)
      pairs_few_kernel<<<dim3(1), dim3(1024), 0, st>>>(p, (int)pairs, loss);
    else
      pairs_kernel<<<dim3((unsigned)((pairs + 3) / 4)), dim3(256), 0, st>>>(p, pairs, w.loss);
    KGE_CHECK_LAUNCH();
    if (g && n > 0) KGE_TRY(run_grad<T>((const T*)s, lds, n, m, sp, labels, t, stats, coef, nullptr, (T*)g, ldg, st));
    return few ? 0 : run_total(w.loss, pairs, loss, st);
  });
}
