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

// ---- pass 1: (M, Z) of every row, or of every part of a row ------------------------------------
// stats[2 i] = M_i, stats[2 i + 1] = Z_i of row part i = row * parts + part.
constexpr int ST = 256, SU = 8;  // threads, 16-byte loads in flight per thread

template <typename T>
__global__ void __launch_bounds__(ST) stats_kernel(const T* __restrict__ s, int64_t lds, int m, int parts, int per,
                                                   const int64_t* __restrict__ labels, Temp t,
                                                   float* __restrict__ stats) {
  __shared__ float redm[ST / 64];
  __shared__ double reds[ST / 64];
  constexpr int N = Vec<T>::N;
  const int64_t row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - row * parts), tid = threadIdx.x;
  if (labels[row] == -1) return;
  const Row<T> r(s + row * lds, m);
  const int v0 = part * per, v1 = min(r.nvec, v0 + per);
  const int je = ((part == 0 && tid < 8) || (part == parts - 1 && tid >= 8)) ? r.edge(tid) : -1;
  float mx = -INFINITY, sm = 0.f;
  if (je >= 0) {
    mx = (float)r.p[je];
    sm = mx == -INFINITY ? 0.f : (mx == mx && mx != INFINITY ? 1.f : NAN);
  }
  const u32x4* vp = r.vecs();
  for (int b = v0; b < v1; b += ST * SU) {
    u32x4 raw[SU];
#pragma unroll
    for (int u = 0; u < SU; ++u) raw[u] = vp[min(b + u * ST + tid, v1 - 1)];
    float bm = mx;
#pragma unroll
    for (int u = 0; u < SU; ++u) {
      float f[N];
      unpack<T>(raw[u], f);
#pragma unroll
      for (int e = 0; e < N; ++e) bm = fmaxf(bm, f[e]);  // a clamped repeat changes no maximum
    }
    const float ref = safe_max(bm);
    sm *= exp2_hw((mx - ref) * t.k2);
    mx = bm;
#pragma unroll
    for (int u = 0; u < SU; ++u) {
      float f[N], a = 0.f;
      unpack<T>(raw[u], f);
#pragma unroll
      for (int e = 0; e < N; ++e) a += exp2_hw((f[e] - ref) * t.k2);
      if (b + u * ST + tid < v1) sm += a;
    }
  }
  const float all = block_max<ST>(mx, redm);
  sm *= exp2_hw((mx - safe_max(all)) * t.k2);
  const double z = block_sum_wave0<ST>(sm, reds);
  if (tid == 0) {
    stats[2 * (int64_t)blockIdx.x] = all;
    stats[2 * (int64_t)blockIdx.x + 1] = (float)z;
  }
}

// ---- the rows' scalars from the parts: one wave per row ----------------------------------------
// MODE 0: logp.  1: policy.  2: logp and coef = 0 (the pairs write theirs afterwards).
template <typename T, int MODE>
__global__ void __launch_bounds__(256) rows_kernel(const T* __restrict__ s, int64_t lds, int64_t n, int m, int parts,
                                                   const int64_t* __restrict__ labels, Temp t,
                                                   const float* __restrict__ part_stats, Policy pol,
                                                   float* __restrict__ stats, float* __restrict__ logp,
                                                   float* __restrict__ coef, double* __restrict__ row_loss) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= n) return;
  const int64_t y = labels[row];
  float mx = -INFINITY;
  double z = 0.0, l = 0.0, loss = 0.0, c = 0.0;
  if (y != -1) {
    const float* ps = part_stats + 2 * row * parts;
    for (int k = lane; k < parts; k += 64) mx = fmaxf(mx, ps[2 * k]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
    for (int k = lane; k < parts; k += 64)
      z += (double)(ps[2 * k + 1] * exp2_hw((ps[2 * k] - safe_max(mx)) * t.k2));
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) z += __shfl_xor(z, off, 64);
    if (lane == 0) l = label_logp<T>(s + row * lds, m, y, mx, z, t.inv);
    if (MODE == 1 && lane == 0) policy_row(pol, row, l, loss, c);
  }
  if (lane != 0) return;
  if (stats) {
    stats[2 * row] = mx;
    stats[2 * row + 1] = (float)z;
  }
  logp[row] = (float)l;
  if (MODE == 1) {
    coef[row] = (float)c;
    row_loss[row] = loss;
  }
  if (MODE == 2) coef[row] = 0.f;
}

// ---- one wave per pair of sequences ------------------------------------------------------------
__global__ void __launch_bounds__(256) pairs_kernel(const float* __restrict__ logp, const int64_t* __restrict__ labels,
                                                    int64_t n, const int64_t* __restrict__ ptr, int64_t pairs,
                                                    const float* __restrict__ ref, double beta, double smooth,
                                                    int average, double scale, float* __restrict__ seq_logp,
                                                    float* __restrict__ coef, double* __restrict__ pair_loss) {
  const int64_t pair = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (pair >= pairs) return;
  int64_t b[3];
  for (int q = 0; q < 3; ++q) {
    const int64_t v = ptr[2 * pair + q];
    b[q] = v < 0 ? 0 : (v > n ? n : v);
  }
  double pi[2], rows[2];
  for (int q = 0; q < 2; ++q) {
    double a = 0.0, k = 0.0;
    for (int64_t i = b[q] + lane; i < b[q + 1]; i += 64)
      if (labels[i] != -1) {
        a += (double)logp[i];
        k += 1.0;
      }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      a += __shfl_xor(a, off, 64);
      k += __shfl_xor(k, off, 64);
    }
    rows[q] = average ? fmax(k, 1.0) : 1.0;
    pi[q] = a / rows[q];
  }
  const double rw = ref ? (double)ref[2 * pair] : 0.0, rl = ref ? (double)ref[2 * pair + 1] : 0.0;
  const double z = beta * ((pi[0] - rw) - (pi[1] - rl));
  const double e = exp(-fabs(z)), lp = log1p(e);
  const double up = (z >= 0 ? e : 1.0) / (1.0 + e);    // sigma(-z)
  const double down = (z >= 0 ? 1.0 : e) / (1.0 + e);  // sigma(z)
  // -log sigma(z) = max(-z, 0) + log1p(e), -log sigma(-z) = max(z, 0) + log1p(e)
  const double loss = (1.0 - smooth) * (fmax(-z, 0.0) + lp) + smooth * (fmax(z, 0.0) + lp);
  const double c = z != z ? z : -scale * beta * ((1.0 - smooth) * up - smooth * down);
  if (lane == 0) {
    seq_logp[2 * pair] = (float)pi[0];
    seq_logp[2 * pair + 1] = (float)pi[1];
    pair_loss[pair] = z != z ? z : scale * loss;
  }
  for (int q = 0; q < 2; ++q)
    for (int64_t i = b[q] + lane; i < b[q + 1]; i += 64)
      if (labels[i] != -1) coef[i] = (float)((q ? -c : c) / rows[q]);
}

// total of the per-row (per-pair) losses: one workgroup, fp64, fixed order
__global__ void __launch_bounds__(256) total_kernel(const double* __restrict__ v, int64_t n, float* __restrict__ out) {
  __shared__ double red[4];
  double a = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 256) a += v[i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) a += __shfl_xor(a, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  if (threadIdx.x == 0) out[0] = (float)((red[0] + red[1]) + (red[2] + red[3]));
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

template <typename T>
__device__ __forceinline__ void store_vec(T* g, bool vec, int j0, const u32x4& v) {
  if (vec) {
    *reinterpret_cast<u32x4*>(g + j0) = v;
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

template <typename T>
__global__ void __launch_bounds__(ST) grad_kernel(const T* s, int64_t lds, int m, int parts, int per,
                                                  const int64_t* __restrict__ labels, Temp t,
                                                  const float* __restrict__ stats, const float* __restrict__ coef,
                                                  const float* __restrict__ gscale, T* g, int64_t ldg) {
  constexpr int N = Vec<T>::N;
  const int64_t row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - row * parts), tid = threadIdx.x;
  const int64_t yl = labels[row];
  const Row<T> r(s + row * lds, m);
  T* gr = g + row * ldg;
  const int v0 = part * per, v1 = min(r.nvec, v0 + per);
  const int je = ((part == 0 && tid < 8) || (part == parts - 1 && tid >= 8)) ? r.edge(tid) : -1;
  const bool vec = same_alignment(r.p, (const T*)gr);
  const u32x4* vp = r.vecs();
  float c = 0.f;
  if (yl != -1) c = (float)((double)coef[row] * (gscale ? (double)gscale[0] : 1.0) * t.inv);
  if (c == 0.f) {
    const u32x4 zero = {0u, 0u, 0u, 0u};
    if (je >= 0) gr[je] = (T)0.f;
    for (int v = v0 + tid; v < v1; v += ST) store_vec<T>(gr, vec, r.head + v * N, zero);
    return;
  }
  const int y = (yl >= 0 && yl < m) ? (int)yl : -1;
  const float mx = safe_max(stats[2 * row]);
  const float cz = (y < 0) ? NAN : c / stats[2 * row + 1];
  if (je >= 0) {
    const float v = -exp2_hw(((float)r.p[je] - mx) * t.k2) * cz;
    gr[je] = (T)(je == y ? v + c : v);
  }
  for (int b = v0; b < v1; b += ST * SU) {
    u32x4 raw[SU];
#pragma unroll
    for (int u = 0; u < SU; ++u) raw[u] = vp[min(b + u * ST + tid, v1 - 1)];
#pragma unroll
    for (int u = 0; u < SU; ++u) {
      const int v = b + u * ST + tid;
      if (v < v1) store_vec<T>(gr, vec, r.head + v * N, grad_vec<T>(raw[u], r.head + v * N, y, mx, t.k2, c, cz));
    }
  }
}

// ---- host side ------------------------------------------------------------------------------------

int elem_size(int dtype) { return dtype == KGE_DT_F32 ? 4 : 2; }

// Parts a row is cut into: enough workgroups to fill the chip when there are few rows, parts of
// at least 16 KiB (one batch of loads is 32 KiB).
constexpr int64_t FILL = 2048, PART_MIN = 16384;
struct Split {
  int parts, per;  // per: 16-byte vectors per part
};
Split split_of(int64_t n, int64_t m, int dtype) {
  const int64_t bytes = m * elem_size(dtype);
  int64_t parts = std::min<int64_t>((FILL + n - 1) / n, (bytes + PART_MIN - 1) / PART_MIN);
  if (parts < 1) parts = 1;
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
  const Split sp = n > 0 ? split_of(n, m, dtype) : Split{1, 1};
  char* b = (char*)base;
  Ws w;
  int64_t o = 0;
  w.part = (float*)(b + o);
  o += round256(n * sp.parts * 8);
  w.stats = (float*)(b + o);
  o += round256(n * 8);
  w.coef = (float*)(b + o);
  o += round256(n * 4);
  w.loss = (double*)(b + o);
  o += round256(std::max(n, pairs) * 8);
  w.bytes = o;
  return w;
}

bool shape_ok(const void* s, int dtype, int64_t lds, int64_t n, int64_t m, const int64_t* labels) {
  return dtype >= KGE_DT_F32 && dtype <= KGE_DT_F16 && n >= 0 && m >= 1 && m < (int64_t)1 << 31 && lds >= (n > 1 ? m : 0) &&
         n <= ((int64_t)1 << 31) / (FILL + 1) && (n == 0 || (s && labels)) &&
         (reinterpret_cast<uintptr_t>(s) % elem_size(dtype)) == 0;
}

template <typename T>
int run_stats(const T* s, int64_t lds, int64_t n, int64_t m, int dtype, const int64_t* labels, Temp t, float* part,
              hipStream_t st) {
  const Split sp = split_of(n, m, dtype);
  stats_kernel<T><<<dim3((unsigned)(n * sp.parts)), dim3(ST), 0, st>>>(s, lds, (int)m, sp.parts, sp.per, labels, t, part);
  KGE_CHECK_LAUNCH();
  return 0;
}

template <typename T, int MODE>
int run_rows(const T* s, int64_t lds, int64_t n, int64_t m, int dtype, const int64_t* labels, Temp t, const float* part,
             const Policy& pol, float* stats, float* logp, float* coef, double* loss, hipStream_t st) {
  const Split sp = split_of(n, m, dtype);
  rows_kernel<T, MODE><<<dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st>>>(s, lds, n, (int)m, sp.parts, labels, t, part,
                                                                            pol, stats, logp, coef, loss);
  KGE_CHECK_LAUNCH();
  return 0;
}

template <typename T>
int run_grad(const T* s, int64_t lds, int64_t n, int64_t m, int dtype, const int64_t* labels, Temp t,
             const float* stats, const float* coef, const float* gscale, T* g, int64_t ldg, hipStream_t st) {
  const Split sp = split_of(n, m, dtype);
  grad_kernel<T><<<dim3((unsigned)(n * sp.parts)), dim3(ST), 0, st>>>(s, lds, (int)m, sp.parts, sp.per, labels, t, stats,
                                                                      coef, gscale, g, ldg);
  KGE_CHECK_LAUNCH();
  return 0;
}

int run_total(const double* v, int64_t n, float* out, hipStream_t st) {
  total_kernel<<<dim3(1), dim3(256), 0, st>>>(v, n, out);
  KGE_CHECK_LAUNCH();
  return 0;
}

#define KGE_TRY(expr)        \
  do {                       \
    const int _r = (expr);   \
    if (_r) return _r;       \
  } while (0)

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
  KGE_REQUIRE(shape_ok(s, dtype, lds, n, m, labels) && temperature > 0.0);
  if (n == 0) return 0;
  const Ws w = ws_of(ws, n, m, dtype, 0);
  KGE_REQUIRE(logp && ws && ws_bytes >= w.bytes && aligned16(ws));
  const Temp t = temp_of(temperature);
  return by_type(dtype, [&](auto* tag) -> int {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    KGE_TRY(run_stats<T>((const T*)s, lds, n, m, dtype, labels, t, w.part, as_stream(stream)));
    return run_rows<T, 0>((const T*)s, lds, n, m, dtype, labels, t, w.part, Policy{}, stats, logp, nullptr, nullptr,
                          as_stream(stream));
  });
}

extern "C" int kge_label_grad(const void* s, int dtype, int64_t lds, int64_t n, int64_t m, const int64_t* labels,
                              double temperature, const float* stats, const float* coef, const float* gscale, void* g,
                              int64_t ldg, void* stream) {
  KGE_REQUIRE(shape_ok(s, dtype, lds, n, m, labels) && temperature > 0.0);
  if (n == 0) return 0;
  KGE_REQUIRE(stats && coef && g && ldg >= (n > 1 ? m : 0) && (reinterpret_cast<uintptr_t>(g) % elem_size(dtype)) == 0);
  const Temp t = temp_of(temperature);
  return by_type(dtype, [&](auto* tag) -> int {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    return run_grad<T>((const T*)s, lds, n, m, dtype, labels, t, stats, coef, gscale, (T*)g, ldg, as_stream(stream));
  });
}

extern "C" int kge_policy_loss(const void* s, int dtype, int64_t lds, int64_t n, int64_t m, const int64_t* labels,
                               const float* advantages, const float* old_logp, const float* ref_logp,
                               const float* weights, double clip_low, double clip_high, double kl, double temperature,
                               double scale, float* loss, float* logp, float* stats, float* coef, void* g, int64_t ldg,
                               void* ws, int64_t ws_bytes, void* stream) {
  KGE_REQUIRE(shape_ok(s, dtype, lds, n, m, labels) && temperature > 0.0 && loss);
  const hipStream_t st = as_stream(stream);
  if (n == 0) return run_total(nullptr, 0, loss, st);
  const Ws w = ws_of(ws, n, m, dtype, 0);
  KGE_REQUIRE(advantages && old_logp && logp && ws && ws_bytes >= w.bytes && aligned16(ws));
  KGE_REQUIRE(!g || (ldg >= (n > 1 ? m : 0) && (reinterpret_cast<uintptr_t>(g) % elem_size(dtype)) == 0));
  const Temp t = temp_of(temperature);
  const Policy pol{advantages, old_logp, ref_logp, weights, clip_low, clip_high, kl, scale};
  if (!stats) stats = w.stats;
  if (!coef) coef = w.coef;
  return by_type(dtype, [&](auto* tag) -> int {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    const T* sp = (const T*)s;
    KGE_TRY(run_stats<T>(sp, lds, n, m, dtype, labels, t, w.part, st));
    KGE_TRY((run_rows<T, 1>(sp, lds, n, m, dtype, labels, t, w.part, pol, stats, logp, coef, w.loss, st)));
    if (g) KGE_TRY(run_grad<T>(sp, lds, n, m, dtype, labels, t, stats, coef, nullptr, (T*)g, ldg, st));
    return run_total(w.loss, n, loss, st);
  });
}

extern "C" int kge_preference_loss(const void* s, int dtype, int64_t lds, int64_t n, int64_t m, const int64_t* labels,
                                   const int64_t* seq_ptr, int64_t pairs, const float* ref_logp, double beta,
                                   double smoothing, int average, double temperature, double scale, float* loss,
                                   float* seq_logp, float* logp, float* stats, float* coef, void* g, int64_t ldg,
                                   void* ws, int64_t ws_bytes, void* stream) {
  KGE_REQUIRE(shape_ok(s, dtype, lds, n, m, labels) && temperature > 0.0 && loss && pairs >= 0);
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
    const T* sp = (const T*)s;
    if (n > 0) {
      KGE_TRY(run_stats<T>(sp, lds, n, m, dtype, labels, t, w.part, st));
      KGE_TRY((run_rows<T, 2>(sp, lds, n, m, dtype, labels, t, w.part, Policy{}, stats, logp, coef, nullptr, st)));
    }
    if (pairs > 0) {
      pairs_kernel<<<dim3((unsigned)((pairs + 3) / 4)), dim3(256), 0, st>>>(logp, labels, n, seq_ptr, pairs, ref_logp,
                                                                            beta, smoothing, average, scale, seq_logp,
                                                                            coef, w.loss);
      KGE_CHECK_LAUNCH();
    }
    if (g && n > 0) KGE_TRY(run_grad<T>(sp, lds, n, m, dtype, labels, t, stats, coef, nullptr, (T*)g, ldg, st));
    return run_total(w.loss, pairs, loss, st);
  });
}
