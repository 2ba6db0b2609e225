// Low-rank adapters of many requests beside a shared projection:
//
//   y_i = W x_i + B_t h_i,   h_i = scale_t A_t x_i,   t = ids[i]          (t = -1: y_i = W x_i)
//
// W [m, d] shared, A_t [r, d] and B_t [m, r] of adapter t in [0, k), rows x_i [d] of n requests in any
// order; fp32 (v_mfma_f32_16x16x4_f32) or bf16 (v_mfma_f32_16x16x32_bf16), sums in fp32, the result
// rounded once.  The gradients for dy:
//
//   u_i = scale_t B_t^T dy_i     dA_t = sum_{i in t} u_i x_i^T     dB_t = sum_{i in t} dy_i h_i^T
//   dx_i = W^T dy_i + A_t^T u_i
//
// The rows are worked on in the order of their adapters (a stable counting sort of the ids: plan), so
// that an adapter is read for 16 of its rows at a time; rows are gathered and scattered through the
// order, never copied.  Four kernels:
//   shrink   h (and u): [<= 16 rows of one adapter] x [d] x [r], the four waves of a workgroup split d
//   project  W x + B h: a tiled product whose epilogue adds B_t h for every adapter among a fragment's 16
//            rows.  Each adapter's product goes into accumulators of its own and is added to its own rows only:
//            an adapter with infinities or NaN cannot reach another request's row.
//   grads    dA / dB: [r] x [rows of one adapter] x [columns] on the fp32 matrix instruction whatever the
//            type (its operands hold one value per lane along the summed axis, so rows need no transpose)
// h and u are kept in fp32; where they meet a bf16 B_t on the bf16 instruction they are split into hi + lo
// (2^-16), both halves in one instruction: 16 ranks fill half of its 32-wide summed axis.
#include <math.h>

#include <type_traits>

#include "common.h"

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Mma;
template <>
struct Mma<__bf16> {
  static constexpr int N = 8;   // elements of a lane's 16 bytes
  static constexpr int KC = 32;  // summed elements of one fragment: 4 lane groups x N
  // c += a b^T over the fragment's KC elements: a row (lane & 15) of a meets a row (lane & 15) of b;
  // c: a's row (lane >> 4) * 4 + reg, b's row lane & 15
  static __device__ __forceinline__ void run(f32x4& c, const u32x4& a, const u32x4& b) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<float> {
  static constexpr int N = 4;
  static constexpr int KC = 16;
  static __device__ __forceinline__ void run(f32x4& c, const u32x4& a, const u32x4& b) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
  }
};

// `valid` (possibly <= 0) elements of a lane's 16 bytes, `stride` elements apart, the rest 0
template <typename T, bool VEC>
__device__ __forceinline__ u32x4 frag(const T* p, int64_t stride, int valid) {
  constexpr int N = Mma<T>::N;
  if (VEC && valid >= N) return *reinterpret_cast<const u32x4*>(p);
  typedef T vec __attribute__((ext_vector_type(N)));
  vec v;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = e < valid ? p[e * stride] : (T)0.f;
  return __builtin_bit_cast(u32x4, v);
}

// ---- plan: rows in the order of their adapters ----------------------------------------------------
// Groups 0 .. k - 1: the adapters, k: rows without one (id -1), k + 1: ids out of range.  One workgroup
// per group counts the ids below its own and lists its own in ascending row order: no atomics.
constexpr int PT = 1024;

__global__ void __launch_bounds__(PT) plan_kernel(const int64_t* __restrict__ ids, int n, int k,
                                                  int* __restrict__ perm, int* __restrict__ sid, int* __restrict__ start) {
  __shared__ int red[2][PT / 64];
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto group = [&](int i) {
    const int64_t t = ids[i];
    return t == -1 ? k : (t < 0 || t >= k ? k + 1 : (int)t);
  };
  int less = 0, mine = 0;
  for (int i = tid; i < n; i += PT) {
    const int x = group(i);
    less += x < g;
    mine += x == g;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    less += __shfl_xor(less, off, 64);
    mine += __shfl_xor(mine, off, 64);
  }
  if (lane == 0) {
    red[0][wave] = less;
    red[1][wave] = mine;
  }
  __syncthreads();
  less = mine = 0;
  for (int w = 0; w < PT / 64; ++w) {
    less += red[0][w];
    mine += red[1][w];
  }
  if (tid == 0) {
    start[g] = less;
    if (g == k + 1) start[k + 2] = n;
  }
  if (mine == 0) return;  // the whole workgroup
  int at = less;
  for (int i0 = 0; i0 < n; i0 += PT) {
    __syncthreads();  // red of the previous round has been read
    const int i = i0 + tid;
    const bool is = i < n && group(i) == g;
    const uint64_t mask = __ballot(is);
    if (lane == 0) red[0][wave] = __popcll(mask);
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < PT / 64; ++w) {
      before += w < wave ? red[0][w] : 0;
      total += red[0][w];
    }
    if (is) {
      const int to = at + before + __popcll(mask & ((1ull << lane) - 1));
      perm[to] = i;
      sid[to] = g;
    }
    at += total;
  }
}

// Row chunks of `per` rows, each of one adapter: chunk c of adapter t has the slot
// start[t] / per + t + c (c < max(1, chunks of t)): distinct, and below n / per + k.
struct Chunk {
  int t, c, row0, rows, chunks;
};
__device__ __forceinline__ Chunk chunk_of(int slot, const int* start, int k, int per) {
  int lo = 0, hi = k - 1;  // the last t with start[t] / per + t <= slot
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] / per + mid <= slot)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int s0 = start[lo], s1 = start[lo + 1];
  Chunk ch;
  ch.t = lo;
  ch.c = slot - (s0 / per + lo);
  ch.chunks = max(1, (s1 - s0 + per - 1) / per);
  ch.row0 = s0 + ch.c * per;
  ch.rows = min(per, s1 - ch.row0);
  return ch;  // an unused slot has c >= chunks (or c < 0 before the first)
}

// ---- shrink: out[i, 0 .. r) = scale_t F_t v_i for the sorted rows i --------------------------------
// F_t element (rank q, column c) at f[t r cols + q fq + c fc].  grid: slots x rank blocks of 16 x splits
// of the columns (each split a slab of its own).
template <typename T, bool VV, bool FV>
__global__ void __launch_bounds__(256) shrink_kernel(const T* __restrict__ v, int64_t ldv, int n, int cols,
                                                     const T* __restrict__ f, int64_t fq, int64_t fc, int k, int r, int rp,
                                                     const float* __restrict__ scales, const int* __restrict__ perm,
                                                     const int* __restrict__ start, int per_split, float* __restrict__ out) {
  constexpr int N = Mma<T>::N, KC = Mma<T>::KC, UN = 4;
  __shared__ f32x4 part[4][64];
  const Chunk ch = chunk_of(blockIdx.x, start, k, 16);
  if (ch.c < 0 || ch.c >= ch.chunks || ch.rows <= 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fs = lane >> 4;
  const int q = blockIdx.y * 16 + fr;
  const int c_lo = blockIdx.z * per_split, c_hi = min(cols, c_lo + per_split);
  const T* vr = v + (int64_t)perm[ch.row0 + min(fr, ch.rows - 1)] * ldv;
  const T* fp = f + (int64_t)ch.t * r * cols + (int64_t)min(q, r - 1) * fq;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = c_lo + wave * KC; c0 < c_hi; c0 += 4 * KC * UN) {
    u32x4 a[UN], b[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int c = c0 + u * 4 * KC + fs * N;
      a[u] = frag<T, FV>(fp + (int64_t)c * fc, fc, c_hi - c);
      b[u] = frag<T, VV>(vr + c, 1, c_hi - c);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) Mma<T>::run(acc, a[u], b[u]);
  }
  part[wave][lane] = acc;
  __syncthreads();
  if (wave != 0 || fr >= ch.rows) return;
  const float sc = scales ? scales[ch.t] : 1.f;
  acc = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
  const int q0 = blockIdx.y * 16 + fs * 4;
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = q0 + e < r ? acc[e] * sc : 0.f;  // ranks up to rp are zeros
  float* o = out + (int64_t)blockIdx.z * n * rp + (int64_t)(ch.row0 + fr) * rp + q0;
  *reinterpret_cast<f32x4*>(o) = acc;
}

// slab 0 += slabs 1 .. splits - 1, in that order
__global__ void __launch_bounds__(256) slabs_kernel(f32x4* __restrict__ x, int64_t count, int splits) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  f32x4 a = x[i];
  for (int s = 1; s < splits; ++s) a += x[i + s * count];
  x[i] = a;
}

// ---- project: y[perm[i], :] = W x + F_t h_i -----------------------------------------------------------
// F_t element (column c, rank q) at f[t r m + c fc + q fq].
constexpr int BM = 128, BN = 128, BKB = 128;  // rows of x, rows of W, bytes of the summed axis per stage

// 16-byte slot of a 128-byte row, XOR-ed with the row: the 16 rows a fragment read touches then lie in
// eight different slots
__device__ __forceinline__ int lds_slot(int row, int slot) { return row * BKB + ((slot ^ (row & 7)) << 4); }

template <typename T>
__device__ __forceinline__ u32x4 h_frag(const float* h, int q0, int fs);
// fp32: ranks q0 + 4 fs .. of the row
template <>
__device__ __forceinline__ u32x4 h_frag<float>(const float* h, int q0, int fs) {
  return *reinterpret_cast<const u32x4*>(h + q0 + fs * 4);
}
// bf16: lane groups 0, 1 the hi parts of ranks q0 + 8 (fs & 1) .., groups 2, 3 the lo parts
template <>
__device__ __forceinline__ u32x4 h_frag<__bf16>(const float* h, int q0, int fs) {
  const float* p = h + q0 + (fs & 1) * 8;
  bf16x8 o;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    __bf16 hi, lo;
    split_bf16(p[e], hi, lo);
    o[e] = fs & 2 ? lo : hi;
  }
  return __builtin_bit_cast(u32x4, o);
}
// the ranks of F that meet them
template <typename T>
__device__ __forceinline__ int f_rank(int q0, int fs) {
  return sizeof(T) == 4 ? q0 + fs * 4 : q0 + (fs & 1) * 8;
}

template <typename T, bool XV, bool WV, bool FV>
__global__ void __launch_bounds__(256) project_kernel(const T* __restrict__ x, int64_t ldx, int n, int d,
                                                      const T* __restrict__ w, int64_t ldw, int m,
                                                      const T* __restrict__ f, int64_t fc, int64_t fq, int k, int r, int rp,
                                                      const float* __restrict__ h, const int* __restrict__ perm,
                                                      const int* __restrict__ sid, T* __restrict__ y, int64_t ldy,
                                                      int row_tiles, int yvec) {
  constexpr int N = Mma<T>::N, KE = BKB / sizeof(T), KC = Mma<T>::KC;
  __shared__ __attribute__((aligned(16))) unsigned char lds[2][(BM + BN) * BKB];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fs = lane >> 4;
  const int wr = wave >> 1, wc = wave & 1;
  const int tile = xcd_remap(blockIdx.x, gridDim.x);
  const int m0 = (tile / row_tiles) * BN, n0 = (tile % row_tiles) * BM;

  const T* src[8];
  int kt[8];  // unused columns of the piece's row are found from its first column
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int row = (tid >> 3) + (j & 3) * 32;
    if (j < 4) {
      const int i = min(n0 + row, n - 1);
      src[j] = x + (int64_t)perm[i] * ldx + (tid & 7) * N;
    } else {
      src[j] = w + (int64_t)min(m0 + row, m - 1) * ldw + (tid & 7) * N;
    }
    kt[j] = (tid & 7) * N;
  }
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  u32x4 reg[8];
  auto load = [&](int k0) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      reg[j] = j < 4 ? frag<T, XV>(src[j] + k0, 1, d - k0 - kt[j]) : frag<T, WV>(src[j] + k0, 1, d - k0 - kt[j]);
  };
  load(0);
  int buf = 0;
  for (int k0 = 0; k0 < d; k0 += KE) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int row = (tid >> 3) + (j & 3) * 32 + (j < 4 ? 0 : BM);
      *reinterpret_cast<u32x4*>(&lds[buf][lds_slot(row, tid & 7)]) = reg[j];
    }
    __syncthreads();
    if (k0 + KE < d) load(k0 + KE);
#pragma unroll
    for (int kc = 0; kc < KE / KC; ++kc) {
      u32x4 xa[4], wb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xa[i] = *reinterpret_cast<const u32x4*>(&lds[buf][lds_slot(wr * 64 + i * 16 + fr, kc * 4 + fs)]);
        wb[i] = *reinterpret_cast<const u32x4*>(&lds[buf][lds_slot(BM + wc * 64 + i * 16 + fr, kc * 4 + fs)]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) Mma<T>::run(acc[i][j], wb[j], xa[i]);
    }
    buf ^= 1;
  }

  // acc[i][j]: x row n0 + wr 64 + i 16 + fr, columns m0 + wc 64 + j 16 + 4 fs + reg
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = n0 + wr * 64 + i * 16 + fr;
    const bool live = row < n;
    const int t = live ? sid[row] : k;
    const float* hr = h + (int64_t)min(row, n - 1) * rp;
    unsigned todo = (unsigned)(__ballot(live && t < k) & 0xffffu);
    while (todo) {  // one adapter after the other (uniform over the wave)
      const int ta = __builtin_amdgcn_readlane(t, __builtin_ctz(todo));
      todo &= ~(unsigned)(__ballot(t == ta) & 0xffffu);
      const T* ft = f + (int64_t)ta * r * m;
      f32x4 add[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) add[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
      for (int q0 = 0; q0 < rp; q0 += 16) {
        const u32x4 hb = t == ta ? h_frag<T>(hr, q0, fs) : (u32x4){0u, 0u, 0u, 0u};
        const int q = f_rank<T>(q0, fs);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int col = min(m0 + wc * 64 + j * 16 + fr, m - 1);
          Mma<T>::run(add[j], frag<T, FV>(ft + (int64_t)col * fc + (int64_t)q * fq, fq, r - q), hb);
        }
      }
      if (t == ta) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += add[j];
      }
    }
    if (!live) continue;
    const float bad = t > k ? NAN : 0.f;  // an id out of range poisons its row
    T* yr = y + (int64_t)perm[row] * ldy;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = m0 + wc * 64 + j * 16 + fs * 4;
      typedef T out4 __attribute__((ext_vector_type(4)));
      out4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (T)(acc[i][j][e] + bad);
      if (yvec && c + 4 <= m) {
        *reinterpret_cast<out4*>(yr + c) = o;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < m) yr[c + e] = o[e];
      }
    }
  }
}

// ---- grads: out_t[q, c] = sum over the sorted rows i of adapter t of h[i, q] v[perm[i], c] -------------
// One wave: 16 ranks x 16 N columns (a lane's 16 bytes of a row of v feed N instructions); the four
// waves of a workgroup take every fourth group of four rows.  Adapters with more than `per` rows are cut into
// chunks that write fp32 slabs, summed afterwards in ascending order.  An adapter without rows gets zeros.
template <typename T, bool VV>
__global__ void __launch_bounds__(256) grads_kernel(const T* __restrict__ v, int64_t ldv, int n, int cols,
                                                    const float* __restrict__ h, int rp, int k, int r,
                                                    const int* __restrict__ perm, const int* __restrict__ start, int per,
                                                    T* __restrict__ out, int64_t oc, int64_t oq, float* __restrict__ slabs) {
  constexpr int N = Mma<T>::N;
  typedef T vec __attribute__((ext_vector_type(N)));
  __shared__ f32x4 part[3][N][64];
  const Chunk ch = chunk_of(blockIdx.x, start, k, per);
  if (ch.c < 0 || ch.c >= ch.chunks) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fs = lane >> 4;
  const int c0 = blockIdx.y * 16 * N + fr * N, q0 = blockIdx.z * 16;
  f32x4 acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int i = wave * 4; i < ch.rows; i += 16) {
    const bool in = i + fs < ch.rows;
    const int row = ch.row0 + min(i + fs, ch.rows - 1);
    const float hv = in ? h[(int64_t)row * rp + q0 + fr] : 0.f;
    const vec x = __builtin_bit_cast(vec, frag<T, VV>(v + (int64_t)perm[row] * ldv + c0, 1, in ? cols - c0 : 0));
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(hv, (float)x[j], acc[j], 0, 0, 0);
  }
  if (wave > 0)
#pragma unroll
    for (int j = 0; j < N; ++j) part[wave - 1][j][lane] = acc[j];
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = (acc[j] + part[0][j][lane]) + (part[1][j][lane] + part[2][j][lane]);
  // acc[j][e]: rank q0 + 4 fs + e, column c0 + j
  if (ch.chunks > 1) {
    float* sl = slabs + (int64_t)blockIdx.x * r * cols;  // [r][cols]
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (q0 + fs * 4 + e < r && c0 + j < cols) sl[(int64_t)(q0 + fs * 4 + e) * cols + c0 + j] = acc[j][e];
    return;
  }
  T* o = out + (int64_t)ch.t * r * cols;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (q0 + fs * 4 + e < r && c0 + j < cols) o[(int64_t)(c0 + j) * oc + (int64_t)(q0 + fs * 4 + e) * oq] = (T)acc[j][e];
}

template <typename T>
__global__ void __launch_bounds__(256) grads_join_kernel(const float* __restrict__ slabs, const int* __restrict__ start,
                                                         int per, int cols, int r, T* __restrict__ out, int64_t oc,
                                                         int64_t oq) {
  const int t = blockIdx.x;
  const int s0 = start[t], chunks = (start[t + 1] - s0 + per - 1) / per;
  if (chunks <= 1) return;
  const int64_t size = (int64_t)r * cols, slot = s0 / per + t;
  for (int64_t i = (int64_t)blockIdx.y * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.y * 256) {
    float a = 0.f;
    for (int c = 0; c < chunks; ++c) a += slabs[(slot + c) * size + i];
    const int64_t q = i / cols, col = i - q * cols;
    out[t * size + col * oc + q * oq] = (T)a;
  }
}

// dst [cols, ldd] = src [rows, lds] transposed, 32 x 32 tiles
template <typename T>
__global__ void __launch_bounds__(256) transpose_kernel(const T* __restrict__ src, int64_t lds_, int rows, int cols,
                                                        T* __restrict__ dst, int64_t ldd) {
  __shared__ T tile[32][33];
  const int c0 = blockIdx.x * 32, r0 = blockIdx.y * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int i = ty; i < 32; i += 8)
    if (r0 + i < rows && c0 + tx < cols) tile[i][tx] = src[(int64_t)(r0 + i) * lds_ + c0 + tx];
  __syncthreads();
  for (int i = ty; i < 32; i += 8)
    if (c0 + i < cols && r0 + tx < rows) dst[(int64_t)(c0 + i) * ldd + r0 + tx] = tile[tx][i];
}

// ---- host side --------------------------------------------------------------------------------------------

int elem_size(int dtype) { return dtype == KGE_DT_F32 ? 4 : 2; }
bool dtype_ok(int dtype) { return dtype == KGE_DT_F32 || dtype == KGE_DT_BF16; }
bool vec_rows(const void* p, int64_t ld, int es) { return aligned16(p) && ld * es % 16 == 0; }
bool ld_ok(int64_t ld, int64_t rows, int64_t cols) { return rows <= 1 || ld >= cols; }
constexpr int64_t MAX_N = (int64_t)1 << 30;
int64_t rank_pad(int64_t r) { return (r + 15) / 16 * 16; }

template <typename F>
int by_type(int dtype, F f) {
  return dtype == KGE_DT_F32 ? f((float*)nullptr) : f((__bf16*)nullptr);
}
template <typename F>
int by_bool(bool b, F f) {
  return b ? f(std::true_type{}) : f(std::false_type{});
}

// Splits of the summed columns of shrink: enough workgroups for two per CU where the rows' slots leave
// CUs idle, at least 1024 columns each.
int shrink_splits(int64_t n, int64_t cols, int64_t k, int64_t rp) {
  const int64_t groups = (std::min<int64_t>(n / 16 + k, n) + 1) * (rp / 16);
  const int64_t want = (2 * kge_num_cus() + groups - 1) / groups, most = std::max<int64_t>(1, cols / 1024);
  return (int)std::max<int64_t>(1, std::min(want, most));
}

// Rows of one chunk of grads: a multiple of 64, so that the launch has about 2048 workgroups
int64_t grads_per(int64_t n, int64_t cols, int64_t k, int64_t r, int es) {
  const int64_t blocks = ((cols * es + 255) / 256) * (rank_pad(r) / 16);
  const int64_t chunks = std::max<int64_t>(1, 2048 / blocks);
  return std::max<int64_t>(64, ((n + chunks - 1) / chunks + 63) / 64 * 64);
}

}  // namespace

extern "C" int kge_adapter_plan(const int64_t* ids, int64_t n, int64_t k, int32_t* perm, int32_t* sid, int32_t* start,
                                void* stream) {
  KGE_REQUIRE(n >= 0 && n <= MAX_N && k >= 1 && k <= (1 << 20) && start && (n == 0 || (ids && perm && sid)));
  plan_kernel<<<dim3((unsigned)(k + 2)), dim3(PT), 0, as_stream(stream)>>>(ids, (int)n, (int)k, perm, sid, start);
  KGE_CHECK_LAUNCH();
  return 0;
}

extern "C" int64_t kge_adapter_shrink_rows(int64_t n, int64_t cols, int64_t k, int64_t r) {
  if (n < 0 || cols < 1 || k < 1 || r < 1) return 0;
  return n * shrink_splits(n, cols, k, rank_pad(r));
}

extern "C" int kge_adapter_shrink(const void* v, int dtype, int64_t ldv, int64_t n, int64_t cols, const void* f,
                                  int f_by_rank, int64_t k, int64_t r, const float* scales, const int32_t* perm,
                                  const int32_t* start, float* out, int64_t out_rows, void* stream) {
  KGE_REQUIRE(dtype_ok(dtype) && n >= 0 && n <= MAX_N && cols >= 1 && cols <= MAX_N && k >= 1 && k <= (1 << 20) && r >= 1 &&
              r <= 1024 && ld_ok(ldv, n, cols));
  if (n == 0) return 0;
  const int es = elem_size(dtype), rp = (int)rank_pad(r);
  const int splits = shrink_splits(n, cols, k, rp);
  KGE_REQUIRE(v && f && perm && start && out && aligned16(out) && out_rows >= n * splits);
  const int64_t per_split = ((cols + splits - 1) / splits + 127) / 128 * 128;
  const int64_t fq = f_by_rank ? cols : 1, fc = f_by_rank ? 1 : r;
  const dim3 grid((unsigned)(n / 16 + k), (unsigned)(rp / 16), (unsigned)splits);
  int rc = by_type(dtype, [&](auto* tag) {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    return by_bool(vec_rows(v, ldv, es), [&](auto vv) {
      return by_bool(f_by_rank && vec_rows(f, cols, es), [&](auto fv) -> int {
        shrink_kernel<T, vv.value, fv.value><<<grid, dim3(256), 0, as_stream(stream)>>>(
            (const T*)v, ldv, (int)n, (int)cols, (const T*)f, fq, fc, (int)k, (int)r, rp, scales, perm, start,
            (int)per_split, out);
        KGE_CHECK_LAUNCH();
        return 0;
      });
    });
  });
  if (rc || splits == 1) return rc;
  const int64_t count = n * rp / 4;
  slabs_kernel<<<dim3((unsigned)((count + 255) / 256)), dim3(256), 0, as_stream(stream)>>>((f32x4*)out, count, splits);
  KGE_CHECK_LAUNCH();
  return 0;
}

extern "C" int kge_adapter_project(const void* x, int dtype, int64_t ldx, int64_t n, int64_t d, const void* w, int64_t ldw,
                                   int64_t m, const void* f, int f_by_rank, int64_t k, int64_t r, const float* h,
                                   const int32_t* perm, const int32_t* sid, void* y, int64_t ldy, void* stream) {
  KGE_REQUIRE(dtype_ok(dtype) && n >= 0 && n <= MAX_N && d >= 1 && d <= MAX_N && m >= 1 && m <= MAX_N && k >= 1 &&
              k <= (1 << 20) && r >= 1 && r <= 1024 && ld_ok(ldx, n, d) && ld_ok(ldw, m, d) && ld_ok(ldy, n, m));
  if (n == 0) return 0;
  const int es = elem_size(dtype), rp = (int)rank_pad(r);
  KGE_REQUIRE(x && w && f && h && perm && sid && y && aligned16(h));
  const int64_t fc = f_by_rank ? 1 : r, fq = f_by_rank ? m : 1;
  const int64_t row_tiles = (n + BM - 1) / BM, tiles = row_tiles * ((m + BN - 1) / BN);
  KGE_REQUIRE(tiles < ((int64_t)1 << 31));
  const int yvec = (reinterpret_cast<uintptr_t>(y) % (4 * es)) == 0 && ldy % 4 == 0;
  return by_type(dtype, [&](auto* tag) {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    return by_bool(vec_rows(x, ldx, es), [&](auto xv) {
      return by_bool(vec_rows(w, ldw, es), [&](auto wv) {
        return by_bool(!f_by_rank && vec_rows(f, r, es), [&](auto fv) -> int {
          project_kernel<T, xv.value, wv.value, fv.value><<<dim3((unsigned)tiles), dim3(256), 0, as_stream(stream)>>>(
              (const T*)x, ldx, (int)n, (int)d, (const T*)w, ldw, (int)m, (const T*)f, fc, fq, (int)k, (int)r, rp, h, perm,
              sid, (T*)y, ldy, (int)row_tiles, yvec);
          KGE_CHECK_LAUNCH();
          return 0;
        });
      });
    });
  });
}

extern "C" int64_t kge_adapter_grads_ws_size(int64_t n, int64_t cols, int64_t k, int64_t r, int dtype) {
  if (n < 0 || cols < 1 || k < 1 || r < 1 || !dtype_ok(dtype)) return 0;
  const int64_t per = grads_per(n, cols, k, r, elem_size(dtype));
  return n <= per ? 0 : (n / per + k) * r * cols;
}

extern "C" int kge_adapter_grads(const void* v, int dtype, int64_t ldv, int64_t n, int64_t cols, const float* h, int64_t k,
                                 int64_t r, const int32_t* perm, const int32_t* start, void* out, int out_by_rank, float* ws,
                                 int64_t ws_elems, void* stream) {
  KGE_REQUIRE(dtype_ok(dtype) && n >= 0 && n <= MAX_N && cols >= 1 && cols <= MAX_N && k >= 1 && k <= (1 << 20) && r >= 1 &&
              r <= 1024 && ld_ok(ldv, n, cols) && start && out && (n == 0 || (v && h && perm)));
  const int es = elem_size(dtype), rp = (int)rank_pad(r);
  const int64_t per = grads_per(n, cols, k, r, es);
  const bool join = n > per;
  KGE_REQUIRE(!join || (ws && ws_elems >= (n / per + k) * r * cols));
  const int64_t oc = out_by_rank ? 1 : r, oq = out_by_rank ? cols : 1;
  const int64_t col_blocks = (cols * es + 255) / 256;
  KGE_REQUIRE(col_blocks <= 65535);
  return by_type(dtype, [&](auto* tag) {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    int rc = by_bool(n > 0 && vec_rows(v, ldv, es), [&](auto vv) -> int {
      grads_kernel<T, vv.value><<<dim3((unsigned)(n / per + k), (unsigned)col_blocks, (unsigned)(rp / 16)), dim3(256), 0,
                                  as_stream(stream)>>>((const T*)v, ldv, (int)n, (int)cols, h, rp, (int)k, (int)r, perm,
                                                       start, (int)per, (T*)out, oc, oq, ws);
      KGE_CHECK_LAUNCH();
      return 0;
    });
    if (rc || !join) return rc;
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((r * cols + 1023) / 1024, 64));
    grads_join_kernel<T><<<dim3((unsigned)k, (unsigned)blocks), dim3(256), 0, as_stream(stream)>>>(
        ws, start, (int)per, (int)cols, (int)r, (T*)out, oc, oq);
    KGE_CHECK_LAUNCH();
    return 0;
  });
}

extern "C" int kge_transpose(const void* src, int dtype, int64_t lds, int64_t rows, int64_t cols, void* dst, int64_t ldd,
                             void* stream) {
  KGE_REQUIRE(dtype_ok(dtype) && rows >= 0 && cols >= 0 && rows <= MAX_N && cols <= MAX_N && ld_ok(lds, rows, cols) &&
              ld_ok(ldd, cols, rows));
  if (rows == 0 || cols == 0) return 0;
  const int64_t bx = (cols + 31) / 32, by = (rows + 31) / 32;
  KGE_REQUIRE(src && dst && by <= 65535 * (int64_t)1024);
  return by_type(dtype, [&](auto* tag) -> int {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    // the y dimension of a grid is limited: bands of rows
    for (int64_t b = 0; b < by; b += 65535) {
      const int64_t r0 = b * 32, nr = std::min<int64_t>(rows - r0, 65535 * (int64_t)32);
      transpose_kernel<T><<<dim3((unsigned)bx, (unsigned)((nr + 31) / 32)), dim3(256), 0, as_stream(stream)>>>(
          (const T*)src + r0 * lds, lds, (int)nr, (int)cols, (T*)dst + r0, ldd);
      KGE_CHECK_LAUNCH();
    }
    return 0;
  });
}
