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
// The rows are worked on in the order of their adapters (plan: a stable counting sort of the ids, a radix sort
// where there are many), so that an adapter is read for 16 of its rows at a time; rows are gathered and scattered
// through the order, never copied.  After it:
//   shrink   h (and u): [<= 16 rows of one adapter] x [d] x [r], the four waves of a workgroup split d
//   project  W x + B h: a tiled product whose epilogue adds B_t h for every adapter among a fragment's 16
//            rows, h of the other rows masked to 0; a slice of B_t with infinities or NaN, whose products with 0
//            would be NaN, is selected into its own rows instead: it cannot reach another request's row.  Long sums for
//            few results are split over workgroups (split_join adds them up in order).
//   grads    dA / dB: [r] x [rows of one adapter] x [columns] on the fp32 matrix instruction whatever the
//            type (its operands hold one value per lane along the summed axis, so rows need no transpose)
// h and u are kept in fp32; where they meet a bf16 B_t on the bf16 instruction they are split into hi + lo
// (2^-16), both halves in one instruction: 16 ranks fill half of its 32-wide summed axis.
#include <math.h>

#include <initializer_list>
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

// A lane's 16 bytes: elements off .. of a row of len, zeros from len on (off may lie beyond it).  No branches: a
// batch of them is in flight together (guarded by branches, each load waits for the one before: the compiler drains
// the loads where the paths meet).  EVEN: len and off are multiples of N, a fragment lies inside or outside.  Rows need
// no alignment beyond their elements' own: the hardware splits a load that crosses a line.
template <typename T, bool EVEN>
__device__ __forceinline__ u32x4 frag(const T* row, int off, int len) {
  constexpr int N = Mma<T>::N;
  u32x4 v;
  if (EVEN) {
    const bool in = off < len;
    __builtin_memcpy(&v, row + (in ? off : 0), 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = in ? v[e] : 0u;
    return v;
  }
  if (len >= N) {  // the row's last N elements where the fragment crosses its end, shifted down
    const int at = min(off, len - N), s = min(off - at, N) * (int)sizeof(T) * 8;
    uint64_t q[2];
    __builtin_memcpy(q, row + at, 16);
    const uint64_t low = s < 64 ? (q[0] >> s) | (s ? q[1] << (64 - s) : 0) : (s < 128 ? q[1] >> (s - 64) : 0);
    const uint64_t high = s < 64 ? q[1] >> s : 0;
    v[0] = (unsigned)low;
    v[1] = (unsigned)(low >> 32);
    v[2] = (unsigned)high;
    v[3] = (unsigned)(high >> 32);
    return v;
  }
  typedef T vec __attribute__((ext_vector_type(N)));
  vec x;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const T z = row[min(off + e, len - 1)];
    x[e] = off + e < len ? z : (T)0.f;
  }
  return __builtin_bit_cast(u32x4, x);
}
// elements off, off + 1, .. of a column: `stride` apart in memory
template <typename T>
__device__ __forceinline__ u32x4 frag_strided(const T* col, int64_t stride, int off, int len) {
  constexpr int N = Mma<T>::N;
  typedef T vec __attribute__((ext_vector_type(N)));
  vec v;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const T z = col[min(off + e, len - 1) * stride];
    v[e] = off + e < len ? z : (T)0.f;
  }
  return __builtin_bit_cast(u32x4, v);
}

// ---- plan: rows in the order of their adapters ----------------------------------------------------
// Groups 0 .. k - 1: the adapters, k: rows without one (id -1), k + 1: ids out of range.  One workgroup
// per group counts the ids below its own and lists its own in ascending row order: no atomics.  PU ids per
// thread are in flight at once; a batch of up to PT PU rows is read once.
constexpr int PT = 1024, PU = 8;

__device__ __forceinline__ void plan_group(int g, const int64_t* __restrict__ ids, int n, int k, int* __restrict__ perm,
                                           int* __restrict__ sid, int* __restrict__ start) {
  __shared__ int red[2][PT / 64], count[PU][PT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int x[PU];
  auto load = [&](int i0) {
    int64_t v[PU];
#pragma unroll
    for (int u = 0; u < PU; ++u) v[u] = i0 + u * PT < n ? ids[min(i0 + u * PT + tid, n - 1)] : 0;
#pragma unroll
    for (int u = 0; u < PU; ++u) {
      const int in = v[u] == -1 ? k : (v[u] < 0 || v[u] >= k ? k + 1 : (int)v[u]);
      x[u] = i0 + u * PT + tid < n ? in : k + 2;
    }
  };
  int less = 0, mine = 0;
  for (int i0 = 0; i0 < n; i0 += PT * PU) {
    load(i0);
#pragma unroll
    for (int u = 0; u < PU; ++u) {
      less += x[u] < g;
      mine += x[u] == g;
    }
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
#pragma unroll
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
  for (int i0 = 0; i0 < n; i0 += PT * PU) {
    if (n > PT * PU) load(i0);
    __syncthreads();  // count of the previous round has been read
    uint64_t mask[PU];
#pragma unroll
    for (int u = 0; u < PU; ++u) {
      mask[u] = __ballot(x[u] == g);
      if (lane == 0) count[u][wave] = __popcll(mask[u]);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < PU; ++u) {
      if (i0 + u * PT >= n) break;
      int before = 0, total = 0;
#pragma unroll
      for (int w = 0; w < PT / 64; ++w) {
        before += w < wave ? count[u][w] : 0;
        total += count[u][w];
      }
      if (x[u] == g) {
        const int to = at + before + __popcll(mask[u] & ((1ull << lane) - 1));
        perm[to] = i0 + u * PT + tid;
        sid[to] = g;
      }
      at += total;
    }
  }
}

// ---- plan of many rows: a stable radix sort by group --------------------------------------------------------
// The plan above reads every id once per group.  Beyond SORT_FROM reads the order comes from one pass (two from 2048
// groups on) over digits of 11 bits: each wave counts the digits of its own rows (sort_count), the counts of a digit
// are summed over the waves in order (sort_scan), and each wave puts its rows where the sums say, equal digits within
// 64 rows in row order by ballots (sort_put): no global atomics, the same order as above.
constexpr int DIGIT = 11, BINS = 1 << DIGIT;

__device__ __forceinline__ int group_of(int64_t v, int k) { return v == -1 ? k : (v < 0 || v >= k ? k + 1 : (int)v); }

__global__ void __launch_bounds__(64) sort_count_kernel(const int64_t* __restrict__ ids, int n, int k, const int* __restrict__ src,
                                                        int shift, int bins, int rows, int* __restrict__ counts) {
  __shared__ int count[BINS];
  const int lane = threadIdx.x;
  const int64_t lo = (int64_t)blockIdx.x * rows, hi = lo + rows < n ? lo + rows : n;
  for (int b = lane; b < bins; b += 64) count[b] = 0;
  __syncthreads();
  for (int64_t i = lo + lane; i < hi; i += 64)
    atomicAdd(&count[(group_of(ids[src ? src[i] : i], k) >> shift) & (BINS - 1)], 1);  // (in LDS; a count has no order)
  __syncthreads();
  for (int b = lane; b < bins; b += 64) counts[(int64_t)b * gridDim.x + blockIdx.x] = count[b];
}

// exclusive sum over a wave; total in every lane
__device__ __forceinline__ int wave_before(int v, int lane, int& total) {
  int x = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off, 64);
    x += lane >= off ? y : 0;
  }
  total = __shfl(x, 63, 64);
  return x - v;
}

// one wave per digit
__global__ void __launch_bounds__(64) sort_scan_kernel(int* __restrict__ counts, int blocks, int* __restrict__ totals) {
  const int lane = threadIdx.x;
  int* c = counts + (int64_t)blockIdx.x * blocks;
  int before = 0;
  for (int b0 = 0; b0 < blocks; b0 += 64) {
    const int v = b0 + lane < blocks ? c[b0 + lane] : 0;
    int total;
    const int x = wave_before(v, lane, total);
    if (b0 + lane < blocks) c[b0 + lane] = before + x;
    before += total;
  }
  if (lane == 0) totals[blockIdx.x] = before;
}

// sid: written by the last pass
__global__ void __launch_bounds__(64) sort_put_kernel(const int64_t* __restrict__ ids, int n, int k, const int* __restrict__ src,
                                                      int shift, int bins, int rows, const int* __restrict__ counts,
                                                      const int* __restrict__ totals, int* __restrict__ dst,
                                                      int* __restrict__ sid) {
  __shared__ int next[BINS];
  const int lane = threadIdx.x;
  const int64_t lo = (int64_t)blockIdx.x * rows, hi = lo + rows < n ? lo + rows : n;
  int before = 0;
  for (int b0 = 0; b0 < bins; b0 += 64) {
    const int b = b0 + lane;
    int total;
    const int x = wave_before(b < bins ? totals[b] : 0, lane, total);
    if (b < bins) next[b] = before + x + counts[(int64_t)b * gridDim.x + blockIdx.x];
    before += total;
  }
  __syncthreads();
  for (int64_t i0 = lo; i0 < hi; i0 += 64) {
    const bool in = i0 + lane < hi;
    const int row = in ? (src ? src[i0 + lane] : (int)(i0 + lane)) : 0;
    const int g = in ? group_of(ids[row], k) : 0, digit = (g >> shift) & (BINS - 1);
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < DIGIT; ++b) {
      const bool one = (digit >> b) & 1;
      const uint64_t ones = __ballot(one);
      same &= one ? ones : ~ones;
    }
    const uint64_t below = same & ((1ull << lane) - 1);
    const int to = next[digit] + __popcll(below);
    __syncthreads();  // every lane has read
    if (in && below == 0) next[digit] += __popcll(same);
    __syncthreads();
    if (in) {
      dst[to] = row;
      if (sid) sid[to] = g;
    }
  }
}

// start[g]: the first place whose group is g or above
__global__ void __launch_bounds__(256) sort_start_kernel(const int* __restrict__ sid, int n, int groups, int* __restrict__ start) {
  const int g = blockIdx.x * 256 + threadIdx.x;
  if (g > groups) return;
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (sid[mid] < g)
      lo = mid + 1;
    else
      hi = mid;
  }
  start[g] = lo;
}

// ---- h of one row, 16 ranks, columns [c_lo, c_hi), by one wave ------------------------------------------------
// The matrix instruction with the same row in all 16 places does the sums; put(q, value) for q < 16 (0 from r on).
// at: the ranks' rows of A_t, ld apart.
template <typename T, bool EVEN, typename F>
__device__ __forceinline__ void h_row(const T* __restrict__ xr, const T* __restrict__ at, int c_lo, int c_hi, int64_t ld, int r,
                                      float sc, int lane, F put) {
  constexpr int N = Mma<T>::N, KC = Mma<T>::KC, U = 4;
  const int fr = lane & 15, fs = lane >> 4;
  const T* ap = at + min(fr, r - 1) * ld;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = c_lo; c0 < c_hi; c0 += KC * U) {
    u32x4 a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * KC + fs * N;
      a[u] = frag<T, EVEN>(ap, c, c_hi);
      b[u] = frag<T, EVEN>(xr, c, c_hi);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) Mma<T>::run(acc, a[u], b[u]);
  }
  if (fr == 0)
#pragma unroll
    for (int e = 0; e < 4; ++e) put(fs * 4 + e, fs * 4 + e < r ? acc[e] * sc : 0.f);
}

// Workgroups 0 .. groups - 1: the plan; the others: h of four rows each, a quarter of the summed axis per wave (no
// plan needed).  One launch for both: at 1024 rows, 64 adapters and d = 512 two took 5.3 + 4.9 us.
template <typename T, bool EVEN>
__global__ void __launch_bounds__(PT) plan_h_kernel(const int64_t* __restrict__ ids, int n, int k, int* __restrict__ perm,
                                                    int* __restrict__ sid, int* __restrict__ start, int groups,
                                                    const T* __restrict__ x, int64_t ldx, int d, const T* __restrict__ a, int r,
                                                    int rp, const float* __restrict__ scales, float* __restrict__ h) {
  __shared__ float part[PT / 64][16];
  if ((int)blockIdx.x < groups) {
    plan_group(blockIdx.x, ids, n, k, perm, sid, start);
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quarter = wave & 3;
  const int64_t row = (int64_t)(blockIdx.x - groups) * 4 + (wave >> 2);
  const int64_t t = row < n ? ids[row] : -1;
  const bool live = t >= 0 && t < k;
  const int each = (d + 4 * Mma<T>::KC - 1) / (4 * Mma<T>::KC) * Mma<T>::KC, c0 = quarter * each;
  for (int q0 = 0; q0 < rp; q0 += 16) {
    if (live)
      h_row<T, EVEN>(x + row * ldx, a + (t * r + q0) * d, c0, min(d, c0 + each), d, min(16, r - q0), 1.f, lane,
               [&](int q, float v) { part[wave][q] = v; });
    __syncthreads();
    if (live && quarter == 0 && lane < 16)
      h[row * rp + q0 + lane] = ((part[wave][lane] + part[wave + 1][lane]) + (part[wave + 2][lane] + part[wave + 3][lane])) *
                                (scales ? scales[t] : 1.f);
    if (q0 + 16 < rp) __syncthreads();
  }
}

// Row chunks of `per` rows, each of one adapter: chunk c of adapter t has the slot
// start[t] / per + t + c (c < max(1, chunks of t)): distinct, and below n / per + k.
struct Chunk {
  int t, c, row0, rows, chunks;
};
__device__ __forceinline__ Chunk chunk_of(int slot, const int* start, int k, int per) {
  // the last t with start[t] / per + t <= slot, 64 candidates at a time (two rounds up to 4096 adapters)
  int lo = 0, hi = k - 1;
  while (hi > lo) {
    const int step = (hi - lo + 64) >> 6, t = lo + (int)(threadIdx.x & 63) * step;
    const bool ok = t <= hi && start[min(t, k - 1)] / per + t <= slot;
    lo += (__popcll(__ballot(ok)) - 1) * step;
    hi = min(hi, lo + step - 1);
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

// ---- shrink: out[i, 0 .. rp) = scale_t F_t v_i for every row i of an adapter ----------------------------
// F_t as [r, cols] (BY_RANK) or [cols, r].  grid: slots x rank blocks of 16 x splits of the columns (each
// split a slab of its own).  128 columns per wave on their way: in bf16 256 took 16.6 against 12.2 us for u of 1024 x
// 14560 (32 adapters of rank 8).  fp32: 25 us there for 75 MB (3 TB/s), half of its loads the 4-byte ones of F's columns.
template <typename T, bool BY_RANK, bool EVEN>
__global__ void __launch_bounds__(256) shrink_kernel(const T* __restrict__ v, int64_t ldv, int n, int cols,
                                                     const T* __restrict__ f, int k, int r, int rp,
                                                     const float* __restrict__ scales, const int* __restrict__ perm,
                                                     const int* __restrict__ start, int per_split, float* __restrict__ out) {
  constexpr int N = Mma<T>::N, KC = Mma<T>::KC, UN = 128 / KC;
  __shared__ f32x4 part[4][64];
  const Chunk ch = chunk_of(blockIdx.x, start, k, 16);
  if (ch.c < 0 || ch.c >= ch.chunks || ch.rows <= 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fs = lane >> 4;
  const int q = blockIdx.y * 16 + fr;
  const int c_lo = blockIdx.z * per_split, c_hi = min(cols, c_lo + per_split);
  const int row = perm[ch.row0 + min(fr, ch.rows - 1)];
  const T* vr = v + (int64_t)row * ldv;
  const T* fp = f + (int64_t)ch.t * r * cols + (int64_t)min(q, r - 1) * (BY_RANK ? cols : 1);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = c_lo + wave * KC; c0 < c_hi; c0 += 4 * KC * UN) {
    u32x4 a[UN], b[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int c = c0 + u * 4 * KC + fs * N;
      a[u] = BY_RANK ? frag<T, EVEN>(fp, c, c_hi) : frag_strided<T>(fp, r, c, c_hi);
      b[u] = frag<T, EVEN>(vr, c, c_hi);
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
  float* o = out + (int64_t)blockIdx.z * n * rp + (int64_t)row * rp + q0;
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
// F_t as [m, r].  128 x 128 tiles (rows of x, rows of W), four waves of 64 x 64, one 32-KiB LDS stage of 128 bytes of the summed axis
// (fp32: two); the next stage waits in registers.  One stage instead of two lets three workgroups share a CU, whose
// phases (loads, products, adapters, stores) overlap: with the short summed axes of embedding tables (512: 8 stages)
// a bf16 tile is latency, not MFMA time.  The slices of eight adapters at a time come into registers behind the last
// stage's products and go to where the stage was.
// 1024 x 14541 x 512, bf16: 30 us without adapters (the traffic of W, x and y needs 9, the products 6), 47 us with 64
// adapters of rank 16 (30 MB more); fp32: 159 us (96 TFLOP/s) and 172 us with 32 of rank 8.  Tried and slower: all of
// x's rows of a workgroup in LDS with W straight into registers (32 / 50 us), a walk over tiles by as many workgroups
// as fit (spills), slices straight into registers (33 / 49 us), sixteen slices at a time from the first stage on (31 /
// 47 us), two stages on their way in registers (33 / 49 us): loads, LDS reads and products need 6 us each and take turns.
constexpr int BKB = 128;  // bytes of the summed axis per stage

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
    o[e] = fs & 2 ? (isfinite(p[e] - (float)hi) ? lo : (__bf16)0.f) : hi;  // (an infinity has no rest)
  }
  return __builtin_bit_cast(u32x4, o);
}

// Adapter slices in LDS: 16 ranks of BN columns, [column][16 ranks].
template <typename T, int BN>
struct Slice {
  static constexpr int ROW = 16 * sizeof(T), BYTES = BN * ROW;
  // where a lane's part of column `col` starts: the ranks its h fragment holds
  static __device__ __forceinline__ int at(int col, int fs) {
    return col * ROW + (sizeof(T) == 4 ? fs : (fs & 1)) * 16;
  }
};
__device__ __forceinline__ bool nonfinite(const u32x4& v, float) {
  bool b = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) b |= (v[e] & 0x7f800000u) == 0x7f800000u;
  return b;
}
__device__ __forceinline__ bool nonfinite(const u32x4& v, __bf16) {
  bool b = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) b |= (v[e] & 0x7f800000u) == 0x7f800000u || (v[e] & 0x7f80u) == 0x7f80u;
  return b;
}

// A thread's 16-byte pieces of one slice: ranks [q0, q0 + 16) of columns [m0, m0 + BN) of an adapter.
template <typename T, int BN, bool EVEN>
struct Piece {
  static constexpr int N = Mma<T>::N, P = 16 / N, IT = (BN * P + 255) / 256;  // pieces per column, per thread

  static __device__ __forceinline__ u32x4 load(const T* ft, int m, int r, int m0, int q0, int it) {
    const int piece = it * 256 + threadIdx.x;
    return frag<T, EVEN>(ft + (int64_t)min(m0 + piece / P, m - 1) * r, q0 + piece % P * N, r);
  }
  static __device__ __forceinline__ void store(unsigned char* to, int it, const u32x4& v) {
    const int piece = it * 256 + threadIdx.x;
    if (piece < BN * P) *reinterpret_cast<u32x4*>(to + piece / P * Slice<T, BN>::ROW + piece % P * 16) = v;
  }
};

// BM 128: the tile above; BM 64: half of its rows, where 128-row tiles leave CUs without work.
// bf16: three workgroups per CU (87 us against two's 92 at 1024 x 14541 x 2048); fragments of odd ranks need the
// registers of two, or they spill.
// BN 64: for at most 64 columns (dx of short queries), all four waves along the rows (a backward pass for dx of 4096 x 32
// from 40000 columns in fp32: 461 us, 657 with tiles of 128).
// SPLIT: `per` elements of the summed axis per workgroup (blockIdx.y), the sums into slabs [split][n][m] of fp32, the
// adapters into the first one's; split_join_kernel adds them up.
template <typename T, int BM, int BN, int STAGES, bool EVEN, bool SPLIT>
__global__ void __launch_bounds__(256, STAGES == 2 || !EVEN ? 2 : 3)
    project_kernel(const T* __restrict__ x, int64_t ldx, int n, int d, const T* __restrict__ w, int64_t ldw, int m,
                   const T* __restrict__ f, int k, int r, int rp, const float* __restrict__ h, const int* __restrict__ perm,
                   const int* __restrict__ sid, T* __restrict__ y, int64_t ldy, int row_tiles, int yvec, int per,
                   float* __restrict__ slabs) {
  constexpr int N = Mma<T>::N, KE = BKB / sizeof(T), KC = Mma<T>::KC;
  constexpr int WC = BN / 64, RW = BM * WC / 4, TM = RW / 16;  // waves along the columns; rows, 16-row fragments per wave
  constexpr int XP = BM / 32, WP = BN / 32;  // pieces of x and of W per thread and stage
  constexpr int STAGE = (BM + BN) * BKB, LDS = STAGES * STAGE > 32768 ? STAGES * STAGE : 32768;
  using PC = Piece<T, BN, EVEN>;
  constexpr int COUNT = 8 / PC::IT;  // slices in LDS (and in registers, on their way) at a time: 32 KiB
  static_assert(COUNT * Slice<T, BN>::BYTES <= LDS, "slices");
  __shared__ __attribute__((aligned(16))) unsigned char lds[LDS];
  __shared__ int owner[BM];
  const int tid = threadIdx.x, lane = tid & 63, fr = lane & 15, fs = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave / WC, wc = wave % WC;
  const int tile = xcd_remap(blockIdx.x, gridDim.x);
  const int m0 = (tile / row_tiles) * BN, n0 = (tile % row_tiles) * BM;
  const int lo = SPLIT ? blockIdx.y * per : 0, hi = SPLIT ? min(d, lo + per) : d;

  const T* src[XP + WP];
  const int kt = (tid & 7) * N;  // first column of this thread's pieces within a stage
#pragma unroll
  for (int j = 0; j < XP + WP; ++j) {
    const int row = (tid >> 3) + j * 32;
    if (j < XP)
      src[j] = x + (int64_t)perm[min(n0 + row, n - 1)] * ldx + kt;
    else
      src[j] = w + (int64_t)min(m0 + row - BM, m - 1) * ldw + kt;
  }
  u32x4 reg[8];
  auto load = [&](int k0) {  // a whole stage
#pragma unroll
    for (int j = 0; j < XP + WP; ++j) __builtin_memcpy(&reg[j], src[j] + k0, 16);
  };
  if (lo + KE <= hi) load(lo);

  // The tile's adapters: sorted rows, so each is a run; slot = its number within the tile (-1: no adapter).
  const int t_lo = n0 + lane < n ? sid[n0 + lane] : k;
  const int t_hi = BM == 128 && n0 + 64 + lane < n ? sid[n0 + 64 + lane] : k;
  const int p_lo = __shfl_up(t_lo, 1, 64), p_hi = __shfl_up(t_hi, 1, 64), mid = __shfl(t_lo, 63, 64);
  const uint64_t b_lo = __ballot(t_lo < k && (lane == 0 || p_lo != t_lo));
  const uint64_t b_hi = __ballot(t_hi < k && (lane == 0 ? mid : p_hi) != t_hi);
  const uint64_t upto = lane == 63 ? ~0ull : (2ull << lane) - 1;
  const int slot_lo = t_lo < k ? __popcll(b_lo & upto) - 1 : -1;
  const int slot_hi = t_hi < k ? __popcll(b_lo) + __popcll(b_hi & upto) - 1 : -1;
  const int slots = SPLIT && blockIdx.y > 0 ? 0 : __popcll(b_lo) + __popcll(b_hi);
  if (wave == 0) {
    if ((b_lo >> lane) & 1) owner[slot_lo] = t_lo;
    if (BM == 128 && ((b_hi >> lane) & 1)) owner[slot_hi] = t_hi;
  }
  // slot (or k + 1: an id out of range) of row `lane` of the half of the tile that this wave's rows lie in
  const int half = wr * RW / 64, lane0 = wr * RW % 64;
  const int mark = (half ? t_hi : t_lo) > k ? -2 : (half ? slot_hi : slot_lo);

  f32x4 acc[TM][4];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  // slices s0 .. of ranks q0 .. on their way into registers; then into LDS: whether any value is infinite or NaN
  auto fetch = [&](int q0, int s0) {
#pragma unroll
    for (int s = 0; s < COUNT; ++s) {
      if (s0 + s >= slots) break;
      const T* ft = f + (int64_t)__builtin_amdgcn_readfirstlane(owner[s0 + s]) * r * m;
#pragma unroll
      for (int it = 0; it < PC::IT; ++it) reg[s * PC::IT + it] = PC::load(ft, m, r, m0, q0, it);
    }
  };
  auto put = [&](int s0) {
    bool bad = false;
#pragma unroll
    for (int s = 0; s < COUNT; ++s) {
      if (s0 + s >= slots) break;
#pragma unroll
      for (int it = 0; it < PC::IT; ++it) {
        bad |= nonfinite(reg[s * PC::IT + it], T());
        PC::store(lds + s * Slice<T, BN>::BYTES, it, reg[s * PC::IT + it]);
      }
    }
    return bad;
  };

  int at = 0;  // the stage being filled
  for (int k0 = lo; k0 < hi; k0 += KE) {
    if (STAGES == 1 && k0 > lo) __syncthreads();  // the stage has been read (of two, the barrier below has seen to it)
    if (k0 + KE <= hi) {
#pragma unroll
      for (int j = 0; j < XP + WP; ++j)
        *reinterpret_cast<u32x4*>(&lds[at + lds_slot((tid >> 3) + j * 32, tid & 7)]) = reg[j];
    } else {  // the rest of the summed axis, zeros behind it
#pragma unroll 1
      for (int row = tid >> 3; row < BM + BN; row += 32) {
        const T* p = row < BM ? x + (int64_t)perm[min(n0 + row, n - 1)] * ldx : w + (int64_t)min(m0 + row - BM, m - 1) * ldw;
        *reinterpret_cast<u32x4*>(&lds[at + lds_slot(row, tid & 7)]) = frag<T, false>(p, k0 + kt, hi);
      }
    }
    __syncthreads();
    if (k0 + 2 * KE <= hi)
      load(k0 + KE);
    else if (k0 + KE >= hi)
      fetch(0, 0);  // behind the last stage's products
#pragma unroll
    for (int kc = 0; kc < KE / KC; ++kc) {
      u32x4 wb[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        wb[j] = *reinterpret_cast<const u32x4*>(&lds[at + lds_slot(BM + wc * 64 + j * 16 + fr, kc * 4 + fs)]);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const u32x4 xa = *reinterpret_cast<const u32x4*>(&lds[at + lds_slot(wr * RW + i * 16 + fr, kc * 4 + fs)]);
        if constexpr (sizeof(T) == 4) {  // the four instructions on one accumulator four apart
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, wb[j])[e],
                                                               __builtin_bit_cast(f32x4, xa)[e], acc[i][j], 0, 0, 0);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) Mma<T>::run(acc[i][j], wb[j], xa);
        }
      }
    }
    if (STAGES == 2) at = STAGE - at;
  }

  // acc[i][j]: x row n0 + wr RW + i 16 + fr, columns m0 + wc 64 + j 16 + 4 fs + reg
  int from[TM];  // the rows' places in x, h and y
#pragma unroll
  for (int i = 0; i < TM; ++i) from[i] = perm[min(n0 + wr * RW + i * 16 + fr, n - 1)];
  u32x4 hf[TM];
  for (int q0 = 0, s0 = 0; slots > 0 && q0 < rp;) {
    if (s0 == 0)
#pragma unroll
      for (int i = 0; i < TM; ++i) hf[i] = h_frag<T>(h + (int64_t)from[i] * rp, q0, fs);
    __syncthreads();  // the last stage or slices have been read
    const bool apart = __syncthreads_or(put(s0));
    const int s_now = s0;
    s0 += COUNT;
    if (s0 >= slots) {
      s0 = 0;
      q0 += 16;
    }
    if (q0 < rp) fetch(q0, s0);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int si = __shfl(mark, lane0 + i * 16 + fr, 64);
      const int first = __builtin_amdgcn_readlane(mark, lane0 + i * 16);
      const int end = __builtin_amdgcn_readlane(mark, lane0 + i * 16 + 15);
      if (first < 0) continue;  // no adapter from this row on
      const int last = min(end < 0 ? slots - 1 : end, s_now + COUNT - 1);
      for (int s = max(first, s_now); s <= last; ++s) {
        const unsigned char* sl = lds + (s - s_now) * Slice<T, BN>::BYTES;
        const bool own = si == s;
        u32x4 hm;
#pragma unroll
        for (int e = 0; e < 4; ++e) hm[e] = own ? hf[i][e] : 0u;
        if (!apart) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            Mma<T>::run(acc[i][j], *reinterpret_cast<const u32x4*>(sl + Slice<T, BN>::at(wc * 64 + j * 16 + fr, fs)), hm);
        } else {  // an infinity times another row's 0 must not reach that row
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            f32x4 next = acc[i][j];  // the same sum in the same order for the adapter's own rows
            Mma<T>::run(next, *reinterpret_cast<const u32x4*>(sl + Slice<T, BN>::at(wc * 64 + j * 16 + fr, fs)), hm);
            if (own) acc[i][j] = next;
          }
        }
      }
    }
  }

#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const float poison = __shfl(mark, lane0 + i * 16 + fr, 64) == -2 ? NAN : 0.f;  // an id out of range
    if (n0 + wr * RW + i * 16 + fr >= n) continue;
    T* yr = y + (int64_t)from[i] * ldy;
    float* sr = SPLIT ? slabs + ((int64_t)blockIdx.y * n + from[i]) * m : nullptr;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = m0 + wc * 64 + j * 16 + fs * 4;
      if (SPLIT) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < m) sr[c + e] = acc[i][j][e] + poison;
        continue;
      }
      typedef T out4 __attribute__((ext_vector_type(4)));
      out4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (T)(acc[i][j][e] + poison);
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

// y = the slabs' sum, in their order
template <typename T>
__global__ void __launch_bounds__(256) split_join_kernel(const float* __restrict__ slabs, int64_t count, int splits, int m,
                                                         T* __restrict__ y, int64_t ldy) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    float a = slabs[i];
    for (int s = 1; s < splits; ++s) a += slabs[s * count + i];
    const int64_t row = i / m;
    y[row * ldy + (i - row * m)] = (T)a;
  }
}

// ---- few requests (serving): unsorted, no plan --------------------------------------------------------------
// (four waves per SIMD: with more registers than it needs hipcc keeps the accumulator in AGPRs and reads it back
// without the wait its last matrix instruction needs; tests/test_mfma_waits.py checks every build)
template <typename T, bool EVEN>
__global__ void __launch_bounds__(256, 4) h_few_kernel(const T* __restrict__ x, int64_t ldx, int n, int d, const T* __restrict__ a,
                                                    int k, int r, int rp, const int64_t* __restrict__ ids,
                                                    const float* __restrict__ scales, float* __restrict__ h) {
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= n) return;
  const int64_t t = ids[row];
  if (t < 0 || t >= k) return;
  for (int q0 = 0; q0 < rp; q0 += 16) {
    float* hr = h + (int64_t)row * rp + q0;
    h_row<T, EVEN>(x + row * ldx, a + (t * r + q0) * d, 0, d, d, min(16, r - q0), scales ? scales[t] : 1.f, threadIdx.x & 63,
             [&](int q, float v) { hr[q] = v; });
  }
}

// A workgroup: 16 columns of y for up to 16 RB rows, its four waves a quarter of the summed axis each; then one
// thread per value adds B_t h.  INLINE: h is worked out by every workgroup for itself (a row or two: A_t comes from
// the L2, and a launch less).
template <typename T, int RB, bool INLINE, bool EVEN>
__global__ void __launch_bounds__(256) project_few_kernel(const T* __restrict__ x, int64_t ldx, int n, int d,
                                                          const T* __restrict__ w, int64_t ldw, int m,
                                                          const T* __restrict__ a, const T* __restrict__ b, int k, int r,
                                                          int rp, const int64_t* __restrict__ ids,
                                                          const float* __restrict__ scales, const float* __restrict__ h,
                                                          T* __restrict__ y, int64_t ldy) {
  constexpr int N = Mma<T>::N, KC = Mma<T>::KC, U = RB == 1 ? 4 : 2;
  typedef T vec __attribute__((ext_vector_type(N)));
  __shared__ f32x4 part[4][RB][64];
  extern __shared__ float hs[];  // INLINE: [n][rp]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fs = lane >> 4;
  const int m0 = blockIdx.x * 16;
  const T* wp = w + (int64_t)min(m0 + fr, m - 1) * ldw;
  const T* xp[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) xp[rb] = x + (int64_t)min(rb * 16 + fr, n - 1) * ldx;
  f32x4 acc[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) acc[rb] = (f32x4){0.f, 0.f, 0.f, 0.f};
  u32x4 wf[U], xf[U][RB];
  auto load = [&](int c0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * 4 * KC + fs * N;
      wf[u] = frag<T, EVEN>(wp, c, d);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) xf[u][rb] = frag<T, EVEN>(xp[rb], c, d);
    }
  };
  load(wave * KC);
  if (INLINE)  // while the first loads are on their way: one wave per (row, 16 ranks)
    for (int u = wave; u < n * (rp / 16); u += 4) {
      const int i = u / (rp / 16), q0 = u % (rp / 16) * 16;
      const int64_t t = ids[i];
      if (t >= 0 && t < k)
        h_row<T, EVEN>(x + i * ldx, a + (t * r + q0) * d, 0, d, d, min(16, r - q0), scales ? scales[t] : 1.f, lane,
                 [&](int q, float v) { hs[i * rp + q0 + q] = v; });
    }
  for (int c0 = wave * KC; c0 < d;) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) Mma<T>::run(acc[rb], wf[u], xf[u][rb]);
    c0 += 4 * KC * U;
    if (c0 < d) load(c0);
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) part[wave][rb][lane] = acc[rb];
  __syncthreads();
  const int c = tid & 15, from = (c >> 2) * 16 + (tid >> 4), e = c & 3;  // part's lane of this thread's value
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = rb * 16 + (tid >> 4);
    if (row >= n || m0 + c >= m) continue;
    float v = (part[0][rb][from][e] + part[1][rb][from][e]) + (part[2][rb][from][e] + part[3][rb][from][e]);
    const int64_t t = ids[row];
    if (t >= 0 && t < k) {
      const T* bt = b + (t * m + m0 + c) * r;
      const float* hr = INLINE ? hs + row * rp : h + (int64_t)row * rp;
      float add = 0.f;
      for (int q = 0; q < r; q += N) {
        const vec bv = __builtin_bit_cast(vec, frag<T, EVEN>(bt, q, r));
#pragma unroll
        for (int z = 0; z < N; ++z)
          if (q + z < r) add = fmaf((float)bv[z], hr[q + z], add);
      }
      v += add;
    } else if (t != -1) {
      v = NAN;  // an id out of range
    }
    y[(int64_t)row * ldy + m0 + c] = (T)v;
  }
}

// ---- grads: out_t[q, c] = sum over the rows i of adapter t of h[i, q] v[i, c] ---------------------------
// One wave: 16 ranks x 16 N columns (a lane's 16 bytes of a row of v feed N instructions); the four
// waves of a workgroup take every fourth group of four rows, GU groups on their way at once.  Adapters with more
// than `per` rows are cut into chunks that write fp32 slabs, summed afterwards in ascending order.  An adapter without
// rows gets zeros.  Both gradients (dA from x and u, dB from dy and h) in one launch.
// fp32, 1024 x 14541 with 32 adapters of rank 8 of skewed sizes: 30 us for 77 MB (2.6 TB/s); its 7300 workgroups are
// short (the search of the chunk, the order, the rows, the sum over the waves, each waiting for the one before).
// Several blocks of columns per workgroup: 27 to 22 us where adapters have equal shares, 5 us more with skewed ones.
template <typename T>
struct Grad {
  const T* v;
  int64_t ldv;
  int cols, blocks;  // blocks: of 16 N columns
  const float* h;
  T* out;
  int64_t oc, oq;  // strides of out's columns and ranks
  float* slabs;
};
constexpr int GU = 4;

// An adapter of more than `per` rows from `row0` on has the slabs first_slab .. + chunks - 1: distinct, as chunks <=
// floor(2 rows / per) there, and below 2 n / per + 1.
__device__ __forceinline__ int64_t first_slab(int row0, int per) { return 2 * (int64_t)row0 / per; }

template <typename T, bool EVEN>
__global__ void __launch_bounds__(256) grads_kernel(Grad<T> g0, Grad<T> g1, int rp, int k, int r,
                                                    const int* __restrict__ perm, const int* __restrict__ start, int per) {
  constexpr int N = Mma<T>::N;
  typedef T vec __attribute__((ext_vector_type(N)));
  __shared__ f32x4 part[4][N][64];
  const int blocks = g0.blocks + g1.blocks, slot = blockIdx.x / blocks, by = blockIdx.x - slot * blocks;
  const Chunk ch = chunk_of(slot, start, k, per);
  if (ch.c < 0 || ch.c >= ch.chunks) return;
  const bool second = by >= g0.blocks;
  const T* __restrict__ v = second ? g1.v : g0.v;
  const float* __restrict__ h = second ? g1.h : g0.h;
  const int64_t ldv = second ? g1.ldv : g0.ldv;
  const int cols = second ? g1.cols : g0.cols, block = second ? by - g0.blocks : by;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fs = lane >> 4;
  const int c0 = block * 16 * N + fr * N, q0 = blockIdx.y * 16;
  f32x4 acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int i0 = wave * 4; i0 < ch.rows; i0 += 16 * GU) {
    int row[GU];
    float hv[GU];
    u32x4 x[GU];
#pragma unroll
    for (int u = 0; u < GU; ++u) row[u] = perm[ch.row0 + min(i0 + u * 16 + fs, ch.rows - 1)];
#pragma unroll
    for (int u = 0; u < GU; ++u) {
      const bool in = i0 + u * 16 + fs < ch.rows;
      hv[u] = in ? h[(int64_t)row[u] * rp + q0 + fr] : 0.f;
      x[u] = frag<T, EVEN>(v + (int64_t)row[u] * ldv, in ? c0 : cols, cols);
    }
#pragma unroll
    for (int u = 0; u < GU; ++u) {
      const vec xv = __builtin_bit_cast(vec, x[u]);
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(hv[u], (float)xv[j], acc[j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j) part[wave][j][lane] = acc[j];
  __syncthreads();
  // each wave sums and stores a quarter of the columns: ranks q0 + 4 fs + e of columns c0 + J wave + j
  constexpr int J = N / 4;
  const int q = q0 + fs * 4, cw = c0 + J * wave;
  f32x4 sum[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int z = J * wave + j;
    sum[j] = (part[0][z][lane] + part[1][z][lane]) + (part[2][z][lane] + part[3][z][lane]);
  }
  if (ch.chunks > 1) {
    float* sl = (second ? g1.slabs : g0.slabs) + (first_slab(ch.row0 - ch.c * per, per) + ch.c) * r * cols;  // [r][cols]
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (q + e < r && cw + j < cols) sl[(int64_t)(q + e) * cols + cw + j] = sum[j][e];
    return;
  }
  T* o = (second ? g1.out : g0.out) + (int64_t)ch.t * r * cols;
  const int64_t oc = second ? g1.oc : g0.oc, oq = second ? g1.oq : g0.oq;
  typedef T quad __attribute__((ext_vector_type(4)));
  if (oq == 1 && r % 4 == 0) {  // dB: four ranks of a column side by side
#pragma unroll
    for (int j = 0; j < J; ++j) {
      quad v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (T)sum[j][e];
      if (q < r && cw + j < cols) *reinterpret_cast<quad*>(o + (int64_t)(cw + j) * oc + q) = v;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (q + e < r && cw + j < cols) o[(int64_t)(cw + j) * oc + (int64_t)(q + e) * oq] = (T)sum[j][e];
}

template <typename T>
__global__ void __launch_bounds__(256) grads_join_kernel(Grad<T> g0, Grad<T> g1, const int* __restrict__ start, int per, int r) {
  const int t = blockIdx.x;
  const int s0 = start[t], chunks = (start[t + 1] - s0 + per - 1) / per;
  if (chunks <= 1) return;
  const int64_t slab = first_slab(s0, per);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const Grad<T>& g = w ? g1 : g0;
    const int64_t size = (int64_t)r * g.cols;
    for (int64_t i = (int64_t)blockIdx.y * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.y * 256) {
      float a = 0.f;
      for (int c = 0; c < chunks; c += 8) {  // eight on their way at once, added in ascending order
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = g.slabs[(slab + min(c + u, chunks - 1)) * size + i];
#pragma unroll
        for (int u = 0; u < 8; ++u) a += c + u < chunks ? v[u] : 0.f;
      }
      const int64_t q = i / g.cols, col = i - q * g.cols;
      g.out[t * size + col * g.oc + q * g.oq] = (T)a;
    }
  }
}

// dst [cols, ldd] = src [rows, lds] transposed, 32 x 32 tiles, for W and (blockIdx.z > 0) every A_t
template <typename T>
struct Flip {
  const T* src;
  int64_t lds, src_next;
  int rows, cols;
  T* dst;
  int64_t ldd, dst_next;
};
template <typename T>
__global__ void __launch_bounds__(256) transpose_kernel(Flip<T> w, Flip<T> a, int w_tiles, int w_across, int a_tiles, int a_across,
                                                        const int* __restrict__ start) {
  __shared__ T tile[32][33];
  int b = blockIdx.x;
  const bool first = b < w_tiles;
  const Flip<T>& z = first ? w : a;
  const T* src = z.src;
  T* dst = z.dst;
  if (!first) {
    b -= w_tiles;
    const int t = b / a_tiles;
    b -= t * a_tiles;
    if (start[t] == start[t + 1]) return;  // no row has this adapter (the whole workgroup)
    src += t * z.src_next;
    dst += t * z.dst_next;
  }
  const int across = first ? w_across : a_across;
  const int c0 = b % across * 32, r0 = b / across * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int i = ty; i < 32; i += 8)
    if (r0 + i < z.rows && c0 + tx < z.cols) tile[i][tx] = src[(int64_t)(r0 + i) * z.lds + c0 + tx];
  __syncthreads();
  for (int i = ty; i < 32; i += 8)
    if (c0 + i < z.cols && r0 + tx < z.rows) dst[(int64_t)(c0 + i) * z.ldd + r0 + tx] = tile[tx][i];
}

// ---- host side --------------------------------------------------------------------------------------------

int elem_size(int dtype) { return dtype == KGE_DT_F32 ? 4 : 2; }
bool dtype_ok(int dtype) { return dtype == KGE_DT_F32 || dtype == KGE_DT_BF16; }
bool ld_ok(int64_t ld, int64_t rows, int64_t cols) { return rows <= 1 || ld >= cols; }
constexpr int64_t MAX_N = (int64_t)1 << 30, MAX_K = 1 << 20, MAX_R = 1024;
constexpr int64_t FEW = 32;  // rows of the serving path
// 128-row tiles per CU below which tiles of 64 rows are taken (8192 x 512 x 512 with 237 adapters, one tile per CU:
// 16.7 against 18.1 us; 1024 x 14541 x 512 with 64, 3.6 per CU: 52 against 47)
constexpr int64_t PROJECT_SMALL = 2;
int64_t rank_pad(int64_t r) { return (r + 15) / 16 * 16; }
int64_t round256(int64_t x) { return (x + 255) & ~(int64_t)255; }

template <typename F>
int by_type(int dtype, F f) {
  return dtype == KGE_DT_F32 ? f((float*)nullptr) : f((__bf16*)nullptr);
}
// f(true or false as a type): whether all lengths are multiples of a fragment's elements
template <typename T, typename F>
int by_even(F f, std::initializer_list<int64_t> lengths) {
  bool even = true;
  for (int64_t l : lengths) even = even && l % Mma<T>::N == 0;
  return even ? f(std::true_type{}) : f(std::false_type{});
}
#define KGE_TRY(expr)      \
  do {                     \
    const int _r = (expr); \
    if (_r) return _r;     \
  } while (0)

bool sizes_ok(int dtype, int64_t n, int64_t d, int64_t m, int64_t k, int64_t r) {
  return dtype_ok(dtype) && n >= 0 && n <= MAX_N && d >= 1 && d <= MAX_N && m >= 1 && m <= MAX_N && k >= 1 && k <= MAX_K &&
         r >= 1 && r <= MAX_R;
}

// Splits of the summed columns of shrink: about four workgroups per CU where the rows' slots are fewer, at
// least 512 columns each.
int shrink_splits(int64_t n, int64_t cols, int64_t k, int64_t rp) {
  const int64_t groups = (std::min<int64_t>(n / 16 + k, n) + 1) * (rp / 16);
  const int64_t want = (4 * kge_num_cus() + groups - 1) / groups, most = std::max<int64_t>(1, cols / 512);
  return (int)std::max<int64_t>(1, std::min(want, most));
}

// Rows of one chunk of grads: up to 1024 rows one chunk per adapter (nothing to join), else 256 (a workgroup's four
// steps; with the join 8192 rows of 512 + 512 columns in bf16 take 16.5 us with one adapter, 19 with 237 of skewed sizes;
// with chunks of 1024 35.5 and 23, of 128 18.5 and 20), more where the launch would exceed about 2048 workgroups
int64_t grads_per(int64_t n, int64_t cols, int64_t r, int es) {
  const int64_t blocks = std::max<int64_t>(1, (cols * es + 255) / 256) * (rank_pad(r) / 16);  // (cols 0: no gradient wanted)
  const int64_t chunks = std::max<int64_t>(1, 2048 / blocks);
  return std::max<int64_t>(n > 1024 ? 256 : 1024, ((n + chunks - 1) / chunks + 63) / 64 * 64);
}
int64_t grads_ws(int64_t n, int64_t cols, int64_t r, int64_t per) {
  return n <= per ? 0 : round256((2 * n / per + 1) * r * cols * 4);
}

// Whether the plan is sorted: by the id reads of the other one, whose fewest rows cost as much as 1024 (a workgroup's
// step) and fewest groups as 512 (they run at once)
// (65536 rows of 237 adapters 46 us against 36 sorted, 2^20 rows 576 against 141, 8192 rows of 16000 adapters 142 against
// 43; below: 32768 rows of 237 27 against 29 and three launches more, 8192 rows of 2000 32 against 54)
constexpr int64_t SORT_FROM = 3 << 23;
bool plan_sorted(int64_t n, int64_t k) { return n > 0 && std::max<int64_t>(n, 1024) * std::max<int64_t>(k + 2, 512) > SORT_FROM; }
// rows of a wave: 512, or what leaves about 1024 waves
int64_t sort_rows(int64_t n) { return std::max<int64_t>(512, (n + 1023) / 1024); }
int64_t sort_bins(int64_t k) { return std::min<int64_t>(k + 2, BINS); }

// what the forward pass leaves for the backward one: the plan and h
struct Save {
  int *perm, *sid, *start;
  float* h;
  int *order, *counts, *totals;  // the sort's
  int64_t bytes;
};
Save save_of(void* base, int64_t n, int64_t d, int64_t k, int64_t r) {
  char* b = (char*)base;
  Save s;
  int64_t o = 0;
  s.perm = (int*)(b + o);
  o += round256(n * 4);
  s.sid = (int*)(b + o);
  o += round256(n * 4);
  s.start = (int*)(b + o);
  o += round256((k + 3) * 4);
  s.h = (float*)(b + o);
  o += round256(n * rank_pad(r) * shrink_splits(n, d, k, rank_pad(r)) * 4);
  s.order = (int*)(b + o);
  if (plan_sorted(n, k)) o += round256(n * 4);
  s.counts = (int*)(b + o);
  if (plan_sorted(n, k)) o += round256(((n + sort_rows(n) - 1) / sort_rows(n)) * sort_bins(k) * 4);
  s.totals = (int*)(b + o);
  if (plan_sorted(n, k)) o += round256(sort_bins(k) * 4);
  s.bytes = o;
  return s;
}

int64_t split_ws(int64_t n, int64_t d, int64_t m, int es);

struct BackWs {
  float* u;
  float* splits;
  void *wt, *at;
  int64_t ldwt;
  int64_t per;
  float *slabs_a, *slabs_b;
  int64_t bytes;
};
BackWs back_ws_of(void* base, int dtype, int64_t n, int64_t d, int64_t m, int64_t k, int64_t r, bool dx, bool da, bool db) {
  const int es = elem_size(dtype);
  char* b = (char*)base;
  BackWs s;
  int64_t o = 0;
  s.u = (float*)(b + o);
  if (dx || da) o += round256(n * rank_pad(r) * shrink_splits(n, m, k, rank_pad(r)) * 4);
  s.ldwt = (m * es + 15) / 16 * 16 / es;
  s.wt = b + o;
  if (dx) o += round256(d * s.ldwt * es);
  s.at = b + o;
  if (dx) o += round256(k * r * d * es);
  s.splits = (float*)(b + o);
  if (dx) o += split_ws(n, m, d, es);
  s.per = grads_per(n, (da ? d : 0) + (db ? m : 0), r, es);
  s.slabs_a = (float*)(b + o);
  if (da) o += grads_ws(n, d, r, s.per);
  s.slabs_b = (float*)(b + o);
  if (db) o += grads_ws(n, m, r, s.per);
  s.bytes = o;
  return s;
}

int run_sort(const int64_t* ids, int64_t n, int64_t k, const Save& s, hipStream_t st) {
  const int rows = (int)sort_rows(n), blocks = (int)((n + rows - 1) / rows), groups = (int)k + 2;
  for (int shift = 0; shift == 0 || groups > 1 << shift; shift += DIGIT) {
    const bool last = groups <= 1 << (shift + DIGIT);
    const int* src = shift == 0 ? nullptr : s.order;
    const int bins = std::min(BINS, ((groups - 1) >> shift) + 1);
    sort_count_kernel<<<dim3(blocks), dim3(64), 0, st>>>(ids, (int)n, (int)k, src, shift, bins, rows, s.counts);
    KGE_CHECK_LAUNCH();
    sort_scan_kernel<<<dim3(bins), dim3(64), 0, st>>>(s.counts, blocks, s.totals);
    KGE_CHECK_LAUNCH();
    sort_put_kernel<<<dim3(blocks), dim3(64), 0, st>>>(ids, (int)n, (int)k, src, shift, bins, rows, s.counts, s.totals,
                                                      last ? s.perm : s.order, last ? s.sid : nullptr);
    KGE_CHECK_LAUNCH();
  }
  sort_start_kernel<<<dim3((unsigned)(groups / 256 + 1)), dim3(256), 0, st>>>(s.sid, (int)n, groups, s.start);
  KGE_CHECK_LAUNCH();
  return 0;
}

// The plan, and h of every row: in the same launch where each row reading its own A_t costs little (24 MiB from
// the L2s, 2048 rows: 8192 rows of 16 columns take 14.1 us, 10.5 by adapter) or hardly two share one, else by adapter
// afterwards.
template <typename T, bool BY_RANK>
int run_shrink(const T* v, int64_t ldv, int64_t n, int64_t cols, const T* f, int64_t k, int64_t r, const float* scales,
               const Save& s, float* out, hipStream_t st);

template <typename T>
int run_plan_h(const int64_t* ids, const T* x, int64_t ldx, int64_t n, int64_t d, const T* a, int64_t k, int64_t r,
               const float* scales, const Save& s, hipStream_t st) {
  const bool with_h = (n <= 2048 && n * r * d * (int64_t)sizeof(T) <= 24 << 20) || k >= n, sorted = plan_sorted(n, k);
  const int64_t groups = sorted ? 0 : k + 2, blocks = groups + (with_h ? (n + 3) / 4 : 0);
  if (sorted) KGE_TRY(run_sort(ids, n, k, s, st));
  if (blocks > 0)
    KGE_TRY(by_even<T>([&](auto even) -> int {
      plan_h_kernel<T, even.value><<<dim3((unsigned)blocks), dim3(PT), 0, st>>>(
          ids, (int)n, (int)k, s.perm, s.sid, s.start, (int)groups, x, ldx, (int)d, a, (int)r, (int)rank_pad(r), scales, s.h);
      KGE_CHECK_LAUNCH();
      return 0;
    }, {d}));
  return with_h || n == 0 ? 0 : run_shrink<T, true>(x, ldx, n, d, a, k, r, scales, s, s.h, st);
}

template <typename T, bool BY_RANK>
int run_shrink(const T* v, int64_t ldv, int64_t n, int64_t cols, const T* f, int64_t k, int64_t r, const float* scales,
               const Save& s, float* out, hipStream_t st) {
  const int rp = (int)rank_pad(r), splits = shrink_splits(n, cols, k, rp);
  const int64_t per_split = ((cols + splits - 1) / splits + 127) / 128 * 128;
  KGE_TRY(by_even<T>([&](auto even) -> int {
    shrink_kernel<T, BY_RANK, even.value>
        <<<dim3((unsigned)(n / 16 + k), (unsigned)(rp / 16), (unsigned)splits), dim3(256), 0, st>>>(
            v, ldv, (int)n, (int)cols, f, (int)k, (int)r, rp, scales, s.perm, s.start, (int)per_split, out);
    KGE_CHECK_LAUNCH();
    return 0;
  }, {cols}));
  if (splits == 1) return 0;
  const int64_t count = n * rp / 4;
  slabs_kernel<<<dim3((unsigned)((count + 255) / 256)), dim3(256), 0, st>>>((f32x4*)out, count, splits);
  KGE_CHECK_LAUNCH();
  return 0;
}

// Elements of the summed axis per workgroup of project (a multiple of a stage's; >= d: no split): where tiles leave
// CUs idle, about two workgroups per CU with eight stages each at least; in fp32 no sum of more than 4096 products,
// whose roundings would show (in one chain dx from 30000 columns was off by 3e-6 of its norm, in eight or ten by
// 1e-6).  A backward pass for dx of 100 x 64 from 40000 columns then takes 97 us in fp32, 68 in bf16.
int64_t project_tiles(int64_t n, int64_t m, int64_t bm) { return (n + bm - 1) / bm * (m <= 64 ? 1 : (m + 127) / 128); }
int64_t split_per(int64_t n, int64_t d, int64_t m, int es) {
  const int64_t stage = BKB / es;
  int64_t tiles = project_tiles(n, m, 128);
  if (tiles < PROJECT_SMALL * kge_num_cus()) tiles = project_tiles(n, m, 64);
  const int64_t want = (2 * kge_num_cus() + tiles - 1) / std::max<int64_t>(1, tiles), most = std::max<int64_t>(1, d / (8 * stage));
  int64_t splits = std::max<int64_t>(1, std::min(want, most));
  if (es == 4) splits = std::max(splits, (d + 4095) / 4096);
  return ((d + splits - 1) / splits + stage - 1) / stage * stage;
}
int64_t split_ws(int64_t n, int64_t d, int64_t m, int es) {
  const int64_t per = split_per(n, d, m, es);
  return per >= d ? 0 : round256((d + per - 1) / per * n * m * 4);
}

template <typename T, int BM, int BN>
int launch_project(const T* x, int64_t ldx, int64_t n, int64_t d, const T* w, int64_t ldw, int64_t m, const T* f, int64_t k,
                   int64_t r, const float* h, const Save& s, T* y, int64_t ldy, float* slabs, hipStream_t st) {
  // fp32 is bound by its matrix instructions: two workgroups per CU with two stages each keep them fed, and
  // share the last round of tiles better than three (133 against 105 TFLOP/s at 4096^3)
  constexpr int STAGES = sizeof(T) == 4 ? 2 : 1;
  const int64_t row_tiles = (n + BM - 1) / BM, tiles = project_tiles(n, m, BM);
  const int64_t per = split_per(n, d, m, sizeof(T)), splits = (d + per - 1) / per;
  KGE_REQUIRE(tiles < ((int64_t)1 << 31) && splits <= 65535);
  const int yvec = (reinterpret_cast<uintptr_t>(y) % (4 * sizeof(T))) == 0 && ldy % 4 == 0;
  KGE_TRY(by_even<T>([&](auto even) -> int {
    auto launch = [&](auto kernel) {
      kernel<<<dim3((unsigned)tiles, (unsigned)splits), dim3(256), 0, st>>>(
          x, ldx, (int)n, (int)d, w, ldw, (int)m, f, (int)k, (int)r, (int)rank_pad(r), h, s.perm, s.sid, y, ldy,
          (int)row_tiles, yvec, (int)per, slabs);
    };
    if (splits == 1)
      launch(project_kernel<T, BM, BN, STAGES, even.value, false>);
    else
      launch(project_kernel<T, BM, BN, STAGES, even.value, true>);
    KGE_CHECK_LAUNCH();
    return 0;
  }, {r}));
  if (splits == 1) return 0;
  split_join_kernel<T><<<dim3((unsigned)std::min<int64_t>((n * m + 255) / 256, 8192)), dim3(256), 0, st>>>(
      slabs, n * m, (int)splits, (int)m, y, ldy);
  KGE_CHECK_LAUNCH();
  return 0;
}

template <typename T>
int run_project(const T* x, int64_t ldx, int64_t n, int64_t d, const T* w, int64_t ldw, int64_t m, const T* f, int64_t k,
                int64_t r, const float* h, const Save& s, T* y, int64_t ldy, float* slabs, hipStream_t st) {
  const bool short_tiles = project_tiles(n, m, 128) < PROJECT_SMALL * kge_num_cus();
  const auto launch = m <= 64 ? (short_tiles ? launch_project<T, 64, 64> : launch_project<T, 128, 64>)
                              : (short_tiles ? launch_project<T, 64, 128> : launch_project<T, 128, 128>);
  return launch(x, ldx, n, d, w, ldw, m, f, k, r, h, s, y, ldy, slabs, st);
}

template <typename T>
int run_grads(Grad<T> g0, Grad<T> g1, int64_t n, int64_t k, int64_t r, const Save& s, int64_t per, hipStream_t st) {
  g0.blocks = (int)((g0.cols * (int64_t)sizeof(T) + 255) / 256);
  g1.blocks = (int)((g1.cols * (int64_t)sizeof(T) + 255) / 256);
  const int64_t wgs = (n / per + k) * ((int64_t)g0.blocks + g1.blocks), cols = (int64_t)g0.cols + g1.cols;
  KGE_REQUIRE(wgs < (int64_t)1 << 31);
  KGE_TRY(by_even<T>([&](auto even) -> int {
    grads_kernel<T, even.value><<<dim3((unsigned)wgs, (unsigned)(rank_pad(r) / 16)), dim3(256), 0, st>>>(
        g0, g1, (int)rank_pad(r), (int)k, (int)r, s.perm, s.start, (int)per);
    KGE_CHECK_LAUNCH();
    return 0;
  }, {g0.cols, g1.cols}));
  if (n <= per) return 0;
  const int64_t join = std::max<int64_t>(1, std::min<int64_t>((r * cols + 255) / 256, 64));
  grads_join_kernel<T><<<dim3((unsigned)k, (unsigned)join), dim3(256), 0, st>>>(g0, g1, s.start, (int)per, (int)r);
  KGE_CHECK_LAUNCH();
  return 0;
}

template <typename T, int RB>
int run_few(const T* x, int64_t ldx, int64_t n, int64_t d, const T* w, int64_t ldw, int64_t m, const T* a, const T* b,
            int64_t k, int64_t r, const int64_t* ids, const float* scales, float* h, T* y, int64_t ldy, hipStream_t st) {
  const int rp = (int)rank_pad(r);
  const dim3 grid((unsigned)((m + 15) / 16));
  const bool here = RB == 1 && n * r * d * (int64_t)sizeof(T) <= 32768 && n * rp * 4 <= 16384;
  return by_even<T>([&](auto even) -> int {
    if (here) {
      project_few_kernel<T, 1, true, even.value><<<grid, dim3(256), (size_t)(n * rp * 4), st>>>(
          x, ldx, (int)n, (int)d, w, ldw, (int)m, a, b, (int)k, (int)r, rp, ids, scales, nullptr, y, ldy);
      KGE_CHECK_LAUNCH();
      return 0;
    }
    h_few_kernel<T, even.value><<<dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st>>>(x, ldx, (int)n, (int)d, a, (int)k, (int)r,
                                                                                   rp, ids, scales, h);
    KGE_CHECK_LAUNCH();
    project_few_kernel<T, RB, false, even.value><<<grid, dim3(256), 0, st>>>(
        x, ldx, (int)n, (int)d, w, ldw, (int)m, a, b, (int)k, (int)r, rp, ids, scales, h, y, ldy);
    KGE_CHECK_LAUNCH();
    return 0;
  }, {d, r});
}

// W^T [d, ldwt] and every A_t^T [d, r]: dx is the projection of dy by them
template <typename T>
int run_transpose(const T* w, int64_t ldw, int64_t m, int64_t d, const T* a, int64_t k, int64_t r, T* wt, int64_t ldwt, T* at,
                  const Save& s, hipStream_t st) {
  const int64_t across = (d + 31) / 32, w_tiles = across * ((m + 31) / 32), a_tiles = across * ((r + 31) / 32);
  KGE_REQUIRE(w_tiles + a_tiles * k < (int64_t)1 << 31);
  transpose_kernel<T><<<dim3((unsigned)(w_tiles + a_tiles * k)), dim3(256), 0, st>>>(
      Flip<T>{w, ldw, 0, (int)m, (int)d, wt, ldwt, 0}, Flip<T>{a, d, r * d, (int)r, (int)d, at, r, r * d}, (int)w_tiles,
      (int)across, (int)a_tiles, (int)across, s.start);
  KGE_CHECK_LAUNCH();
  return 0;
}

}  // namespace

extern "C" int64_t kge_adapter_save_size(int64_t n, int64_t d, int64_t k, int64_t r) {
  return sizes_ok(KGE_DT_F32, n, d, 1, k, r) ? save_of(nullptr, n, d, k, r).bytes : 0;
}

extern "C" int64_t kge_adapter_forward_ws_size(int dtype, int64_t n, int64_t d, int64_t m, int64_t k, int64_t r,
                                               int for_backward) {
  return sizes_ok(dtype, n, d, m, k, r) && n > 0 && (for_backward || n > FEW) ? split_ws(n, d, m, elem_size(dtype)) : 0;
}

extern "C" int kge_adapter_forward(const void* x, int dtype, int64_t ldx, int64_t n, int64_t d, const void* w, int64_t ldw,
                                   int64_t m, const void* a, const void* b, int64_t k, int64_t r, const int64_t* ids,
                                   const float* scales, void* y, int64_t ldy, void* save, int64_t save_bytes, int for_backward,
                                   void* ws, int64_t ws_bytes, void* stream) {
  KGE_REQUIRE(sizes_ok(dtype, n, d, m, k, r) && ld_ok(ldx, n, d) && ld_ok(ldw, m, d) && ld_ok(ldy, n, m));
  KGE_REQUIRE(save && aligned16(save) && save_bytes >= save_of(save, n, d, k, r).bytes);
  KGE_REQUIRE(n == 0 || (x && w && a && b && ids && y));
  const int64_t ws_least = kge_adapter_forward_ws_size(dtype, n, d, m, k, r, for_backward);
  KGE_REQUIRE(ws_bytes >= ws_least && (ws_least == 0 || (ws && aligned16(ws))));
  const Save s = save_of(save, n, d, k, r);
  const hipStream_t st = as_stream(stream);
  return by_type(dtype, [&](auto* tag) -> int {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    const T *xt = (const T*)x, *wt = (const T*)w, *at = (const T*)a, *bt = (const T*)b;
    T* yt = (T*)y;
    if (!for_backward && n <= FEW) {
      if (n == 0) return 0;
      return n <= 16 ? run_few<T, 1>(xt, ldx, n, d, wt, ldw, m, at, bt, k, r, ids, scales, s.h, yt, ldy, st)
                     : run_few<T, 2>(xt, ldx, n, d, wt, ldw, m, at, bt, k, r, ids, scales, s.h, yt, ldy, st);
    }
    KGE_TRY(run_plan_h<T>(ids, xt, ldx, n, d, at, k, r, scales, s, st));
    if (n == 0) return 0;
    return run_project<T>(xt, ldx, n, d, wt, ldw, m, bt, k, r, s.h, s, yt, ldy, (float*)ws, st);
  });
}

extern "C" int64_t kge_adapter_backward_ws_size(int dtype, int64_t n, int64_t d, int64_t m, int64_t k, int64_t r, int dx,
                                                int da, int db) {
  return sizes_ok(dtype, n, d, m, k, r) ? back_ws_of(nullptr, dtype, n, d, m, k, r, dx, da, db).bytes : 0;
}

extern "C" int kge_adapter_backward(const void* dy, int dtype, int64_t lddy, int64_t n, int64_t m, const void* x, int64_t ldx,
                                    int64_t d, const void* w, int64_t ldw, const void* a, const void* b, int64_t k, int64_t r,
                                    const float* scales, void* save, int64_t save_bytes, void* dx, int64_t lddx, void* da,
                                    void* db, void* ws, int64_t ws_bytes, void* stream) {
  KGE_REQUIRE(sizes_ok(dtype, n, d, m, k, r) && ld_ok(lddy, n, m) && ld_ok(ldx, n, d) && ld_ok(ldw, m, d) &&
              ld_ok(lddx, n, d));
  KGE_REQUIRE(save && aligned16(save) && save_bytes >= save_of(save, n, d, k, r).bytes);
  KGE_REQUIRE(n == 0 || (dy && x && w && a && b));
  const Save s = save_of(save, n, d, k, r);
  const BackWs q = back_ws_of(ws, dtype, n, d, m, k, r, dx, da, db);
  KGE_REQUIRE(ws_bytes >= q.bytes && (q.bytes == 0 || (ws && aligned16(ws))));
  const hipStream_t st = as_stream(stream);
  return by_type(dtype, [&](auto* tag) -> int {
    typedef typename std::remove_pointer<decltype(tag)>::type T;
    const T *dyt = (const T*)dy, *xt = (const T*)x, *wt = (const T*)w, *at = (const T*)a, *bt = (const T*)b;
    if (n > 0 && (dx || da)) KGE_TRY((run_shrink<T, false>(dyt, lddy, n, m, bt, k, r, scales, s, q.u, st)));
    if (n > 0 && dx) {
      KGE_TRY(run_transpose<T>(wt, ldw, m, d, at, k, r, (T*)q.wt, q.ldwt, (T*)q.at, s, st));
      KGE_TRY(run_project<T>(dyt, lddy, n, m, (const T*)q.wt, q.ldwt, d, (const T*)q.at, k, r, q.u, s, (T*)dx, lddx, q.splits, st));
    }
    const Grad<T> ga{xt, ldx, (int)d, 0, q.u, (T*)da, 1, d, q.slabs_a}, gb{dyt, lddy, (int)m, 0, s.h, (T*)db, r, 1, q.slabs_b};
    const Grad<T> none{nullptr, 0, 0, 0, nullptr, nullptr, 0, 0, nullptr};
    if (!da && !db) return 0;
    return run_grads<T>(da ? ga : gb, da && db ? gb : none, n, k, r, s, q.per, st);
  });
}
