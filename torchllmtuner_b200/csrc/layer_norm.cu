// LayerNorm for sm_100a, forward and backward, bf16 or fp32 storage with fp32 statistics.
//   forward   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), h = (x - m) r, y = h w + b
//   backward  g = dy w, dx = r (g - mean g - h mean(g h)), dw = sum_rows dy h, db = sum_rows dy
// (reference call sites: llmtuner/models/qwen/qwen3_5/multimodal.py:47-290, llmtuner/models/kimi/kimi_k3/multimodal.py:146-914)
//
// Bound by memory: the forward reads x and writes y, the backward reads x and dy and writes dx. A row is owned by TR threads, each with NV
// 16-byte vectors in registers, so a row is read once; the variance is the mean of squared deviations (a second sum over registers, not a
// difference of two large sums). 16384 x 1152 bf16: forward 15 us (4.9 TB/s, writes stay in L2), backward 28 us (4.1 TB/s: the column sums leave
// room for 8 warps an SM, and their issue slots are half used) and 2.7 us for the sums over blocks. fp32: 41 and 61 us (floors 23 and 35). 1151 columns
// of bf16, where every row starts elsewhere in its granule: 34 and 85 us; beside the wider registers its elements are masked and weights read one by one.
// Rows of any width and any 2- or 4-byte start are read as the aligned 16-byte granules that hold them: with `s` elements of a row's first
// granule belonging to the row before, vector i holds columns [V i - s, V i - s + V). Only granules with at least one element of the row are
// touched (such a granule lies in the same page as that element), foreign elements are replaced by zero and never written. A group takes every
// num_groups-th row, and num_groups is a multiple of V, so `s` and with it the column of every register is the same for all its rows: weights
// and the sums of their gradients stay in registers.
#include <initializer_list>
#include "kernels.h"
#include "vec_io.cuh"

namespace llmt {

template <typename T>
struct Granule { static constexpr int V = 16 / (int)sizeof(T); };

// Sums of (a, b) over the TR threads of a group in a fixed order. One barrier per call: two buffers alternate, and no warp can be two calls ahead.
template <bool WARP>
__device__ __forceinline__ float2 group_sum2(float2 v, int tr, float2* red, int& buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (WARP || tr == 32) return v;
  const int grp = threadIdx.x / tr, w = (threadIdx.x - grp * tr) >> 5, nw = tr >> 5;
  float2* r = red + buf * 32 + grp * nw;               // at most 32 warps in a block
  if ((threadIdx.x & 31) == 0) r[w] = v;
  named_bar_sync(1 + grp, tr);
  float2 t = r[0];
  for (int i = 1; i < nw; ++i) {
    t.x += r[i].x;
    t.y += r[i].y;
  }
  buf ^= 1;
  return t;
}

// This thread's place in the rows of its group: shift `s`, first column of each vector, and whether a vector lies in the row at all / entirely.
// ALIGNED: every row starts on a granule and is a whole number of them.
template <int V, bool ALIGNED>
struct RowPlace {
  int s, D, tr, t;
  __device__ __forceinline__ int col(int i) const { return (i * tr + t) * V - (ALIGNED ? 0 : s); }
  __device__ __forceinline__ bool any(int i) const { return col(i) < D; }                       // (i, t) = (0, 0) starts at -s > -V
  __device__ __forceinline__ bool all(int i) const { return ALIGNED ? any(i) : col(i) >= 0 && col(i) + V <= D; }
  __device__ __forceinline__ bool has(int i, int j) const { return ALIGNED ? any(i) : col(i) + j >= 0 && col(i) + j < D; }
};
template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ void load_cols(const T* row, const RowPlace<V, ALIGNED>& p, int i, Raw<T, V>& r) {
  r.zero();
  if (p.any(i)) r.load(row + p.col(i));
}
// Foreign elements become zero.
template <int V, bool ALIGNED>
__device__ __forceinline__ void mask_cols(const RowPlace<V, ALIGNED>& p, int i, float* f) {
  if (ALIGNED || p.all(i)) return;                      // an aligned thread outside the row has loaded zeros
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (!p.has(i, j)) f[j] = 0.f;
}
template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ void store_cols(T* row, const RowPlace<V, ALIGNED>& p, int i, const float* f) {
  if (p.all(i)) {
    store_vec<T, V>(row + p.col(i), f);
  } else if (!ALIGNED && p.any(i)) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (p.has(i, j)) store_vec<T, 1>(row + p.col(i) + j, f + j);
  }
}
template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ void load_weights(const T* w, const RowPlace<V, ALIGNED>& p, int i, Raw<T, V>& r) {
  if constexpr (ALIGNED) {
    load_cols(w, p, i, r);
    return;
  }
  float f[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    f[j] = 0.f;
    if (p.has(i, j)) load_vec<T, 1>(w + p.col(i) + j, f + j);
  }
  r.set(f);                                             // exact: the values came from T
}
template <typename T>
__device__ __forceinline__ int shift_of(const T* row) { return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T)); }

// WARP: one warp per row, eight rows per block. Otherwise the block is one group.
template <typename T, int NV, bool WARP, bool ALIGNED>
__global__ void __launch_bounds__(WARP ? 256 : 512, WARP && NV <= 5 ? 2 : 1)
layer_norm_fwd_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, const T* __restrict__ b, T* __restrict__ y,
                      float* __restrict__ mean, float* __restrict__ rstd, int R, int D, int tr, float eps) {
  constexpr int V = Granule<T>::V;
  __shared__ float2 red[2 * 32];
  const int grp = WARP ? threadIdx.x >> 5 : 0, groups = WARP ? 8 : 1;
  const int64_t step = (int64_t)gridDim.x * groups;
  int64_t row = (int64_t)blockIdx.x * groups + grp;
  if (row >= R) return;                                 // whole groups leave together
  const RowPlace<V, ALIGNED> p{shift_of(x + row * ldx), D, tr, WARP ? (int)threadIdx.x & 31 : (int)threadIdx.x};
  int buf = 0;
  Raw<T, V> wr[NV], br[NV], xr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) load_cols(x + row * ldx, p, i, xr[i]);
  if constexpr (!ALIGNED) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      load_weights(w, p, i, wr[i]);
      load_weights(b, p, i, br[i]);
    }
  }
  const float inv_d = 1.f / (float)D;
  for (; row < R; row += step) {
    float v[NV][V], sum = 0.f, sq = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      xr[i].get(v[i]);
      mask_cols(p, i, v[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) sum += v[i][j];
    }
    if (row + step < R) {                               // the next row is on its way while this one is reduced
#pragma unroll
      for (int i = 0; i < NV; ++i) load_cols(x + (row + step) * ldx, p, i, xr[i]);
    }
    const float m = group_sum2<WARP>(make_float2(sum, 0.f), tr, red, buf).x * inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] -= m;
        if (p.has(i, j)) sq += v[i][j] * v[i][j];
      }
    const float r = rsqrtf(group_sum2<WARP>(make_float2(sq, 0.f), tr, red, buf).x * inv_d + eps);
    if (p.t == 0) {
      mean[row] = m;
      rstd[row] = r;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float wv[V], bv[V];
      if constexpr (ALIGNED) {                          // from L1: registers are better spent on rows in flight
        load_weights(w, p, i, wr[i]);
        load_weights(b, p, i, br[i]);
      }
      wr[i].get(wv);
      br[i].get(bv);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = v[i][j] * r * wv[j] + bv[j];
      store_cols(y + row * (int64_t)D, p, i, v[i]);
    }
  }
}

// partial [grid][2][D]: sums of dy h and of dy over the block's rows. WARP: one warp per row, eight rows per block; otherwise the block is one
// group. The sums of a column stay in registers over all rows (2 V NV of them, so an SM holds 256 threads); the next row is fetched before this
// one is reduced.
template <typename T, int NV, bool WARP, bool ALIGNED, int THREADS>
__global__ void __launch_bounds__(THREADS, NV <= 2 ? 2 : 1) layer_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, int64_t ldx,
                                                                                 const T* __restrict__ w, const float* __restrict__ mean,
                                                                                 const float* __restrict__ rstd, T* __restrict__ dx,
                                                                                 float* __restrict__ partial, int R, int D, int tr) {
  constexpr int V = Granule<T>::V;
  __shared__ float2 red[2 * 32];
  extern __shared__ __align__(16) float sums[];         // only with several groups
  const int grp = WARP ? threadIdx.x >> 5 : 0, groups = WARP ? THREADS / 32 : 1;
  const int64_t step = (int64_t)gridDim.x * groups;
  int64_t row = (int64_t)blockIdx.x * groups + grp;
  const RowPlace<V, ALIGNED> p{row < R ? shift_of(x + row * ldx) : 0, D, tr, WARP ? (int)threadIdx.x & 31 : (int)threadIdx.x};
  int buf = 0;
  float dw[NV][V], db[NV][V];
  Raw<T, V> wr[NV], xr[NV], gr[NV];
  float m = 0.f, r = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.f;
    wr[i].zero();
    if (row < R) {
      load_cols(x + row * ldx, p, i, xr[i]);
      load_cols(dy + row * (int64_t)D, p, i, gr[i]);
    }
  }
  if (row < R) {
    m = mean[row];
    r = rstd[row];
    if constexpr (!ALIGNED) {
#pragma unroll
      for (int i = 0; i < NV; ++i) load_weights(w, p, i, wr[i]);
    }
  }
  const float inv_d = 1.f / (float)D;
  for (; row < R; row += step) {
    float2 s = make_float2(0.f, 0.f);
    const float rr = r, mr = -m * r;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float h[V], g[V], wv[V];
      xr[i].get(h);
      gr[i].get(g);
      if constexpr (ALIGNED) load_weights(w, p, i, wr[i]);
      wr[i].get(wv);
      mask_cols(p, i, h);
      mask_cols(p, i, g);                               // a zero gradient keeps a foreign column out of every sum
#pragma unroll
      for (int j = 0; j < V; ++j) {
        h[j] = h[j] * rr + mr;
        dw[i][j] += g[j] * h[j];
        db[i][j] += g[j];
        g[j] *= wv[j];
        s.x += g[j];
        s.y += g[j] * h[j];
      }
    }
    Raw<T, V> xn[NV], gn[NV];
    if (row + step < R) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        load_cols(x + (row + step) * ldx, p, i, xn[i]);
        load_cols(dy + (row + step) * (int64_t)D, p, i, gn[i]);
      }
      m = mean[row + step];
      r = rstd[row + step];
    }
    s = group_sum2<WARP>(s, tr, red, buf);
    // r (g w - mean - h k) with h = x r + mr, as one polynomial in x: fewer live registers than keeping h and g. Times r at the end: r^2 leaves fp32
    // where the values are small and eps is 0 (a spread below 5e-20)
    const float k = s.y * inv_d, c0 = s.x * inv_d + mr * k, c1 = rr * k;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float h[V], g[V], wv[V];
      xr[i].get(h);
      gr[i].get(g);
      if constexpr (ALIGNED) load_weights(w, p, i, wr[i]);
      wr[i].get(wv);
#pragma unroll
      for (int j = 0; j < V; ++j) g[j] = rr * (g[j] * wv[j] - (c1 * h[j] + c0));
      store_cols(dx + row * (int64_t)D, p, i, g);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      xr[i] = xn[i];
      gr[i] = gn[i];
    }
  }
  float* out = partial + (int64_t)blockIdx.x * 2 * D;
  if constexpr (!WARP) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = p.col(i) + j;
        if (p.has(i, j)) {
          out[c] = dw[i][j];
          out[D + c] = db[i][j];
        }
      }
    return;
  }
  // the sums of the eight warps meet in a tree; a thread's columns are the same in every warp where rows are aligned, else they are shifted by
  // the row: then the warps are added one after another
  if constexpr (ALIGNED) {
    float4* box = reinterpret_cast<float4*>(sums);      // [4 warps][2 NV V / 4][32 lanes]
    constexpr int Q = 2 * NV * V / 4;
#pragma unroll
    for (int half = 4; half > 0; half >>= 1) {
      if (grp >= half && grp < 2 * half) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const float* f = q < Q / 2 ? &dw[q * 4 / V][q * 4 % V] : &db[(q - Q / 2) * 4 / V][(q - Q / 2) * 4 % V];
          box[((grp - half) * Q + q) * 32 + p.t] = make_float4(f[0], f[1], f[2], f[3]);
        }
      }
      __syncthreads();
      if (grp < half) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          float* f = q < Q / 2 ? &dw[q * 4 / V][q * 4 % V] : &db[(q - Q / 2) * 4 / V][(q - Q / 2) * 4 % V];
          const float4 o = box[(grp * Q + q) * 32 + p.t];
          f[0] += o.x; f[1] += o.y; f[2] += o.z; f[3] += o.w;
        }
      }
      __syncthreads();
    }
    if (grp == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (p.any(i)) {
          store_vec<float, V>(out + p.col(i), dw[i]);
          store_vec<float, V>(out + D + p.col(i), db[i]);
        }
    }
    return;
  }
  for (int k = 0; k < groups; ++k) {                    // the groups of a block are added in their order
    if (grp == k) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int c = p.col(i) + j;
          if (p.has(i, j)) {
            sums[c] = k == 0 ? dw[i][j] : sums[c] + dw[i][j];
            sums[D + c] = k == 0 ? db[i][j] : sums[D + c] + db[i][j];
          }
        }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < 2 * D; c += THREADS) out[c] = sums[c];
}

// dw | db [2 D] in T = column sums of partial [P][2 D]: 32 columns per block, its 32 warps take every 32nd row, fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_colsum_kernel(const float* __restrict__ partial, T* __restrict__ dw, T* __restrict__ db, int P, int D) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < 2 * D) {
#pragma unroll 4
    for (int q = wid; q < P; q += 32) s += partial[(int64_t)q * 2 * D + c];
  }
  part[wid][lane] = s;
  __syncthreads();
  s = warp_sum(part[lane][wid]);
  const int oc = blockIdx.x * 32 + wid;
  if (lane == 0 && oc < 2 * D) store_vec<T, 1>(oc < D ? dw + oc : db + oc - D, &s);
}

int sm_count();

// Threads per row and vectors per thread. Forward: a warp per row while that is at most 8 vectors a thread (no barrier); beyond, 4 vectors.
// Backward: a warp per row up to 5 vectors (what registers hold beside two sums per column), beyond 4 vectors and one group per block.
struct LnShape { int tr, nv, groups; };
static LnShape ln_fwd_shape(int vecs) {
  if (vecs <= 256) return {32, vecs <= 192 ? (vecs + 31) / 32 : 8, 8};
  return {(vecs + 127) / 128 * 32, 4, 1};
}
static LnShape ln_bwd_shape(int vecs) {
  if (vecs <= 160) return {32, (vecs + 31) / 32, 8};
  return {(vecs + 127) / 128 * 32, 4, 1};
}
constexpr int kLnMaxVecs = 2048;

// Granules of a row: of one that starts anywhere, or (`aligned`) on a granule.
template <typename T>
static int ln_vecs(int D, bool aligned) { return (D + (aligned ? 1 : 2) * (Granule<T>::V - 1)) / Granule<T>::V; }
template <typename T>
static bool ln_aligned(const void* x, int64_t ldx, int D) {
  return !((reinterpret_cast<uintptr_t>(x) & 15) || ldx % Granule<T>::V || D % Granule<T>::V);
}

template <typename T>
static int ln_bwd_grid(int R, const LnShape& s) {
  const int V = Granule<T>::V;
  const int most = sm_count() * (s.tr == 32 ? (s.nv <= 2 ? 2 : 1) : s.tr >= 256 ? 1 : 256 / s.tr);
  const int64_t need = ((int64_t)R + s.groups - 1) / s.groups;
  if (need >= most) return most / V * V;                 // not beyond what the machine holds at once
  return ((int)need + V - 1) / V * V;
}

// All rows of an operand lie at row * ld; every operand has the same granule shift in the same row.
template <typename T>
static bool ln_same_shift(const void* x, int64_t ldx, int D, std::initializer_list<const void*> dense) {
  const uintptr_t bx = reinterpret_cast<uintptr_t>(x);
  if (bx % sizeof(T)) return false;
  for (const void* d : dense)
    if ((reinterpret_cast<uintptr_t>(d) & 15) != (bx & 15)) return false;
  return (ldx - D) % Granule<T>::V == 0;
}

template <typename T>
static int ln_fwd(const void* x, int64_t ldx, const void* w, const void* b, void* y, float* mean, float* rstd, int R, int D, float eps,
                  cudaStream_t stream) {
  if (R <= 0 || D <= 0) return R == 0 ? 0 : -10;
  const uintptr_t wb = reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(b);
  const bool aligned = ln_aligned<T>(x, ldx, D) && !(wb & 15);
  const int vecs = ln_vecs<T>(D, aligned);
  if (!ln_same_shift<T>(x, ldx, D, {y}) || ldx < D || vecs > kLnMaxVecs || wb % sizeof(T)) return -10;
  const LnShape s = ln_fwd_shape(vecs);
  const int V = Granule<T>::V, threads = s.tr * s.groups;
  const int most = sm_count() * (s.tr == 32 ? (s.nv <= 2 ? 4 : s.nv <= 5 ? 2 : 1) : 1024 / threads);
  const int64_t need = ((int64_t)R + s.groups - 1) / s.groups;
  const int grid = ((int)(need < most ? need : most) + V - 1) / V * V;
  const T *xp = reinterpret_cast<const T*>(x), *wp = reinterpret_cast<const T*>(w), *bp = reinterpret_cast<const T*>(b);
#define LLMT_LN(N, W)                                                                                                                          \
  if (s.nv == N && (s.tr == 32) == W) {                                                                                                        \
    if (aligned) layer_norm_fwd_kernel<T, N, W, true><<<grid, threads, 0, stream>>>(xp, ldx, wp, bp, reinterpret_cast<T*>(y), mean, rstd, R, D, s.tr, eps);  \
    else layer_norm_fwd_kernel<T, N, W, false><<<grid, threads, 0, stream>>>(xp, ldx, wp, bp, reinterpret_cast<T*>(y), mean, rstd, R, D, s.tr, eps);         \
    return cudaGetLastError() == cudaSuccess ? 0 : -3;                                                                                         \
  }
  LLMT_LN(1, true) LLMT_LN(2, true) LLMT_LN(3, true) LLMT_LN(4, true) LLMT_LN(5, true) LLMT_LN(6, true) LLMT_LN(8, true) LLMT_LN(4, false)
#undef LLMT_LN
  return -4;
}

template <typename T>
static int ln_bwd(const void* dy, const void* x, int64_t ldx, const void* w, const float* mean, const float* rstd, void* dx, float* partial, int P,
                  void* dw, void* db, int R, int D, cudaStream_t stream) {
  if (R <= 0 || D <= 0) return -10;
  const uintptr_t wp_ = reinterpret_cast<uintptr_t>(w);
  const bool aligned = ln_aligned<T>(x, ldx, D) && !(wp_ & 15);
  const int vecs = ln_vecs<T>(D, aligned);
  if (!ln_same_shift<T>(x, ldx, D, {dy, dx}) || ldx < D || vecs > kLnMaxVecs) return -10;
  if ((wp_ | reinterpret_cast<uintptr_t>(dw) | reinterpret_cast<uintptr_t>(db)) % sizeof(T)) return -10;
  const LnShape s = ln_bwd_shape(vecs);
  const int grid = ln_bwd_grid<T>(R, s), threads = s.tr * s.groups;
  if (grid > P) return -10;
  constexpr int V = Granule<T>::V;
  const size_t smem = s.groups == 1 ? 0 : aligned ? (size_t)4 * 2 * s.nv * V * 32 * sizeof(float) : (size_t)2 * D * sizeof(float);   // at most 40 KB
  const T *gp = reinterpret_cast<const T*>(dy), *xp = reinterpret_cast<const T*>(x), *wp = reinterpret_cast<const T*>(w);
#define LLMT_LN(N, W, TH)                                                                                                                      \
  if (s.nv == N && (s.tr == 32) == W && threads <= TH && (TH == 256 || threads > 256)) {                                                       \
    if (aligned) layer_norm_bwd_kernel<T, N, W, true, TH><<<grid, threads, smem, stream>>>(gp, xp, ldx, wp, mean, rstd, reinterpret_cast<T*>(dx), partial, R, D, s.tr); \
    else layer_norm_bwd_kernel<T, N, W, false, TH><<<grid, threads, smem, stream>>>(gp, xp, ldx, wp, mean, rstd, reinterpret_cast<T*>(dx), partial, R, D, s.tr);        \
  }
  LLMT_LN(1, true, 256) LLMT_LN(2, true, 256) LLMT_LN(3, true, 256) LLMT_LN(4, true, 256) LLMT_LN(5, true, 256)
  LLMT_LN(4, false, 256) LLMT_LN(4, false, 512)
#undef LLMT_LN
  if (cudaGetLastError() != cudaSuccess) return -3;
  layer_norm_colsum_kernel<T><<<(2 * D + 31) / 32, 1024, 0, stream>>>(partial, reinterpret_cast<T*>(dw), reinterpret_cast<T*>(db), grid, D);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// Rows of `partial` that a backward may write, whatever the alignment of its operands.
template <typename T>
static int ln_partials(int R, int D) {
  const int a = ln_bwd_grid<T>(R, ln_bwd_shape(ln_vecs<T>(D, true))), b = ln_bwd_grid<T>(R, ln_bwd_shape(ln_vecs<T>(D, false)));
  return a > b ? a : b;
}

}  // namespace llmt

using namespace llmt;

// Widest rows: that start anywhere, or (`whole`: 16-byte granules) whose rows and weights all start on a granule.
extern "C" int llmt_layer_norm_max_width(int f32, int whole) {
  const int V = f32 ? Granule<float>::V : Granule<__nv_bfloat16>::V;
  return kLnMaxVecs * V - (whole ? 0 : 2 * (V - 1));
}
extern "C" int llmt_layer_norm_fwd(const void* x, int64_t ldx, const void* w, const void* b, void* y, float* mean, float* rstd, int R, int D,
                                   float eps, int f32, cudaStream_t stream) {
  return f32 ? ln_fwd<float>(x, ldx, w, b, y, mean, rstd, R, D, eps, stream) : ln_fwd<__nv_bfloat16>(x, ldx, w, b, y, mean, rstd, R, D, eps, stream);
}
extern "C" int llmt_layer_norm_bwd_partials(int R, int D, int f32) { return f32 ? ln_partials<float>(R, D) : ln_partials<__nv_bfloat16>(R, D); }
extern "C" int llmt_layer_norm_bwd(const void* dy, const void* x, int64_t ldx, const void* w, const float* mean, const float* rstd, void* dx,
                                   float* partial, int P, void* dw, void* db, int R, int D, int f32, cudaStream_t stream) {
  return f32 ? ln_bwd<float>(dy, x, ldx, w, mean, rstd, dx, partial, P, dw, db, R, D, stream)
             : ln_bwd<__nv_bfloat16>(dy, x, ldx, w, mean, rstd, dx, partial, P, dw, db, R, D, stream);
}
