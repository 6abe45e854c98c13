// Rotary positions for sm_100a: the rotation of part of a head, the same behind a per-head RMS norm, and the tables with frequencies scaled
// for long contexts. bf16 or fp32 storage, fp32 arithmetic, angles in 64 bits.
// (reference call sites: llmtuner/models/qwen/qwen3_5_moe/rotary.py:1-108, llmtuner/models/deepseek/deepseek_v4/rotary.py:9-100)
//
// Of a head of `d` channels the 2 P from `off` on rotate, the others pass. Pair j is (off + j, off + P + j) in the half layout and
// (off + 2 j, off + 2 j + 1) in the interleaved one:  y1 = x1 cos_j - x2 sin_j,  y2 = x2 cos_j + x1 sin_j;  the gradient is the rotation back.
// Heads lie `head_stride` and tokens `tok_stride` elements apart, tables [T][P] with a row stride of their own.
#include <initializer_list>
#include "kernels.h"
#include "vec_io.cuh"

namespace llmt {

int sm_count();

struct RopeShape {
  int T, d, off, P, interleaved;
  const float *cosb, *sinb;
  int64_t ldt;
  float sign;                    // 1 rotates, -1 rotates back
};
struct RopeOperand {
  const void* x;
  void* y;
  int64_t x_tok, x_head, y_tok, y_head;
  int H;
};

// V table values from column j on; 16-byte loads where `wide` (base and row stride on 16 bytes) and the column allow them.
template <int V>
__device__ __forceinline__ void load_table(const float* t, int j, bool wide, float* f) {
  if (V % 4 == 0 && wide && (j & 3) == 0) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float4 q = *reinterpret_cast<const float4*>(t + j + 4 * i);
      f[4 * i] = q.x; f[4 * i + 1] = q.y; f[4 * i + 2] = q.z; f[4 * i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = t[j + i];
  }
}

// ------------------------------------------------------------------------------------------ rotation
// A thread owns one unit of one token and walks over the heads of a share of them, so its cos and sin are read once: a pair of vectors (half
// layout), a vector that holds whole pairs (interleaved), or a vector that passes. Neighbouring threads own neighbouring units, then
// neighbouring heads, so a warp touches one run of memory. V values per vector by divisibility and alignment (rope_vec); at V = 1 an
// interleaved unit is the two halves of a pair. Bound by memory.
template <typename T, int V, bool PAIRS>
__global__ void __launch_bounds__(256) rope_kernel(RopeShape s, RopeOperand a, RopeOperand b, int units, int shares, int tokens_per_block) {
  constexpr bool SCALAR_PAIRS = PAIRS && V == 1;
  constexpr int N = PAIRS ? V / 2 : V;                  // table values of a unit
  const int per_token = units * shares;
  const int lt = threadIdx.x / per_token, r = threadIdx.x - lt * per_token;
  const int64_t t = (int64_t)blockIdx.x * tokens_per_block + lt;
  if (lt >= tokens_per_block || t >= s.T) return;
  const bool wide = !((reinterpret_cast<uintptr_t>(s.cosb) | reinterpret_cast<uintptr_t>(s.sinb)) & 15) && (s.ldt & 3) == 0;
  // blocks may have fewer threads than a token has units and shares: then a thread takes several (the loop runs once otherwise)
  for (int w = r; w < per_token; w += tokens_per_block == 1 ? blockDim.x : per_token) {
    const int share = w / units, u = w - share * units;
    const int rot_units = PAIRS ? (SCALAR_PAIRS ? s.P : 2 * s.P / V) : s.P / V;
    const bool rot = u < rot_units;
    int c0, c1 = 0;                                     // columns of the unit's vector(s)
    if (rot) {
      c0 = PAIRS ? s.off + u * (SCALAR_PAIRS ? 2 : V) : s.off + u * V;
      c1 = SCALAR_PAIRS ? c0 + 1 : c0 + s.P;
    } else {
      c0 = (u - rot_units) * V;
      if (c0 >= s.off) c0 += 2 * s.P;
    }
    float c[SCALAR_PAIRS ? 1 : N > 0 ? N : 1], n[SCALAR_PAIRS ? 1 : N > 0 ? N : 1];
    if (rot) {
      const int j = PAIRS ? (SCALAR_PAIRS ? u : u * N) : u * V;
      load_table<SCALAR_PAIRS ? 1 : (N > 0 ? N : 1)>(s.cosb + t * s.ldt, j, wide, c);
      load_table<SCALAR_PAIRS ? 1 : (N > 0 ? N : 1)>(s.sinb + t * s.ldt, j, wide, n);
#pragma unroll
      for (int i = 0; i < (SCALAR_PAIRS ? 1 : N > 0 ? N : 1); ++i) n[i] *= s.sign;
    }
    const int heads = a.H + b.H;
#pragma unroll 4
    for (int h = share; h < heads; h += shares) {
      const bool first = h < a.H;
      const int hh = first ? h : h - a.H;
      const T* px = first ? reinterpret_cast<const T*>(a.x) + t * a.x_tok + hh * a.x_head : reinterpret_cast<const T*>(b.x) + t * b.x_tok + hh * b.x_head;
      T* py = first ? reinterpret_cast<T*>(a.y) + t * a.y_tok + hh * a.y_head : reinterpret_cast<T*>(b.y) + t * b.y_tok + hh * b.y_head;
      if (!rot) {
        Raw<T, V> raw;
        raw.load(px + c0);
        raw.store(py + c0);
        continue;
      }
      float x1[V], y1[V];
      load_vec<T, V>(px + c0, x1);
      if constexpr (PAIRS && !SCALAR_PAIRS) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          y1[2 * i] = x1[2 * i] * c[i] - x1[2 * i + 1] * n[i];
          y1[2 * i + 1] = x1[2 * i + 1] * c[i] + x1[2 * i] * n[i];
        }
        store_vec<T, V>(py + c0, y1);
      } else {
        float x2[V], y2[V];
        load_vec<T, V>(px + c1, x2);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          y1[i] = x1[i] * c[i] - x2[i] * n[i];
          y2[i] = x2[i] * c[i] + x1[i] * n[i];
        }
        store_vec<T, V>(py + c0, y1);
        store_vec<T, V>(py + c1, y2);
      }
    }
  }
}

static bool div_by(int v, std::initializer_list<int64_t> xs) {
  for (int64_t x : xs)
    if (x % v) return false;
  return true;
}
// The widest vector (at most `most` values) that divides the parts of a head and fits every address.
static int rope_vec(const RopeShape& s, const RopeOperand& a, const RopeOperand& b, int size, int most) {
  for (int v = most; v > 1; v /= 2) {
    const int64_t part = s.interleaved ? 2 * s.P : s.P;
    if (!div_by(v, {part, s.off, s.d, a.x_tok, a.x_head, a.y_tok, a.y_head})) continue;
    if (b.H && !div_by(v, {b.x_tok, b.x_head, b.y_tok, b.y_head})) continue;
    const uintptr_t bytes = v * size < 16 ? v * size : 16;
    uintptr_t at = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y);
    if (b.H) at |= reinterpret_cast<uintptr_t>(b.x) | reinterpret_cast<uintptr_t>(b.y);
    if (at % bytes == 0) return v;
  }
  return 1;
}

template <typename T, int V, bool PAIRS>
static int rope_launch(const RopeShape& s, const RopeOperand& a, const RopeOperand& b, cudaStream_t stream) {
  const int rot = PAIRS ? (V == 1 ? s.P : 2 * s.P / V) : s.P / V;
  const int units = rot + (s.d - 2 * s.P) / V, heads = a.H + b.H;
  const int shares = heads >= 16 ? heads / 4 : heads >= 2 ? (heads + 1) / 2 : 1;        // up to four heads per thread
  const int per_token = units * shares;
  const int tokens = per_token >= 256 ? 1 : 256 / per_token;
  const int threads = per_token >= 256 ? 256 : tokens * per_token;
  const int64_t blocks = ((int64_t)s.T + tokens - 1) / tokens;
  if (blocks > 0x7fffffff) return -10;
  rope_kernel<T, V, PAIRS><<<(int)blocks, threads, 0, stream>>>(s, a, b, units, shares, tokens);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
template <typename T>
static int rope_dispatch(const RopeShape& s, const RopeOperand& a, const RopeOperand& b, cudaStream_t stream) {
  const int v = rope_vec(s, a, b, sizeof(T), 16 / (int)sizeof(T));
#define LLMT_ROPE(N) \
  if (v == N) return s.interleaved ? rope_launch<T, N, true>(s, a, b, stream) : rope_launch<T, N, false>(s, a, b, stream);
  if constexpr (sizeof(T) == 2) { LLMT_ROPE(8) }
  LLMT_ROPE(4) LLMT_ROPE(2) LLMT_ROPE(1)
#undef LLMT_ROPE
  return -4;
}

// ------------------------------------------------------------------------------------------ per-head norm + rotation
// n = x * rsqrt(mean x^2 + eps) * (w + shift) (no weight: factor 1), then the rotation. The gradient: g = rotation back of dy,
//   dx = r (g w' - x r^2 mean(g w' x)),  dw = sum over tokens and heads of g x r;  r is computed again from x, which is read anyway.
// Wide form: a group of G lanes per head, 8 channels per lane (16 bytes of bf16); the partner of a lane's channels is in the lane P / 8 away
// (half layout) and comes by shuffle, or in the lane itself (interleaved). A group walks over a share of one token's heads, so tables and
// weights are loaded once per token and operand. Needs d, off and P (interleaved: 2 P) divisible by 8, d <= 256 and 16-byte addresses.
// General form: a warp per head, the normalised head in shared memory, any d <= 1024.
struct NormOperand {
  const void *x, *w;
  void* y;                       // forward: the result; backward: dx
  const void* dy;                // backward only
  int64_t x_tok, x_head, y_tok, y_head, dy_tok, dy_head;
  int H;
};
struct NormArgs {
  RopeShape s;
  NormOperand q, k;
  float eps, shift;
  float* partial;                // backward: [grid][2][d]
};

template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Rotation of a lane's 8 channels: `mine` in, out in place. rot: 0 passes, 1 first half, 2 second half, 3 interleaved.
template <int G>
__device__ __forceinline__ void rotate_lane(float* v, int rot, int partner, const float* c, const float* n) {
  float o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xffffffffu, v[i], partner, G);
  if (rot == 3) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = v[2 * i], b = v[2 * i + 1];
      v[2 * i] = a * c[i] - b * n[i];
      v[2 * i + 1] = b * c[i] + a * n[i];
    }
  } else if (rot == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * c[i] - o[i] * n[i];
  } else if (rot == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * c[i] + o[i] * n[i];
  }
}

// Where lane `g` of a group stands: its kind of rotation, partner and first table column.
struct LanePlace { int rot, partner, col; };
__device__ __forceinline__ LanePlace lane_place(const RopeShape& s, int g) {
  const int c = g * 8;
  LanePlace p{0, g, 0};
  if (c < s.off || c >= s.off + 2 * s.P) return p;
  if (s.interleaved) return {3, g, (c - s.off) / 2};
  const int step = s.P / 8;
  if (c < s.off + s.P) return {1, g + step, c - s.off};
  return {2, g - step, c - s.off - s.P};
}
__device__ __forceinline__ void lane_tables(const RopeShape& s, const LanePlace& p, int64_t t, bool wide, float* c, float* n) {
#pragma unroll
  for (int i = 0; i < 8; ++i) { c[i] = 1.f; n[i] = 0.f; }
  if (p.rot == 0) return;
  if (p.rot == 3) {
    load_table<4>(s.cosb + t * s.ldt, p.col, wide, c);
    load_table<4>(s.sinb + t * s.ldt, p.col, wide, n);
  } else {
    load_table<8>(s.cosb + t * s.ldt, p.col, wide, c);
    load_table<8>(s.sinb + t * s.ldt, p.col, wide, n);
  }
}
template <typename T>
__device__ __forceinline__ void lane_weight(const void* w, int c, int d, float shift, float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = 1.f;
  if (w == nullptr || c >= d) return;
  load_vec<T, 8>(reinterpret_cast<const T*>(w) + c, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] += shift;
}

template <typename T, int G>
__global__ void __launch_bounds__(256) qk_norm_rope_part_fwd_kernel(const __grid_constant__ NormArgs a, int shares) {
  const RopeShape& s = a.s;
  constexpr int GPB = 256 / G;
  const int g = threadIdx.x % G;
  const int64_t item = (int64_t)blockIdx.x * GPB + threadIdx.x / G;
  int64_t t = item / shares;
  const int share = (int)(item - t * shares);
  const bool live = t < s.T;
  if (!live) t = s.T - 1;                               // the whole warp stays in the shuffles
  const bool in = g * 8 < s.d;
  const bool wide = !((reinterpret_cast<uintptr_t>(s.cosb) | reinterpret_cast<uintptr_t>(s.sinb)) & 15) && (s.ldt & 3) == 0;
  const LanePlace p = lane_place(s, g);
  float c[8], n[8], w[8];
  lane_tables(s, p, t, wide, c, n);
  const float inv_d = 1.f / (float)s.d;
#pragma unroll
  for (int op = 0; op < 2; ++op) {
    const NormOperand& o = op ? a.k : a.q;
    lane_weight<T>(o.w, g * 8, s.d, a.shift, w);
    const int rounds = (o.H + shares - 1) / shares;     // equal for all groups of a warp
#pragma unroll 2
    for (int i = 0; i < rounds; ++i) {
      const int h = i * shares + share;
      const bool on = in && h < o.H;
      float x[8];
      Raw<T, 8> raw;
      raw.zero();
      if (on) raw.load(reinterpret_cast<const T*>(o.x) + t * o.x_tok + h * o.x_head + g * 8);
      raw.get(x);
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sq += x[j] * x[j];
      const float r = rsqrtf(lanes_sum<G>(sq) * inv_d + a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= r * w[j];
      rotate_lane<G>(x, p.rot, p.partner, c, n);
      if (on && live) store_vec<T, 8>(reinterpret_cast<T*>(o.y) + t * o.y_tok + h * o.y_head + g * 8, x);
    }
  }
}

template <typename T, int G>
__global__ void __launch_bounds__(256, 3) qk_norm_rope_part_bwd_kernel(const __grid_constant__ NormArgs a, int shares) {
  const RopeShape& s = a.s;
  constexpr int GPB = 256 / G;
  __shared__ float sums[2][G * 8];
  const int g = threadIdx.x % G, grp = threadIdx.x / G;
  const bool in = g * 8 < s.d;
  const bool wide = !((reinterpret_cast<uintptr_t>(s.cosb) | reinterpret_cast<uintptr_t>(s.sinb)) & 15) && (s.ldt & 3) == 0;
  const LanePlace p = lane_place(s, g);
  const float inv_d = 1.f / (float)s.d;
  float dw[2][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[0][i] = dw[1][i] = 0.f;
  const int64_t items = (int64_t)s.T * shares, step = (int64_t)gridDim.x * GPB;
  const int64_t base = (int64_t)blockIdx.x * GPB;
  for (int64_t b0 = base; b0 < items; b0 += step) {     // uniform in the block
    const int64_t item = b0 + grp;
    const bool live = item < items;
    const int64_t t = (live ? item : items - 1) / shares;
    const int share = (int)((live ? item : items - 1) - t * shares);
    float c[8], n[8], w[8];
    lane_tables(s, p, t, wide, c, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = -n[i];
#pragma unroll
    for (int op = 0; op < 2; ++op) {
      const NormOperand& o = op ? a.k : a.q;
      lane_weight<T>(o.w, g * 8, s.d, a.shift, w);
      const int rounds = (o.H + shares - 1) / shares;
#pragma unroll 2
      for (int i = 0; i < rounds; ++i) {
        const int h = i * shares + share;
        const bool on = in && live && h < o.H;
        float x[8], d[8];
        Raw<T, 8> rx, rd;
        rx.zero();
        rd.zero();
        if (on) {
          rx.load(reinterpret_cast<const T*>(o.x) + t * o.x_tok + h * o.x_head + g * 8);
          rd.load(reinterpret_cast<const T*>(o.dy) + t * o.dy_tok + h * o.dy_head + g * 8);
        }
        rx.get(x);
        rd.get(d);
        rotate_lane<G>(d, p.rot, p.partner, c, n);
        float sq = 0.f, dot = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sq += x[j] * x[j];
          dot += d[j] * w[j] * x[j];
        }
#pragma unroll
        for (int m = G / 2; m > 0; m >>= 1) {
          sq += __shfl_xor_sync(0xffffffffu, sq, m);
          dot += __shfl_xor_sync(0xffffffffu, dot, m);
        }
        const float r = rsqrtf(sq * inv_d + a.eps), k = r * r * r * dot * inv_d;
        float out[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          out[j] = r * d[j] * w[j] - x[j] * k;
          if (on) dw[op][j] += d[j] * x[j] * r;          // a masked lane's r may be infinite (eps 0)
        }
        if (on) store_vec<T, 8>(reinterpret_cast<T*>(o.y) + t * o.y_tok + h * o.y_head + g * 8, out);
      }
    }
  }
  if (a.partial == nullptr) return;
  for (int k = 0; k < GPB; ++k) {                       // the groups of a block in their order
    if (grp == k && in) {
#pragma unroll
      for (int op = 0; op < 2; ++op)
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[op][g * 8 + j] = k == 0 ? dw[op][j] : sums[op][g * 8 + j] + dw[op][j];
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 2 * s.d; i += 256) a.partial[(int64_t)blockIdx.x * 2 * s.d + i] = i < s.d ? sums[0][i] : sums[1][i - s.d];
}

// General form. Four warps per block, each with one head at a time; buf: the head before the rotation.
constexpr int kAnyWarps = 4;
__device__ __forceinline__ float rotated(const RopeShape& s, const float* buf, int c, int64_t t, float sign) {
  const int j = c - s.off;
  if (j < 0 || j >= 2 * s.P) return buf[c];
  const int at = s.interleaved ? j >> 1 : (j < s.P ? j : j - s.P);
  const bool second = s.interleaved ? j & 1 : j >= s.P;
  const int partner = s.interleaved ? (second ? c - 1 : c + 1) : (second ? c - s.P : c + s.P);
  const float co = s.cosb[t * s.ldt + at], si = sign * s.sinb[t * s.ldt + at];
  return second ? buf[c] * co + buf[partner] * si : buf[c] * co - buf[partner] * si;
}

template <typename T, bool BWD>
__global__ void __launch_bounds__(32 * kAnyWarps) qk_norm_rope_any_kernel(const __grid_constant__ NormArgs a) {
  extern __shared__ float smem[];
  const RopeShape& s = a.s;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, d = s.d;
  float* buf = smem + wid * (BWD ? 3 * d : d);          // BWD: dy | sums of dwq | sums of dwk
  if (BWD)
    for (int c = lane; c < 2 * d; c += 32) buf[d + c] = 0.f;
  const int heads = a.q.H + a.k.H;
  const int64_t items = (int64_t)s.T * heads;
  for (int64_t item = (int64_t)blockIdx.x * kAnyWarps + wid; item < items; item += (int64_t)gridDim.x * kAnyWarps) {
    const int64_t t = item / heads;
    int h = (int)(item - t * heads);
    const int op = h >= a.q.H;
    const NormOperand& o = op ? a.k : a.q;
    if (op) h -= a.q.H;
    const T* px = reinterpret_cast<const T*>(o.x) + t * o.x_tok + h * o.x_head;
    T* py = reinterpret_cast<T*>(o.y) + t * o.y_tok + h * o.y_head;
    const T* pw = reinterpret_cast<const T*>(o.w);
    auto weight = [&](int c) { float f = 1.f; if (pw != nullptr) { load_vec<T, 1>(pw + c, &f); f += a.shift; } return f; };
    float sq = 0.f;
    __syncwarp();                                       // the head before has been read from the buffer
    for (int c = lane; c < d; c += 32) {
      float x;
      load_vec<T, 1>(px + c, &x);
      sq += x * x;
      if (BWD) load_vec<T, 1>(reinterpret_cast<const T*>(o.dy) + t * o.dy_tok + h * o.dy_head + c, buf + c);
      else buf[c] = x;
    }
    const float r = rsqrtf(warp_sum(sq) / (float)d + a.eps);
    __syncwarp();
    if (!BWD) {
      for (int c = lane; c < d; c += 32) buf[c] *= r * weight(c);
      __syncwarp();
      for (int c = lane; c < d; c += 32) {
        const float y = rotated(s, buf, c, t, 1.f);
        store_vec<T, 1>(py + c, &y);
      }
    } else {
      float dot = 0.f;
      for (int c = lane; c < d; c += 32) {
        float x;
        load_vec<T, 1>(px + c, &x);
        const float g = rotated(s, buf, c, t, -1.f);
        dot += g * weight(c) * x;
        buf[d + op * d + c] += g * x * r;
      }
      const float k = r * r * r * warp_sum(dot) / (float)d;
      for (int c = lane; c < d; c += 32) {
        float x;
        load_vec<T, 1>(px + c, &x);
        const float out = r * rotated(s, buf, c, t, -1.f) * weight(c) - x * k;
        store_vec<T, 1>(py + c, &out);
      }
    }
  }
  if (!BWD || a.partial == nullptr) return;
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * d; i += blockDim.x) {
    float v = 0.f;
    for (int w = 0; w < kAnyWarps; ++w) v += smem[w * 3 * d + d + i];
    a.partial[(int64_t)blockIdx.x * 2 * d + i] = v;
  }
}

// dwq | dwk in T from partial [P][2 d], in a fixed order; either may be absent.
template <typename T>
__global__ void __launch_bounds__(1024) qk_weight_sum_kernel(const float* __restrict__ partial, T* __restrict__ dwq, T* __restrict__ dwk, int P, int d) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < 2 * d) {
#pragma unroll 4
    for (int q = wid; q < P; q += 32) v += partial[(int64_t)q * 2 * d + c];
  }
  part[wid][lane] = v;
  __syncthreads();
  v = warp_sum(part[lane][wid]);
  const int oc = blockIdx.x * 32 + wid;
  if (lane != 0 || oc >= 2 * d) return;
  T* out = oc < d ? dwq : dwk;
  if (out != nullptr) store_vec<T, 1>(out + (oc < d ? oc : oc - d), &v);
}

static bool norm_wide(const NormArgs& a, int size, bool bwd) {
  const RopeShape& s = a.s;
  if (s.d > 256 || !div_by(8, {s.d, s.off, s.interleaved ? 2 * s.P : s.P})) return false;
  for (const NormOperand* o : {&a.q, &a.k}) {
    if (!o->H) continue;
    uintptr_t at = reinterpret_cast<uintptr_t>(o->x) | reinterpret_cast<uintptr_t>(o->y) | reinterpret_cast<uintptr_t>(o->w);
    if (!div_by(16 / size, {o->x_tok, o->x_head, o->y_tok, o->y_head})) return false;
    if (bwd) {
      at |= reinterpret_cast<uintptr_t>(o->dy);
      if (!div_by(16 / size, {o->dy_tok, o->dy_head})) return false;
    }
    if (at & 15) return false;
  }
  return true;
}
// Groups that share a token's heads: two to four heads per group and operand keep loads in flight without reading the tables too often.
static int norm_shares(const NormArgs& a) {
  const int h = a.q.H > a.k.H ? a.q.H : a.k.H;
  return h >= 8 ? h / 4 : h >= 2 ? h / 2 : 1;
}
static int norm_bwd_grid(const NormArgs& a, bool wide) {
  const int64_t items = wide ? (int64_t)a.s.T * norm_shares(a) : (int64_t)a.s.T * (a.q.H + a.k.H);
  const int G = a.s.d > 128 ? 32 : a.s.d > 64 ? 16 : 8;
  const int64_t need = wide ? (items + 256 / G - 1) / (256 / G) : (items + kAnyWarps - 1) / kAnyWarps;
  const int64_t most = (int64_t)sm_count() * (wide ? 3 : a.s.d <= 512 ? 8 : 4);
  return (int)(need < most ? need : most);
}

template <typename T>
static int norm_fwd(const NormArgs& a, cudaStream_t stream) {
  if (norm_wide(a, sizeof(T), false)) {
    const int G = a.s.d > 128 ? 32 : a.s.d > 64 ? 16 : 8, shares = norm_shares(a);
    const int64_t blocks = ((int64_t)a.s.T * shares + 256 / G - 1) / (256 / G);
    if (blocks > 0x7fffffff) return -10;
    if (G == 32) qk_norm_rope_part_fwd_kernel<T, 32><<<(int)blocks, 256, 0, stream>>>(a, shares);
    else if (G == 16) qk_norm_rope_part_fwd_kernel<T, 16><<<(int)blocks, 256, 0, stream>>>(a, shares);
    else qk_norm_rope_part_fwd_kernel<T, 8><<<(int)blocks, 256, 0, stream>>>(a, shares);
  } else {
    const int64_t items = (int64_t)a.s.T * (a.q.H + a.k.H), need = (items + kAnyWarps - 1) / kAnyWarps;
    const int64_t most = (int64_t)sm_count() * 64;
    qk_norm_rope_any_kernel<T, false><<<(int)(need < most ? need : most), 32 * kAnyWarps, kAnyWarps * a.s.d * sizeof(float), stream>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
template <typename T>
static int norm_bwd(const NormArgs& a, int P, void* dwq, void* dwk, cudaStream_t stream) {
  const bool wide = norm_wide(a, sizeof(T), true);
  const int grid = norm_bwd_grid(a, wide);
  if (a.partial != nullptr && grid > P) return -10;
  if (wide) {
    const int shares = norm_shares(a);
    if (a.s.d > 128) qk_norm_rope_part_bwd_kernel<T, 32><<<grid, 256, 0, stream>>>(a, shares);
    else if (a.s.d > 64) qk_norm_rope_part_bwd_kernel<T, 16><<<grid, 256, 0, stream>>>(a, shares);
    else qk_norm_rope_part_bwd_kernel<T, 8><<<grid, 256, 0, stream>>>(a, shares);
  } else {
    qk_norm_rope_any_kernel<T, true><<<grid, 32 * kAnyWarps, kAnyWarps * 3 * a.s.d * sizeof(float), stream>>>(a);
  }
  if (cudaGetLastError() != cudaSuccess) return -3;
  if (a.partial != nullptr)
    qk_weight_sum_kernel<T><<<(2 * a.s.d + 31) / 32, 1024, 0, stream>>>(a.partial, reinterpret_cast<T*>(dwq), reinterpret_cast<T*>(dwk), grid, a.s.d);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// ------------------------------------------------------------------------------------------ tables
// cos, sin [T][P] of factor-scaled angles position * inv_j. The product is taken in 64 bits, in units of pi, and brought into [-1, 1] there:
// at position 131072 an fp32 angle is off by up to 2^-8 rad. What remains is exact enough in fp32, where sincospif takes over.
constexpr int kMaxFreqs = 256;
struct Freqs { double inv_pi[kMaxFreqs]; };            // inv_j / pi
template <bool VEC>
__global__ void __launch_bounds__(256) rope_tables_kernel(const int64_t* __restrict__ pos, const __grid_constant__ Freqs f, float factor,
                                                          float* __restrict__ cosb, float* __restrict__ sinb, int64_t T, int P) {
  constexpr int V = VEC ? 4 : 1;
  const int per_row = P / V;
  const int64_t total = T * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / per_row;
    const int j = (int)(i - t * per_row) * V;
    const double p = (double)pos[t];
    float c[V], n[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const double a = p * f.inv_pi[j + v];
      sincospif((float)(a - 2.0 * rint(0.5 * a)), n + v, c + v);
      c[v] *= factor;
      n[v] *= factor;
    }
    if constexpr (VEC) {
      *reinterpret_cast<float4*>(cosb + t * P + j) = make_float4(c[0], c[1], c[2], c[3]);
      *reinterpret_cast<float4*>(sinb + t * P + j) = make_float4(n[0], n[1], n[2], n[3]);
    } else {
      cosb[t * P + j] = c[0];
      sinb[t * P + j] = n[0];
    }
  }
}

static bool rope_shape_ok(const RopeShape& s) { return s.T >= 0 && s.d > 0 && s.P > 0 && s.off >= 0 && s.off + 2 * s.P <= s.d && s.ldt >= s.P; }

}  // namespace llmt

using namespace llmt;

extern "C" int llmt_rope(const LlmtRopeShape* sh, const LlmtHeads* a, const LlmtHeads* b, int f32, cudaStream_t stream) {
  const RopeShape s{sh->T, sh->d, sh->off, sh->P, sh->interleaved, sh->cosb, sh->sinb, sh->ldt, sh->sign};
  if (!rope_shape_ok(s)) return -10;
  const RopeOperand x{a->x, a->y, a->x_tok, a->x_head, a->y_tok, a->y_head, a->H};
  RopeOperand y{nullptr, nullptr, 0, 0, 0, 0, 0};
  if (b != nullptr) y = RopeOperand{b->x, b->y, b->x_tok, b->x_head, b->y_tok, b->y_head, b->H};
  if (s.T == 0 || x.H + y.H == 0) return 0;
  return f32 ? rope_dispatch<float>(s, x, y, stream) : rope_dispatch<__nv_bfloat16>(s, x, y, stream);
}

static NormArgs norm_args(const LlmtRopeShape* sh, const LlmtHeads* q, const LlmtHeads* k, float eps, float shift, float* partial) {
  NormArgs a{};
  a.s = RopeShape{sh->T, sh->d, sh->off, sh->P, sh->interleaved, sh->cosb, sh->sinb, sh->ldt, 1.f};
  auto take = [](const LlmtHeads* h) {
    return h == nullptr ? NormOperand{}
                        : NormOperand{h->x, h->w, h->y, h->dy, h->x_tok, h->x_head, h->y_tok, h->y_head, h->dy_tok, h->dy_head, h->H};
  };
  a.q = take(q);
  a.k = take(k);
  a.eps = eps;
  a.shift = shift;
  a.partial = partial;
  return a;
}
extern "C" int llmt_qk_norm_rope_part_max_dim() { return 1024; }
extern "C" int llmt_qk_norm_rope_part_fwd(const LlmtRopeShape* sh, const LlmtHeads* q, const LlmtHeads* k, float eps, float shift, int f32,
                                          cudaStream_t stream) {
  const NormArgs a = norm_args(sh, q, k, eps, shift, nullptr);
  if (!rope_shape_ok(a.s) || a.s.d > 1024) return -10;
  if (a.s.T == 0 || a.q.H + a.k.H == 0) return 0;
  return f32 ? norm_fwd<float>(a, stream) : norm_fwd<__nv_bfloat16>(a, stream);
}
// Rows of `partial` ([rows][2][d]) that the backward writes for any alignment of its operands.
extern "C" int llmt_qk_norm_rope_part_partials(int T, int Hq, int Hk, int d) {
  NormArgs a{};
  a.s.T = T; a.s.d = d; a.q.H = Hq; a.k.H = Hk;
  const int w = norm_bwd_grid(a, true), n = norm_bwd_grid(a, false);
  return w > n ? w : n;
}
extern "C" int llmt_qk_norm_rope_part_bwd(const LlmtRopeShape* sh, const LlmtHeads* q, const LlmtHeads* k, float eps, float shift, float* partial, int P,
                                          void* dwq, void* dwk, int f32, cudaStream_t stream) {
  const NormArgs a = norm_args(sh, q, k, eps, shift, partial);
  if (!rope_shape_ok(a.s) || a.s.d > 1024 || a.s.T == 0 || a.q.H + a.k.H == 0) return -10;
  return f32 ? norm_bwd<float>(a, P, dwq, dwk, stream) : norm_bwd<__nv_bfloat16>(a, P, dwq, dwk, stream);
}

extern "C" int llmt_rope_tables(const int64_t* pos, const double* inv, int P, double factor, float* cosb, float* sinb, int64_t T, cudaStream_t stream) {
  if (P <= 0 || P > kMaxFreqs || T < 0) return -10;
  if (T == 0) return 0;
  Freqs f{};
  for (int j = 0; j < P; ++j) f.inv_pi[j] = inv[j] / 3.14159265358979323846;
  const bool vec = P % 4 == 0 && !((reinterpret_cast<uintptr_t>(cosb) | reinterpret_cast<uintptr_t>(sinb)) & 15);
  const int64_t need = (T * (vec ? P / 4 : P) + 255) / 256, most = (int64_t)sm_count() * 32;
  const int grid = (int)(need < most ? need : most);
  if (vec) rope_tables_kernel<true><<<grid, 256, 0, stream>>>(pos, f, (float)factor, cosb, sinb, T, P);
  else rope_tables_kernel<false><<<grid, 256, 0, stream>>>(pos, f, (float)factor, cosb, sinb, T, P);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
