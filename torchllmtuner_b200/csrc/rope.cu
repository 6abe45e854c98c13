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

// For V channels from c0 on: the factor of the channel and of its partner when rotating by `sign`, and how far away the partner is (0: the channel
// passes).
template <int V>
__device__ __forceinline__ void channel_tables(const RopeShape& s, int c0, int64_t t, float sign, float* c, float* n, int* gap) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int at = c0 + j - s.off;
    c[j] = 1.f;
    n[j] = 0.f;
    gap[j] = 0;
    if (at < 0 || at >= 2 * s.P) continue;
    const bool second = s.interleaved ? at & 1 : at >= s.P;
    const int pair = s.interleaved ? at >> 1 : second ? at - s.P : at, step = s.interleaved ? 1 : s.P;
    c[j] = s.cosb[t * s.ldt + pair];
    n[j] = s.sinb[t * s.ldt + pair] * (second ? sign : -sign);
    gap[j] = second ? -step : step;
  }
}

// ------------------------------------------------------------------------------------------ rotation
// A thread owns one unit of one token in up to four heads, so its cos and sin are read once: a pair of vectors (half layout), a vector that
// holds whole pairs (interleaved), or a vector that passes. Neighbouring threads own neighbouring units, then neighbouring heads, so a warp
// touches one run of memory; the heads of a thread are `shares` apart and all their loads are issued before the first is used. V values per
// vector by divisibility and alignment (rope_vec); at V = 1 an interleaved unit is the two halves of a pair. Bound by memory: 16384 tokens of 32 heads
// of 72 in pairs take 24 us a direction, 6.4 TB/s.
constexpr int kRopeHeads = 4;
struct RopeWork {
  RopeOperand o;
  int shares, tokens;            // threads of one token and unit; tokens of a block
};
template <typename T, int V, bool PAIRS>
__global__ void __launch_bounds__(256) rope_kernel(RopeShape s, RopeWork wa, RopeWork wb, int units) {
  constexpr bool SCALAR_PAIRS = PAIRS && V == 1, TWO = !PAIRS || SCALAR_PAIRS;       // TWO: the pair's members are in two vectors
  constexpr int N = SCALAR_PAIRS ? 1 : PAIRS ? V / 2 : V;                              // table values of a unit
  const RopeWork& k = blockIdx.y ? wb : wa;
  const int per_token = units * k.shares;
  const int lt = per_token >= 256 ? 0 : threadIdx.x / per_token;
  const int64_t t = (int64_t)blockIdx.x * k.tokens + lt;
  if (lt >= k.tokens || t >= s.T) return;
  const bool wide = !((reinterpret_cast<uintptr_t>(s.cosb) | reinterpret_cast<uintptr_t>(s.sinb)) & 15) && (s.ldt & 3) == 0;
  const int rot_units = PAIRS ? (SCALAR_PAIRS ? s.P : 2 * s.P / V) : s.P / V;
  const int64_t x_step = k.o.x_head * k.shares, y_step = k.o.y_head * k.shares;
  // one round unless a token has more than 256 threads' work
  for (int w = threadIdx.x - lt * per_token; w < per_token; w += 256) {
    const int share = w / units, u = w - share * units;
    const bool rot = u < rot_units;
    int c0, gap = 0;                                    // first column, distance to the partner's vector
    if (rot) {
      c0 = s.off + u * (SCALAR_PAIRS ? 2 : V);
      gap = SCALAR_PAIRS ? 1 : s.P;
    } else {
      c0 = (u - rot_units) * V;
      if (c0 >= s.off) c0 += 2 * s.P;
    }
    const T* px = reinterpret_cast<const T*>(k.o.x) + t * k.o.x_tok + share * k.o.x_head + c0;
    T* py = reinterpret_cast<T*>(k.o.y) + t * k.o.y_tok + share * k.o.y_head + c0;
    Raw<T, V> r1[kRopeHeads], r2[TWO ? kRopeHeads : 1];
#pragma unroll
    for (int i = 0; i < kRopeHeads; ++i)
      if (share + i * k.shares < k.o.H) {
        r1[i].load(px + i * x_step);
        if (TWO && rot) r2[TWO ? i : 0].load(px + i * x_step + gap);
      }
    if (!rot) {
#pragma unroll
      for (int i = 0; i < kRopeHeads; ++i)
        if (share + i * k.shares < k.o.H) r1[i].store(py + i * y_step);
      continue;
    }
    float c[N], n[N];
    load_table<N>(s.cosb + t * s.ldt, u * N, wide, c);
    load_table<N>(s.sinb + t * s.ldt, u * N, wide, n);
#pragma unroll
    for (int i = 0; i < N; ++i) n[i] *= s.sign;
#pragma unroll
    for (int i = 0; i < kRopeHeads; ++i) {
      if (share + i * k.shares >= k.o.H) continue;
      float x1[V], y1[V];
      r1[i].get(x1);
      if constexpr (TWO) {
        float x2[V], y2[V];
        r2[i].get(x2);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          y1[j] = x1[j] * c[j] - x2[j] * n[j];
          y2[j] = x2[j] * c[j] + x1[j] * n[j];
        }
        store_vec<T, V>(py + i * y_step, y1);
        store_vec<T, V>(py + i * y_step + gap, y2);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          y1[2 * j] = x1[2 * j] * c[j] - x1[2 * j + 1] * n[j];
          y1[2 * j + 1] = x1[2 * j + 1] * c[j] + x1[2 * j] * n[j];
        }
        store_vec<T, V>(py + i * y_step, y1);
      }
    }
  }
}

// Pairs that straddle vectors (half layout with P or off no multiple of the vector, interleaved pairs that start on an odd channel): a thread owns V
// channels in a row, which it reads and writes as vectors, and reads their partners one by one (they are in L1). 9000 x 20 heads of 80, 34 rotated: 20 us
// a direction in bf16 (floor 9), 24 in fp32 (18).
template <typename T, int V>
__global__ void __launch_bounds__(256) rope_gather_kernel(RopeShape s, RopeWork wa, RopeWork wb) {
  const RopeWork& k = blockIdx.y ? wb : wa;
  const int units = s.d / V, per_token = units * k.shares;
  const int lt = per_token >= 256 ? 0 : threadIdx.x / per_token;
  const int64_t t = (int64_t)blockIdx.x * k.tokens + lt;
  if (lt >= k.tokens || t >= s.T) return;
  const int64_t x_step = k.o.x_head * k.shares, y_step = k.o.y_head * k.shares;
  for (int w = threadIdx.x - lt * per_token; w < per_token; w += 256) {
    const int share = w / units, c0 = (w - share * units) * V;
    const T* px = reinterpret_cast<const T*>(k.o.x) + t * k.o.x_tok + share * k.o.x_head + c0;
    T* py = reinterpret_cast<T*>(k.o.y) + t * k.o.y_tok + share * k.o.y_head + c0;
    Raw<T, V> r[kRopeHeads];
#pragma unroll
    for (int i = 0; i < kRopeHeads; ++i)
      if (share + i * k.shares < k.o.H) r[i].load(px + i * x_step);
    float c[V], n[V];
    int gap[V];
    channel_tables<V>(s, c0, t, s.sign, c, n, gap);
#pragma unroll
    for (int i = 0; i < kRopeHeads; ++i) {
      if (share + i * k.shares >= k.o.H) continue;
      float x[V];
      r[i].get(x);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (gap[j] == 0) continue;                       // passes
        float q;
        load_vec<T, 1>(px + i * x_step + j + gap[j], &q);
        x[j] = x[j] * c[j] + q * n[j];
      }
      store_vec<T, V>(py + i * y_step, x);
    }
  }
}

static bool div_by(int v, std::initializer_list<int64_t> xs) {
  for (int64_t x : xs)
    if (x % v) return false;
  return true;
}
// The widest vector (at most `most` values) that divides a head and fits every address, and, with `pairs`, the parts of a head as well.
static int rope_vec(const RopeShape& s, const RopeOperand& a, const RopeOperand& b, int size, int most, bool pairs) {
  for (int v = most; v > 1; v /= 2) {
    const int64_t part = s.interleaved ? 2 * s.P : s.P;
    if (pairs && !div_by(v, {part, s.off})) continue;
    if (!div_by(v, {s.d, a.x_tok, a.x_head, a.y_tok, a.y_head})) continue;
    if (b.H && !div_by(v, {b.x_tok, b.x_head, b.y_tok, b.y_head})) continue;
    const uintptr_t bytes = v * size < 16 ? v * size : 16;
    uintptr_t at = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y);
    if (b.H) at |= reinterpret_cast<uintptr_t>(b.x) | reinterpret_cast<uintptr_t>(b.y);
    if (at % bytes == 0) return v;
  }
  return 1;
}

// GATHER: rope_gather_kernel, else rope_kernel with pairs side by side (PAIRS) or in halves.
template <typename T, int V, bool PAIRS, bool GATHER>
static int rope_launch(const RopeShape& s, const RopeOperand& a, const RopeOperand& b, cudaStream_t stream) {
  const int units = GATHER ? s.d / V : (PAIRS ? (V == 1 ? s.P : 2 * s.P / V) : s.P / V) + (s.d - 2 * s.P) / V;
  int64_t blocks = 0;
  auto work = [&](const RopeOperand& o) {
    RopeWork w{o, (o.H + kRopeHeads - 1) / kRopeHeads, 1};
    if (o.H == 0) return w;
    // few tokens: one head per thread, so that the machine is filled first
    if ((int64_t)s.T * units * w.shares < (int64_t)sm_count() * 1024) w.shares = o.H;
    if (units * w.shares < 256) w.tokens = 256 / (units * w.shares);
    const int64_t need = ((int64_t)s.T + w.tokens - 1) / w.tokens;
    if (need > blocks) blocks = need;
    return w;
  };
  const RopeWork wa = work(a.H ? a : b), wb = work(b);
  if (blocks > 0x7fffffff) return -10;
  const dim3 grid((int)blocks, a.H && b.H ? 2 : 1);
  if constexpr (GATHER) rope_gather_kernel<T, V><<<grid, 256, 0, stream>>>(s, wa, wb);
  else rope_kernel<T, V, PAIRS><<<grid, 256, 0, stream>>>(s, wa, wb, units);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
template <typename T>
static int rope_dispatch(const RopeShape& s, const RopeOperand& a, const RopeOperand& b, cudaStream_t stream) {
  constexpr int kMost = 16 / (int)sizeof(T);
  const int v = rope_vec(s, a, b, sizeof(T), kMost, true), g = rope_vec(s, a, b, sizeof(T), kMost, false);
  // the partners one by one cost less than narrow vectors for everything (9000 x 20 heads of 80, 34 rotated in halves: 36 us with V = 1)
  if (g >= 4 * v || (g > v && v == 1)) {
#define LLMT_ROPE(N) if (g == N) return rope_launch<T, N, false, true>(s, a, b, stream);
    if constexpr (sizeof(T) == 2) { LLMT_ROPE(8) }
    LLMT_ROPE(4) LLMT_ROPE(2)
#undef LLMT_ROPE
  }
#define LLMT_ROPE(N) \
  if (v == N) return s.interleaved ? rope_launch<T, N, true, false>(s, a, b, stream) : rope_launch<T, N, false, false>(s, a, b, stream);
  if constexpr (sizeof(T) == 2) { LLMT_ROPE(8) }
  LLMT_ROPE(4) LLMT_ROPE(2) LLMT_ROPE(1)
#undef LLMT_ROPE
  return -4;
}

// ------------------------------------------------------------------------------------------ per-head norm + rotation
// n = x * rsqrt(mean x^2 + eps) * (w + shift) (no weight: factor 1), then the rotation. The gradient: g = rotation back of dy,
//   dx = r (g w' - x r^2 mean(g w' x)),  dw = sum over tokens and heads of g x r;  r is computed again from x, which is read anyway.
// Wide form: a group of G lanes per head, 8 channels per lane (16 bytes of bf16). The rotation is linear, so with the weights folded into the
// tables a channel is r (x cw + x' nw), x' its partner: in the lane itself (interleaved), or in the lane P / 8 away (half layout), from where the
// lane's raw 16 bytes come by shuffle. A channel that passes has cw = w, nw = 0. A group takes several heads of one token, so tables and weights are
// loaded once for them and several loads are in flight. Needs d, off and P (interleaved: 2 P) divisible by 8, d <= 256 and 16-byte addresses.
// 8192 tokens of 16 + 4 heads of 256, a quarter rotating: forward 32 us (168 MB, 5.2 TB/s), backward 56 us in two launches (252 MB, 4.5 TB/s). What
// stays is instructions and the chain load - sum - scale at 16 to 32 warps an SM, not DRAM: the next chunk fetched into L2 changed nothing.
// fp32: 52 and 79 us, at the floors (51 and 77). Issue slots: 73 % forward under ncu, DRAM at 45 % of its peak there.
// Gather form (below): any parts of a head up to d = 256. General form: a warp per head, the normalised head in shared memory, any d <= 1024. Both are
// bound by instructions: 8192 tokens of 16 + 4 heads of 200, 50 rotated in halves, bf16: 95 us forward, 99 backward (floors 20 and 30); 4096 tokens of 4 + 4
// heads of 520: 44 and 184 (10 and 16).
struct NormOperand {
  const void *x, *w;
  void* y;                       // forward: the result; backward: dx
  const void* dy;                // backward only
  int64_t x_tok, x_head, y_tok, y_head, dy_tok, dy_head;
  int H;
};
struct NormArgs {
  RopeShape s;
  NormOperand q, k;              // backward: q alone
  float eps, shift;
  float* partial;                // backward: [grid][d]
};

// Where lane `g` of a group stands: its kind of rotation (0 passes, 1 first half, 2 second half, 3 interleaved), partner and first table column.
struct LanePlace { int rot, partner, col; };
template <bool PAIRS>
__device__ __forceinline__ LanePlace lane_place(const RopeShape& s, int g) {
  const int c = g * 8;
  if (c < s.off || c >= s.off + 2 * s.P) return {0, g, 0};
  if (PAIRS) return {3, g, (c - s.off) / 2};
  const int step = s.P / 8;
  if (c < s.off + s.P) return {1, g + step, c - s.off};
  return {2, g - step, c - s.off - s.P};
}
// The factor of each of the lane's channels and of its partner, rotating forwards (sign 1) or back (-1).
template <bool PAIRS>
__device__ __forceinline__ void lane_tables(const RopeShape& s, const LanePlace& p, int64_t t, bool wide, float sign, float2* c, float2* n) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[i] = make_float2(1.f, 1.f);
    n[i] = make_float2(0.f, 0.f);
  }
  if (p.rot == 0) return;
  constexpr int N = PAIRS ? 4 : 8;
  float fc[N], fn[N];
  load_table<N>(s.cosb + t * s.ldt, p.col, wide, fc);
  load_table<N>(s.sinb + t * s.ldt, p.col, wide, fn);
  const float f = PAIRS || p.rot == 1 ? -sign : sign;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (PAIRS) {
      c[i] = make_float2(fc[i], fc[i]);
      n[i] = mul2(make_float2(fn[i], fn[i]), make_float2(f, -f));
    } else {
      c[i] = make_float2(fc[2 * i], fc[2 * i + 1]);
      n[i] = mul2(make_float2(fn[2 * i], fn[2 * i + 1]), make_float2(f, f));
    }
  }
}
template <typename T>
__device__ __forceinline__ void lane_weight(const void* w, int c, int d, float shift, float2* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = make_float2(1.f, 1.f);
  if (w == nullptr || c >= d) return;
  Raw<T, 8> r;
  r.load(reinterpret_cast<const T*>(w) + c);
  get2(r, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = add2(f[i], make_float2(shift, shift));
}
// The partners of the lane's 8 channels (pairs x).
template <typename T, int G, bool PAIRS>
__device__ __forceinline__ void partners(const Raw<T, 8>& raw, const float2* x, int partner, float2* o) {
  if constexpr (PAIRS) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = make_float2(x[i].y, x[i].x);
  } else {
    Raw<T, 8> q;
#pragma unroll
    for (int i = 0; i < Raw<T, 8>::kWords; ++i) q.w[i] = __shfl_sync(0xffffffffu, raw.w[i], partner, G);
    get2(q, o);
  }
}

// A group takes every shares-th head of one token, HB at a time; the loads of the next HB are issued before these are used, the first before the
// tables' and weights'. Two at a time: four take 115 registers, and then two blocks an SM (43 us instead of 32). blockIdx.y: queries or keys.
template <typename T, int G, bool PAIRS, int HB>
__global__ void __launch_bounds__(256) qk_norm_rope_part_fwd_kernel(const __grid_constant__ NormArgs a, int q_shares, int k_shares) {
  const RopeShape& s = a.s;
  const NormOperand& o = blockIdx.y ? a.k : a.q;
  const unsigned shares = blockIdx.y ? k_shares : q_shares;
  constexpr int GPB = 256 / G;
  const int g = threadIdx.x % G;
  if (blockIdx.x * GPB >= (unsigned)s.T * shares) return;      // queries and keys need different numbers of blocks
  const unsigned item = blockIdx.x * GPB + threadIdx.x / G;
  const unsigned token = item / shares;
  const int share = (int)(item - token * shares);
  const bool live = token < (unsigned)s.T, on = live && g * 8 < s.d;
  const int64_t t = live ? token : s.T - 1;             // the whole warp stays in the shuffles
  const T* px = reinterpret_cast<const T*>(o.x) + t * o.x_tok + share * o.x_head + g * 8;
  T* py = reinterpret_cast<T*>(o.y) + t * o.y_tok + share * o.y_head + g * 8;
  const int64_t x_step = o.x_head * shares, y_step = o.y_head * shares;
  const int each = (o.H + (int)shares - 1) / (int)shares, mine = on ? (o.H - share + (int)shares - 1) / (int)shares : 0;    // heads: at most; this group's
  Raw<T, 8> raw[HB], ahead[HB];
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    raw[i].zero();
    if (i < mine) raw[i].load(px + i * x_step);
  }
  const bool wide = !((reinterpret_cast<uintptr_t>(s.cosb) | reinterpret_cast<uintptr_t>(s.sinb)) & 15) && (s.ldt & 3) == 0;
  const LanePlace p = lane_place<PAIRS>(s, g);
  float2 cw[4], nw[4];
  {
    float2 w[4], wp[4];
    lane_tables<PAIRS>(s, p, t, wide, 1.f, cw, nw);
    lane_weight<T>(o.w, g * 8, s.d, a.shift, w);
    if (PAIRS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) wp[j] = make_float2(w[j].y, w[j].x);
    } else {
      lane_weight<T>(o.w, p.partner * 8, s.d, a.shift, wp);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      cw[j] = mul2(cw[j], w[j]);
      nw[j] = mul2(nw[j], wp[j]);
    }
  }
  const float inv_d = 1.f / (float)s.d;
  for (int first = 0; first < each; first += HB) {
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      ahead[i].zero();
      if (first + HB + i < mine) ahead[i].load(px + (first + HB + i) * x_step);
    }
    float sq[HB];
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      float2 x[4], q = make_float2(0.f, 0.f);
      get2(raw[i], x);
#pragma unroll
      for (int j = 0; j < 4; ++j) q = fma2(x[j], x[j], q);
      sq[i] = q.x + q.y;
    }
#pragma unroll
    for (int m = G / 2; m > 0; m >>= 1)
#pragma unroll
      for (int i = 0; i < HB; ++i) sq[i] += __shfl_xor_sync(0xffffffffu, sq[i], m);
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      float2 x[4], q[4];
      get2(raw[i], x);
      partners<T, G, PAIRS>(raw[i], x, p.partner, q);
      const float r = rsqrtf(sq[i] * inv_d + a.eps);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = mul2(make_float2(r, r), fma2(x[j], cw[j], mul2(q[j], nw[j])));
      if (first + i < mine) store2(py + (first + i) * y_step, x);
      raw[i] = ahead[i];
    }
  }
}

// The same split for the gradient. A chunk is a part (`parts` of them) of a token's shares; the groups take chunks in turn, so that neighbouring groups
// read neighbouring memory at a time, and walk over a chunk's shares, HB heads each. The operands of the next heads are fetched before these sums
// are taken; a group holds its sums of the weight's gradient.
template <typename T, int G, bool PAIRS, int HB>
__global__ void __launch_bounds__(256, 2) qk_norm_rope_part_bwd_kernel(const __grid_constant__ NormArgs a, int shares, int parts) {
  const RopeShape& s = a.s;
  const NormOperand& o = a.q;
  constexpr int GPB = 256 / G;
  __shared__ float sums[GPB][G * 8 + 4];
  const unsigned groups = gridDim.x * GPB, chunks = (unsigned)s.T * parts;
  const int per = (shares + parts - 1) / parts;          // shares of a chunk
  const int g = threadIdx.x % G, grp = threadIdx.x / G;
  const bool in = g * 8 < s.d;
  const bool wide = !((reinterpret_cast<uintptr_t>(s.cosb) | reinterpret_cast<uintptr_t>(s.sinb)) & 15) && (s.ldt & 3) == 0;
  const LanePlace p = lane_place<PAIRS>(s, g);
  const float inv_d = 1.f / (float)s.d;
  float2 dw[4], w[4], c[4], n[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) dw[i] = make_float2(0.f, 0.f);
  lane_weight<T>(o.w, g * 8, s.d, a.shift, w);
  Raw<T, 8> rx[HB], rd[HB];
  // operands of the heads of `share` in token t
  auto fetch = [&](bool valid, int64_t tok, int sh, Raw<T, 8>* x, Raw<T, 8>* d) {
    const T* px = reinterpret_cast<const T*>(o.x) + tok * o.x_tok + sh * o.x_head + g * 8;
    const T* pd = reinterpret_cast<const T*>(o.dy) + tok * o.dy_tok + sh * o.dy_head + g * 8;
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      x[i].zero();
      d[i].zero();
      if (valid && sh + i * shares < o.H) {
        x[i].load(px + i * (shares * o.x_head));
        d[i].load(pd + i * (shares * o.dy_head));
      }
    }
  };
  unsigned chunk = blockIdx.x * GPB + grp;
  int64_t t = chunk / (unsigned)parts;
  int begin = (int)(chunk - (unsigned)t * parts) * per;
  fetch(in && chunk < chunks && begin < shares, t, begin, rx, rd);
  // every group of the block runs as many rounds: whole warps stay in the shuffles
  for (unsigned round = 0; round < chunks; round += groups) {
    const bool on = in && chunk < chunks;
    const int64_t tok = t;
    const int from = begin;
    chunk += groups;
    t = chunk / (unsigned)parts;
    begin = (int)(chunk - (unsigned)t * parts) * per;
    lane_tables<PAIRS>(s, p, on ? tok : 0, wide, -1.f, c, n);
    for (int step = 0; step < per; ++step) {
      const int share = from + step;
      const bool live = on && share < shares, last = step + 1 == per;
      Raw<T, 8> nx[HB], nd[HB];
      const int nshare = last ? begin : share + 1;
      fetch(in && nshare < shares && (last ? chunk < chunks : on), last ? t : tok, nshare, nx, nd);
      float2 d[HB][4];
      float sq[HB], dot[HB];
#pragma unroll
      for (int i = 0; i < HB; ++i) {
        float2 x[4], q[4], e[4], s2 = make_float2(0.f, 0.f), d2 = s2;
        get2(rd[i], e);
        partners<T, G, PAIRS>(rd[i], e, p.partner, q);
        get2(rx[i], x);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          d[i][j] = fma2(e[j], c[j], mul2(q[j], n[j]));
          s2 = fma2(x[j], x[j], s2);
          d2 = fma2(mul2(d[i][j], w[j]), x[j], d2);
        }
        sq[i] = s2.x + s2.y;
        dot[i] = d2.x + d2.y;
      }
#pragma unroll
      for (int m = G / 2; m > 0; m >>= 1)
#pragma unroll
        for (int i = 0; i < HB; ++i) {
          sq[i] += __shfl_xor_sync(0xffffffffu, sq[i], m);
          dot[i] += __shfl_xor_sync(0xffffffffu, dot[i], m);
        }
      T* py = reinterpret_cast<T*>(o.y) + tok * o.y_tok + share * o.y_head + g * 8;
#pragma unroll
      for (int i = 0; i < HB; ++i) {
        if (live && share + i * shares < o.H) {          // a dead head's r may be infinite (eps 0)
          const float r = rsqrtf(sq[i] * inv_d + a.eps), k = -(dot[i] * inv_d * r * r * r);
          float2 x[4], out[4];
          get2(rx[i], x);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 dr = mul2(d[i][j], make_float2(r, r));
            dw[j] = fma2(dr, x[j], dw[j]);
            out[j] = fma2(dr, w[j], mul2(x[j], make_float2(k, k)));
          }
          store2(py + i * (shares * o.y_head), out);
        }
        rx[i] = nx[i];
        rd[i] = nd[i];
      }
    }
  }
  if (a.partial == nullptr) return;
  if (in) {
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<float2*>(&sums[grp][g * 8 + 2 * j]) = dw[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < s.d; i += 256) {        // the groups of a block in their order
    float v = 0.f;
#pragma unroll 4
    for (int k = 0; k < GPB; ++k) v += sums[k][i];
    a.partial[(int64_t)blockIdx.x * s.d + i] = v;
  }
}

// The form for everything else up to d = 256: a lane still holds 8 channels (read and written VL at a time, as d and the addresses allow), and the
// partners come through shared memory: channel c lies at (c % 8) G + c / 8, so that neighbouring lanes read neighbouring words whatever P and off.
template <typename T, int VL>
__device__ __forceinline__ void load_lane(const T* p, int c, int d, float* f) {
#pragma unroll
  for (int i = 0; i < 8; i += VL) {
#pragma unroll
    for (int j = 0; j < VL; ++j) f[i + j] = 0.f;
    if (c + i < d) load_vec<T, VL>(p + i, f + i);
  }
}
template <typename T, int VL>
__device__ __forceinline__ void store_lane(T* p, int c, int d, const float* f) {
#pragma unroll
  for (int i = 0; i < 8; i += VL)
    if (c + i < d) store_vec<T, VL>(p + i, f + i);
}
// The partners of the lane's channels; `box`: 8 G words of the lane's group.
template <int G>
__device__ __forceinline__ void gather_lane(float* box, int g, const float* x, const int* at, float* q) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j) box[j * G + g] = x[j];
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = box[at[j]];
}
template <int G>
__device__ __forceinline__ void lane_channels(const RopeShape& s, int g, int64_t t, float sign, float* c, float* n, int* at) {
  channel_tables<8>(s, g * 8, t, sign, c, n, at);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int p = g * 8 + j + at[j];
    at[j] = (p & 7) * G + (p >> 3);
  }
}
template <typename T, int VL>
__device__ __forceinline__ void lane_weights(const void* w, int c, int d, float shift, float* f) {
  if (w == nullptr) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 1.f;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f[j] = 0.f;
    if (c + j < d) {
      load_vec<T, 1>(reinterpret_cast<const T*>(w) + c + j, f + j);
      f[j] += shift;
    }
  }
}
constexpr int kGatherHeads = 2;
template <typename T, int G, int VL>
__global__ void __launch_bounds__(256) qk_norm_rope_gather_fwd_kernel(const __grid_constant__ NormArgs a, int q_shares, int k_shares) {
  const RopeShape& s = a.s;
  const NormOperand& o = blockIdx.y ? a.k : a.q;
  const unsigned shares = blockIdx.y ? k_shares : q_shares;
  constexpr int GPB = 256 / G;
  __shared__ float boxes[GPB][8 * G];
  if (blockIdx.x * GPB >= (unsigned)s.T * shares) return;
  const int g = threadIdx.x % G, c0 = g * 8;
  const unsigned item = blockIdx.x * GPB + threadIdx.x / G, token = item / shares;
  const int share = (int)(item - token * shares);
  const bool live = token < (unsigned)s.T;
  const int64_t t = live ? token : s.T - 1;             // the whole warp stays in the shuffles
  float x[kGatherHeads][8];
#pragma unroll
  for (int i = 0; i < kGatherHeads; ++i) {
    const int h = share + i * (int)shares;
    load_lane<T, VL>(reinterpret_cast<const T*>(o.x) + t * o.x_tok + (int64_t)h * o.x_head + c0, live && h < o.H ? c0 : s.d, s.d, x[i]);
  }
  float c[8], n[8], w[8];
  int at[8];
  lane_channels<G>(s, g, t, 1.f, c, n, at);
  lane_weights<T, VL>(o.w, c0, s.d, a.shift, w);
#pragma unroll
  for (int i = 0; i < kGatherHeads; ++i) {
    float sq = 0.f, q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sq += x[i][j] * x[i][j];
#pragma unroll
    for (int m = G / 2; m > 0; m >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, m);
    const float r = rsqrtf(sq / (float)s.d + a.eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[i][j] *= r * w[j];
    gather_lane<G>(boxes[threadIdx.x / G], g, x[i], at, q);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[i][j] = at[j] == j * G + g ? x[i][j] : x[i][j] * c[j] + q[j] * n[j];      // its own partner: it passes
    const int h = share + i * (int)shares;
    store_lane<T, VL>(reinterpret_cast<T*>(o.y) + t * o.y_tok + (int64_t)h * o.y_head + c0, live && h < o.H ? c0 : s.d, s.d, x[i]);
  }
}

template <typename T, int G, int VL>
__global__ void __launch_bounds__(256, 2) qk_norm_rope_gather_bwd_kernel(const __grid_constant__ NormArgs a, int shares) {
  const RopeShape& s = a.s;
  const NormOperand& o = a.q;
  constexpr int GPB = 256 / G;
  __shared__ float boxes[GPB][8 * G];
  const int g = threadIdx.x % G, grp = threadIdx.x / G, c0 = g * 8;
  const unsigned items = (unsigned)s.T * shares, groups = gridDim.x * GPB;
  const unsigned each = items / groups, more = items % groups, me = blockIdx.x * GPB + grp;      // the first `more` groups have one item more
  unsigned item = me * each + (me < more ? me : more);
  const unsigned end = item + each + (me < more ? 1 : 0), rounds = each + (more ? 1 : 0);
  int64_t t = item / (unsigned)shares, tables_of = -1;
  int share = (int)(item - (unsigned)t * shares);
  float dw[8], w[8], c[8], n[8];
  int at[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    dw[j] = c[j] = n[j] = 0.f;
    at[j] = j * G + g;
  }
  lane_weights<T, VL>(o.w, c0, s.d, a.shift, w);
  for (unsigned round = 0; round < rounds; ++round, ++item) {
    const bool live = item < end;
    float x[kGatherHeads][8], d[kGatherHeads][8];
#pragma unroll
    for (int i = 0; i < kGatherHeads; ++i) {
      const int h = share + i * shares, from = live && h < o.H ? c0 : s.d;
      load_lane<T, VL>(reinterpret_cast<const T*>(o.x) + t * o.x_tok + (int64_t)h * o.x_head + c0, from, s.d, x[i]);
      load_lane<T, VL>(reinterpret_cast<const T*>(o.dy) + t * o.dy_tok + (int64_t)h * o.dy_head + c0, from, s.d, d[i]);
    }
    if (live && t != tables_of) {
      lane_channels<G>(s, g, t, -1.f, c, n, at);
      tables_of = t;
    }
#pragma unroll
    for (int i = 0; i < kGatherHeads; ++i) {
      const int h = share + i * shares;
      float q[8], sq = 0.f, dot = 0.f;
      gather_lane<G>(boxes[grp], g, d[i], at, q);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (at[j] != j * G + g) d[i][j] = d[i][j] * c[j] + q[j] * n[j];
        sq += x[i][j] * x[i][j];
        dot += d[i][j] * w[j] * x[i][j];
      }
#pragma unroll
      for (int m = G / 2; m > 0; m >>= 1) {
        sq += __shfl_xor_sync(0xffffffffu, sq, m);
        dot += __shfl_xor_sync(0xffffffffu, dot, m);
      }
      if (live && h < o.H) {                             // a dead head's r may be infinite (eps 0)
        const float r = rsqrtf(sq / (float)s.d + a.eps), k = dot / (float)s.d * r * r * r;
        float out[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float dr = d[i][j] * r;
          if (c0 + j < s.d) dw[j] += dr * x[i][j];
          out[j] = dr * w[j] - x[i][j] * k;
        }
        store_lane<T, VL>(reinterpret_cast<T*>(o.y) + t * o.y_tok + (int64_t)h * o.y_head + c0, c0, s.d, out);
      }
    }
    if (++share == shares) {
      share = 0;
      ++t;
    }
  }
  if (a.partial == nullptr) return;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) boxes[grp][c0 + j] = dw[j];
  __syncthreads();
  for (int i = threadIdx.x; i < s.d; i += 256) {        // the groups of a block in their order
    float v = 0.f;
#pragma unroll 4
    for (int k = 0; k < GPB; ++k) v += boxes[k][i];
    a.partial[(int64_t)blockIdx.x * s.d + i] = v;
  }
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
  float* buf = smem + wid * (BWD ? 2 * d : d);          // BWD: dy | sums of dw
  if (BWD)
    for (int c = lane; c < d; c += 32) buf[d + c] = 0.f;
  const int heads = a.q.H + a.k.H;
  const int64_t items = (int64_t)s.T * heads;
  for (int64_t item = (int64_t)blockIdx.x * kAnyWarps + wid; item < items; item += (int64_t)gridDim.x * kAnyWarps) {
    const int64_t t = item / heads;
    int h = (int)(item - t * heads);
    const bool key = h >= a.q.H;
    const NormOperand& o = key ? a.k : a.q;
    if (key) h -= a.q.H;
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
        buf[d + c] += g * x * r;
      }
      const float k = warp_sum(dot) / (float)d * r * r * r;
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
  for (int i = threadIdx.x; i < d; i += blockDim.x) {
    float v = 0.f;
    for (int w = 0; w < kAnyWarps; ++w) v += smem[w * 2 * d + d + i];
    a.partial[(int64_t)blockIdx.x * d + i] = v;
  }
}

// dw [d] in T from partial [P][d], in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) qk_weight_sum_kernel(const float* __restrict__ partial, T* __restrict__ dw, int P, int d) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < d) {
#pragma unroll 4
    for (int q = wid; q < P; q += 32) v += partial[(int64_t)q * d + c];
  }
  part[wid][lane] = v;
  __syncthreads();
  v = warp_sum(part[lane][wid]);
  const int oc = blockIdx.x * 32 + wid;
  if (lane == 0 && oc < d) store_vec<T, 1>(dw + oc, &v);
}

// Values per access that d and the addresses of a call allow (16 bytes at most).
static int norm_vec(const NormArgs& a, int size, bool bwd) {
  for (int v = 16 / size; v > 1; v /= 2) {
    const uintptr_t bytes = v * size;
    bool ok = a.s.d % v == 0;
    for (const NormOperand* o : {&a.q, &a.k}) {
      if (!o->H) continue;
      uintptr_t at = reinterpret_cast<uintptr_t>(o->x) | reinterpret_cast<uintptr_t>(o->y);
      ok = ok && div_by(v, {o->x_tok, o->x_head, o->y_tok, o->y_head});
      if (bwd) {
        at |= reinterpret_cast<uintptr_t>(o->dy);
        ok = ok && div_by(v, {o->dy_tok, o->dy_head});
      }
      ok = ok && at % bytes == 0;
    }
    if (ok) return v;
  }
  return 1;
}
// 2: the wide form, 1: the gather form, 0: the general one.
static int norm_form(const NormArgs& a, int size, bool bwd) {
  const RopeShape& s = a.s;
  if (s.d > 256) return 0;
  const bool aligned = !((reinterpret_cast<uintptr_t>(a.q.w) | reinterpret_cast<uintptr_t>(a.k.w)) & 15);
  return aligned && div_by(8, {s.d, s.off, s.interleaved ? 2 * s.P : s.P}) && norm_vec(a, size, bwd) == 16 / size ? 2 : 1;
}
// Heads per group (a power of two): loads in flight and tables read seldom, or one where there are too few tokens to fill the machine that way; more
// than four only where the machine is filled three times. Forward up to eight, read two at a time, backward two (registers).
static int norm_lanes(int d) { return d > 128 ? 32 : d > 64 ? 16 : 8; }
static int norm_heads(const NormArgs& a, int H, int most) {
  int n = 1;
  while (n < most && n < H) n *= 2;
  while (n > 1 && (int64_t)a.s.T * ((H + n - 1) / n) * norm_lanes(a.s.d) < (int64_t)sm_count() * 1024 * (n > 4 ? 3 : 1)) n /= 2;
  return n;
}
static int norm_bwd_grid(const NormArgs& a, int form) {
  const int n = norm_heads(a, a.q.H, 2), H = a.q.H;
  const int64_t items = (int64_t)a.s.T * (form == 2 ? (H + n - 1) / n : form == 1 ? (H + kGatherHeads - 1) / kGatherHeads : H);
  const int lanes = form == 2 ? norm_lanes(a.s.d) : a.s.d > 128 ? 32 : 16, per = form ? 256 / lanes : kAnyWarps;
  const int64_t need = (items + per - 1) / per, most = (int64_t)sm_count() * (form ? 2 : 4);
  return (int)(need < most ? need : most);
}

template <typename T>
static int norm_fwd(const NormArgs& a, cudaStream_t stream) {
  const int form = norm_form(a, sizeof(T), false);
  if (form) {
    const int G = form == 2 ? norm_lanes(a.s.d) : a.s.d > 128 ? 32 : 16, H = a.q.H > a.k.H ? a.q.H : a.k.H;
    const int n = form == 2 ? norm_heads(a, H, 8) : kGatherHeads, hb = n < 2 ? n : 2;
    const int qs = a.q.H ? (a.q.H + n - 1) / n : 1, ks = a.k.H ? (a.k.H + n - 1) / n : 1;
    const int64_t items = (int64_t)a.s.T * (qs > ks ? qs : ks);
    if (items > 0x7fffff00) return -10;
    // without queries the keys take their place
    NormArgs b = a;
    if (a.q.H == 0) { b.q = a.k; b.k.H = 0; }
    const dim3 grid((unsigned)((items + 256 / G - 1) / (256 / G)), b.k.H ? 2 : 1);
    const int s0 = a.q.H ? qs : ks, vl = norm_vec(a, sizeof(T), false);
    if (form == 2) {
#define LLMT_QK(L, I, N) \
  if (G == L && (bool)a.s.interleaved == I && hb == N) qk_norm_rope_part_fwd_kernel<T, L, I, N><<<grid, 256, 0, stream>>>(b, s0, ks);
#define LLMT_QK3(L, I) LLMT_QK(L, I, 1) LLMT_QK(L, I, 2)
      LLMT_QK3(32, true) LLMT_QK3(32, false) LLMT_QK3(16, true) LLMT_QK3(16, false) LLMT_QK3(8, true) LLMT_QK3(8, false)
#undef LLMT_QK3
#undef LLMT_QK
    } else {
#define LLMT_QK(L, N) if (G == L && vl == N) qk_norm_rope_gather_fwd_kernel<T, L, N><<<grid, 256, 0, stream>>>(b, s0, ks);
      if constexpr (sizeof(T) == 2) { LLMT_QK(32, 8) LLMT_QK(16, 8) }
      LLMT_QK(32, 4) LLMT_QK(16, 4) LLMT_QK(32, 2) LLMT_QK(16, 2) LLMT_QK(32, 1) LLMT_QK(16, 1)
#undef LLMT_QK
    }
  } else {
    const int64_t items = (int64_t)a.s.T * (a.q.H + a.k.H), need = (items + kAnyWarps - 1) / kAnyWarps;
    const int64_t most = (int64_t)sm_count() * 64;
    qk_norm_rope_any_kernel<T, false><<<(int)(need < most ? need : most), 32 * kAnyWarps, kAnyWarps * a.s.d * sizeof(float), stream>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
template <typename T>
static int norm_bwd(const NormArgs& a, int P, void* dw, cudaStream_t stream) {
  const int form = norm_form(a, sizeof(T), true), grid = norm_bwd_grid(a, form);
  if (a.partial != nullptr && grid > P) return -10;
  if (form) {
    const int G = form == 2 ? norm_lanes(a.s.d) : a.s.d > 128 ? 32 : 16;
    const int n = form == 2 ? norm_heads(a, a.q.H, 2) : kGatherHeads, shares = (a.q.H + n - 1) / n, vl = norm_vec(a, sizeof(T), true);
    if ((int64_t)a.s.T * shares > 0x7fffff00) return -10;
    if (form == 2) {
      // a token at a time, or parts of one while the groups have fewer than six chunks each (the last round would be a large part of the time)
      int parts = 1;
      while (2 * parts <= shares && (int64_t)a.s.T * parts < (int64_t)6 * grid * (256 / G)) parts *= 2;
#define LLMT_QK(L, I, N) \
  if (G == L && (bool)a.s.interleaved == I && n == N) qk_norm_rope_part_bwd_kernel<T, L, I, N><<<grid, 256, 0, stream>>>(a, shares, parts);
#define LLMT_QK2(L, I) LLMT_QK(L, I, 1) LLMT_QK(L, I, 2)
      LLMT_QK2(32, true) LLMT_QK2(32, false) LLMT_QK2(16, true) LLMT_QK2(16, false) LLMT_QK2(8, true) LLMT_QK2(8, false)
#undef LLMT_QK2
#undef LLMT_QK
    } else {
#define LLMT_QK(L, N) if (G == L && vl == N) qk_norm_rope_gather_bwd_kernel<T, L, N><<<grid, 256, 0, stream>>>(a, shares);
      if constexpr (sizeof(T) == 2) { LLMT_QK(32, 8) LLMT_QK(16, 8) }
      LLMT_QK(32, 4) LLMT_QK(16, 4) LLMT_QK(32, 2) LLMT_QK(16, 2) LLMT_QK(32, 1) LLMT_QK(16, 1)
#undef LLMT_QK
    }
  } else {
    qk_norm_rope_any_kernel<T, true><<<grid, 32 * kAnyWarps, kAnyWarps * 2 * a.s.d * sizeof(float), stream>>>(a);
  }
  if (cudaGetLastError() != cudaSuccess) return -3;
  if (a.partial != nullptr) qk_weight_sum_kernel<T><<<(a.s.d + 31) / 32, 1024, 0, stream>>>(a.partial, reinterpret_cast<T*>(dw), grid, a.s.d);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// ------------------------------------------------------------------------------------------ tables
// cos, sin [T][P] of factor-scaled angles position * inv_j. The product is taken in 64 bits in quarter turns, a = position inv_j 2 / pi, and split
// there into the nearest whole number q and the rest f in [-1/2, 1/2]: at position 131072 an fp32 angle is off by up to 2^-8 rad. Then
// cos and sin of x = f pi / 2, |x| <= pi / 4, are Taylor sums (the terms left out are below 2^-29) and q mod 4 says which of them, with which
// sign, is the angle's. Rounding by adding and taking away 1.5 2^52 leaves q in the low bits of the sum; double-to-integer and rounding
// instructions, which run at a quarter of the rate, bounded the first form of this kernel (sincospif of a rounded difference: 37 us for 131072 x 64
// against the 10 us that the writes take; now 16 us). Under ncu 60 % of the issue slots are used while the SMs are busy (three quarters of the time), the
// 64-bit pipe 10 %. Positions up to 2^50 (the quarter turns must stay below 2^51).
constexpr int kMaxFreqs = 256;
struct Freqs { double quarter[kMaxFreqs]; };           // inv_j * 2 / pi
__device__ __forceinline__ void angle_tables(double p, double quarter, float factor, float& c, float& n) {
  const double a = p * quarter, magic = 6755399441055744.0;                            // 1.5 * 2^52
  const double t = a + magic;
  const int q = __double2loint(t);
  const float x = (float)(a - (t - magic)) * 1.57079632679489662f, z = x * x;
  float si = 1.f / 362880.f, co = -1.f / 3628800.f;
  si = si * z - 1.f / 5040.f;
  si = si * z + 1.f / 120.f;
  si = si * z - 1.f / 6.f;
  si = si * z * x + x;
  co = co * z + 1.f / 40320.f;
  co = co * z - 1.f / 720.f;
  co = co * z + 1.f / 24.f;
  co = co * z - 0.5f;
  co = co * z + 1.f;
  c = (q & 1) ? si : co;
  n = (q & 1) ? co : si;
  c *= ((q + 1) & 2) ? -factor : factor;
  n *= (q & 2) ? -factor : factor;
}
// A thread keeps the frequencies of its V columns and walks over rows.
template <bool VEC>
__global__ void __launch_bounds__(256, 6) rope_tables_kernel(const int64_t* __restrict__ pos, const __grid_constant__ Freqs f, float factor,
                                                          float* __restrict__ cosb, float* __restrict__ sinb, int64_t T, int P) {
  constexpr int V = VEC ? 4 : 1;
  const int per_row = P / V, rows = 256 / per_row;      // at most 256 columns: a row fits a block
  const int sub = threadIdx.x / per_row, j = (threadIdx.x - sub * per_row) * V;
  if (sub >= rows) return;
  double quarter[V];
#pragma unroll
  for (int v = 0; v < V; ++v) quarter[v] = f.quarter[j + v];
  const int64_t step = (int64_t)gridDim.x * rows;
  int64_t t = (int64_t)blockIdx.x * rows + sub, next = t < T ? pos[t] : 0;
  for (; t < T; t += step) {
    const double p = (double)next;
    if (t + step < T) next = pos[t + step];              // a row ahead
    float c[V], n[V];
#pragma unroll
    for (int v = 0; v < V; ++v) angle_tables(p, quarter[v], factor, c[v], n[v]);
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
// Rows of `partial` ([rows][d]) that the backward of H heads writes for any alignment of its operands.
extern "C" int llmt_qk_norm_rope_part_partials(int T, int H, int d) {
  NormArgs a{};
  a.s.T = T; a.s.d = d; a.q.H = H;
  int most = 0;
  for (int form = 0; form < 3; ++form) {
    const int g = norm_bwd_grid(a, form);
    most = g > most ? g : most;
  }
  return most;
}
extern "C" int llmt_qk_norm_rope_part_bwd(const LlmtRopeShape* sh, const LlmtHeads* x, float eps, float shift, float* partial, int P, void* dw, int f32,
                                          cudaStream_t stream) {
  const NormArgs a = norm_args(sh, x, nullptr, eps, shift, partial);
  if (!rope_shape_ok(a.s) || a.s.d > 1024 || a.s.T == 0 || a.q.H == 0) return -10;
  return f32 ? norm_bwd<float>(a, P, dw, stream) : norm_bwd<__nv_bfloat16>(a, P, dw, stream);
}

extern "C" int llmt_rope_tables(const int64_t* pos, const double* inv, int P, double factor, float* cosb, float* sinb, int64_t T, cudaStream_t stream) {
  if (P <= 0 || P > kMaxFreqs || T < 0) return -10;
  if (T == 0) return 0;
  Freqs f{};
  for (int j = 0; j < P; ++j) f.quarter[j] = inv[j] * 2.0 / 3.14159265358979323846;
  const bool vec = P % 4 == 0 && !((reinterpret_cast<uintptr_t>(cosb) | reinterpret_cast<uintptr_t>(sinb)) & 15);
  const int rows = 256 / (vec ? P / 4 : P);
  const int64_t need = (T + rows - 1) / rows, most = (int64_t)sm_count() * 6;
  const int grid = (int)(need < most ? need : most);
  if (vec) rope_tables_kernel<true><<<grid, 256, 0, stream>>>(pos, f, (float)factor, cosb, sinb, T, P);
  else rope_tables_kernel<false><<<grid, 256, 0, stream>>>(pos, f, (float)factor, cosb, sinb, T, P);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
