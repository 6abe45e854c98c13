// Linear layers with an epilogue: y = act(x W^T + b) + r, and what their gradients need (reference call sites: the biased projections, two-layer
// MLPs and mergers of llmtuner/models/qwen/qwen3_5/multimodal.py:47-290 and llmtuner/models/kimi/kimi_k3/multimodal.py:146-914).
//   z = x W^T + b,  y = act(z) + r;   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_rows dz,  dr = dy.
//
// The products run on tcgen05 with the roles of gemm.cu: one warp issues TMA loads, one the products, sixteen drain the accumulator; persistent
// workers, each one CTA (128-row tiles) or a pair of CTAs (256-row tiles, cta_group::2). The epilogue of the forward adds the bias, applies the
// activation and adds the residual in fp32 and rounds once; for the backward it also writes z (rounded to bf16: act' of the rounded z is off by
// at most |act''| |z| 2^-9, of the order of the rounding of dz itself, which the products take as bf16). Against the same formulas in 32 bits the
// results of a layer with an activation are therefore off by 0.0024 of their norm instead of the 0.00165 of one rounding; without one only the order of
// additions differs. The bias gradient is summed in fp32 from dz before it is rounded.
//
// Bound by the tensor pipe and by the operands' way from L2. 16384 x 1152 -> 4608 with gelu_tanh: forward 119 us (1.46 PFLOP/s; 107 plain), dx 115,
// dW 114, dz 80 (453 MB at 5.7 TB/s), one at a time. Back to back the power cap holds the SMs at 1440 MHz instead of 1965: 154, 148, 144 and 96.
// Rows that TMA cannot read (widths that are no multiple of 8) are copied first: 9000 x 1001 -> 999 with gelu and residual 120 us for all of it, and a
// single row of 4097 -> 4095 37 us (23 as the library's product and expressions, which read the weight once).
#include <atomic>
#include "activations.cuh"
#include "common.cuh"
#include "kernels.h"
#include "vec_io.cuh"

namespace llmt {

int sm_count();
int make_tmap_bf16(CUtensorMap* out, const void* base, int rank, const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box);

constexpr int kLM = 128;                 // rows of a CTA's tile
constexpr int kLK = 64;                  // 64 bf16: one 128-byte swizzle row
constexpr int kLEpiWarps = 16;
constexpr int kLThreads = 64 + 32 * kLEpiWarps;
constexpr int kLMaxStages = 8;
constexpr int kLStageA = kLM * kLK * 2;
constexpr int kLSmem = 227 * 1024;
constexpr int kLPatch = 2048;            // of an epilogue warp: 32 rows of 64 bytes
constexpr int kLStage = kLPatch + 128;     // and 32 bias values
constexpr int kLSlack = 512;              // for the 1024-byte alignment of the stages; dynamic shared memory starts on 1024 bytes (checked)
constexpr int kLSmemFixed = kLEpiWarps * kLStage + kLSlack + 512 /*barriers*/;      // leaves four stages of 128 x 256 tiles to the byte
constexpr int kMaxWorkers = 160;
constexpr int kLMostSize = 0x7fffffff - 511;             // rows and features: the end of the last tile is still a 32-bit number

// What becomes of a product: stored as it is, or (`fwd`) with bias, activation and residual.
struct LinOut {
  int M, N;
  __nv_bfloat16* C;
  int64_t ldc;
  const void* bias;
  int bias_f32;
  const __nv_bfloat16* res;
  int64_t ldres;
  __nv_bfloat16* pre;
  int64_t ldpre;
  int vec;                               // every row of C and res starts on 16 bytes and N is a multiple of 8; those of pre always do, padded
};
// The tiles of a product and who computes them. A tile is kLM * CG rows by `bn` columns (a multiple of 32, at most 512): up to 256 columns by one
// MMA per 16 deep slice, and the accumulator is double buffered in TMEM, so that a tile is drained under the next one's products; the columns
// beyond 256 by a second MMA, and then there is one accumulator. The last column of tiles may be narrower (its products
// are issued with fewer columns and take that much less time). The k-blocks of a tile are cut into `splits` parts, each a unit of work. Units of
// whole tiles go to the workers in turn, part by part, so that the workers read the same k-blocks at a time; the units of narrow tiles follow,
// worker w taking narrow_begin[w] .. narrow_begin[w + 1].
struct LinPlan {
  int bn, num_m, full_n, splits, kb;
  int stages, stage_bytes, b2_offset, workers;      // b2_offset: of the second MMA's columns of B in a stage
  float* ws;                             // splits > 1: [splits][tiles][rows / 32][bn / 4][32][4] partial sums
  int narrow_begin[kMaxWorkers + 1];
};
struct LinArgs {
  LinOut out;
  LinPlan plan;
  int* status;
};

__device__ __forceinline__ uint32_t lin_idesc(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// One unit: tile row, first column, columns computed (a multiple of 32), index of the tile, k-blocks [kb0, kb1).
struct LinUnit { int m, n0, width, tile, part, kb0, kb1; };
// The units of worker `w` one after another; false when there are no more.
struct LinWalk {
  int next, narrow, narrow_end;
  __device__ __forceinline__ LinWalk(const LinPlan& p, int w) : next(w), narrow(p.narrow_begin[w]), narrow_end(p.narrow_begin[w + 1]) {}
  __device__ __forceinline__ bool step(const LinPlan& p, int N, int group, LinUnit& u) {
    const int whole = p.num_m * p.full_n;
    if (next < whole * p.splits) {
      u.part = next / whole;
      u.tile = next - u.part * whole;
      // super-rows of `group` tile rows are swept column by column, so concurrent tiles cover a near-square patch and share operands in L2
      const int per = group * p.full_n, g = u.tile / per, first = g * group;
      const int gm = p.num_m - first < group ? p.num_m - first : group;
      const int r = u.tile - g * per;
      u.m = first + r % gm;
      u.n0 = (r / gm) * p.bn;
      u.width = p.bn;
      next += p.workers;
    } else if (narrow < narrow_end) {
      u.part = narrow / p.num_m;
      u.m = narrow - u.part * p.num_m;
      u.tile = whole + u.m;
      u.n0 = p.full_n * p.bn;
      u.width = (N - u.n0 + 31) & ~31;
      ++narrow;
    } else {
      return false;
    }
    u.kb0 = (int)((int64_t)p.kb * u.part / p.splits);
    u.kb1 = (int)((int64_t)p.kb * (u.part + 1) / p.splits);
    return true;
  }
};

// A warp's patch is 32 rows x 32 columns. In its staging buffer rows are 64 bytes; their 16-byte chunks are XORed with the row so that neither a lane
// per row nor eight lanes over two rows meet a bank twice.
__device__ __forceinline__ uint32_t patch_at(int row, int chunk) { return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4); }
// The residual's patch into the staging buffer. Rows on 16 bytes: asynchronously (wait_patch), clamped instead of skipped where the patch leaves the
// matrix. Others: a lane per column.
__device__ __forceinline__ void load_patch(uint8_t* stg, const LinOut& o, int row0, int col, int end, int lane) {
  if (o.vec) {
    const int cc = lane & 3, c = col + cc * 8 < end ? col + cc * 8 : 0;
    const __nv_bfloat16* p = o.res + c;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int rr = it * 8 + (lane >> 2);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(stg + patch_at(rr, cc))), "l"(p + (int64_t)min(row0 + rr, o.M - 1) * o.ldres)
                   : "memory");
    }
    return;
  }
  if (col + lane >= end) return;
#pragma unroll 1
  for (int first = 0; first < 32; first += 16) {         // 16 rows in flight (32 cost spills: 41 us instead of 39 for 16384 x 1152 x 1152 on the other path)
    __nv_bfloat16 v[16];
#pragma unroll
    for (int rr = 0; rr < 16; ++rr) v[rr] = o.res[(int64_t)min(row0 + first + rr, o.M - 1) * o.ldres + col + lane];
#pragma unroll
    for (int rr = 0; rr < 16; ++rr) *reinterpret_cast<__nv_bfloat16*>(stg + patch_at(first + rr, lane >> 3) + (lane & 7) * 2) = v[rr];
  }
}
__device__ __forceinline__ void wait_patch() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// The staging buffer's patch to global memory, along its rows.
__device__ __forceinline__ void store_patch(const uint8_t* stg, __nv_bfloat16* p, int64_t ld, bool vec, int M, int row0, int col, int end, int lane) {
  if (vec) {
    const int cc = lane & 3;
    if (col + cc * 8 >= end) return;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int rr = it * 8 + (lane >> 2);
      const uint4 v = *reinterpret_cast<const uint4*>(stg + patch_at(rr, cc));
      if (row0 + rr < M) *reinterpret_cast<uint4*>(p + (int64_t)(row0 + rr) * ld + col + cc * 8) = v;
    }
    return;
  }
  if (col + lane >= end) return;
  p += (int64_t)row0 * ld + col + lane;
#pragma unroll 16
  for (int rr = 0; rr < 32; ++rr)
    if (row0 + rr < M) p[rr * ld] = *reinterpret_cast<const __nv_bfloat16*>(stg + patch_at(rr, lane >> 3) + (lane & 7) * 2);
}
// Row `lane` of a patch, rounded, into the staging buffer.
__device__ __forceinline__ void stage_row(uint8_t* stg, int lane, const float2* v) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(stg + patch_at(lane, j)) =
        make_uint4(pack_bf16x2(v[4 * j].x, v[4 * j].y), pack_bf16x2(v[4 * j + 1].x, v[4 * j + 1].y), pack_bf16x2(v[4 * j + 2].x, v[4 * j + 2].y),
                   pack_bf16x2(v[4 * j + 3].x, v[4 * j + 3].y));
}

// A warp's patch of sums (`acc`: the 32 columns of row row0 + lane, in pairs) becomes results: z = sum + bias, act(z) + residual in fp32, one
// rounding. Columns from `end` on belong to another tile or to none. The bf16 rows are turned around in the warp's staging buffer, so that global
// accesses run along rows; the residual comes the same way: asked for by early_patch before the sums are there, or here where z goes first.
template <int ACT, bool RES>
__device__ __forceinline__ void early_patch(const LinOut& o, uint8_t* stg, int lane, int row0, int col0, int end) {
  if (!RES || (ACT != kActNone && o.pre != nullptr)) return;
  __syncwarp();                                          // the patch before has been read
  load_patch(stg, o, row0, col0, end, lane);
}
template <bool FWD, int ACT, bool RES>
__device__ __forceinline__ void finish_patch(const LinOut& o, uint8_t* stg, int lane, int row0, int col0, int end, float2* acc) {
  if (FWD && o.bias != nullptr) {                        // a value per lane, to where every lane reads them all
    const int c = col0 + lane;
    float b = 0.f;
    if (c < end) {
      if (o.bias_f32) b = reinterpret_cast<const float*>(o.bias)[c];
      else b = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(o.bias)[c]);
    }
    float* bs = reinterpret_cast<float*>(stg + kLPatch);
    __syncwarp();
    bs[lane] = b;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 v = *reinterpret_cast<const float4*>(bs + 4 * j);
      acc[2 * j] = add2(acc[2 * j], make_float2(v.x, v.y));
      acc[2 * j + 1] = add2(acc[2 * j + 1], make_float2(v.z, v.w));
    }
  }
  if (FWD && ACT != kActNone && o.pre != nullptr) {
    __syncwarp();
    stage_row(stg, lane, acc);
    __syncwarp();
    store_patch(stg, o.pre, o.ldpre, true, o.M, row0, col0, end, lane);
    if (RES) {
      __syncwarp();
      load_patch(stg, o, row0, col0, end, lane);
    }
  }
  if (FWD) {
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] = activate<ACT>(acc[j]);
  }
  if (FWD && RES) {
    wait_patch();
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 v = *reinterpret_cast<const uint4*>(stg + patch_at(lane, j));
      float q[8];
      unpack_bf16x2(v.x, q); unpack_bf16x2(v.y, q + 2); unpack_bf16x2(v.z, q + 4); unpack_bf16x2(v.w, q + 6);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[4 * j + i] = add2(acc[4 * j + i], make_float2(q[2 * i], q[2 * i + 1]));
    }
  }
  __syncwarp();
  stage_row(stg, lane, acc);
  __syncwarp();
  store_patch(stg, o.C, o.ldc, o.vec, o.M, row0, col0, end, lane);
}

// Says that sums have been read: they are in registers (tcgen05.wait::ld has returned, the fence before it orders the reads), so the arrival has no
// memory to release, and a release would wait for every store that the thread has in flight (16384 x 1152 -> 4608 with gelu_tanh and z: 133 us, 125).
__device__ __forceinline__ void arrive_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// WIDE: tiles of more than 256 columns (CTA pairs only).
template <int CG, bool WIDE, bool A_MN, bool B_MN, bool SPLIT, bool FWD, int ACT, bool RES>
__global__ void __launch_bounds__(kLThreads, 1) linear_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                                                              const __grid_constant__ CUtensorMap tmB2, const __grid_constant__ LinArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (smem - smem_raw > kLSlack) {                       // the same in every block: none goes on
    if (threadIdx.x == 0) report_status(a.status, kStatusBadArgument, 900, (int)(smem - smem_raw));
    return;
  }
  const LinPlan& plan = a.plan;
  const int stages = plan.stages, stage_bytes = plan.stage_bytes;
  uint8_t* epi = smem + stages * stage_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(epi + kLEpiWarps * kLStage);
  uint64_t* empty = full + kLMaxStages;
  uint64_t* tfull = empty + kLMaxStages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // known to be the same in the whole warp
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
  const int worker = blockIdx.x / CG;
  constexpr int kGroup = 16 / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], CG * kLEpiWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    if constexpr (CG == 2) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
    else { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  }
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  LinWalk walk(plan, worker);
  LinUnit u;
  constexpr int accs = WIDE ? 1 : 2;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    // The whole warp walks the loop with uniform control flow and one lane issues: inside a branch of one lane every TMA instruction took about 75
    // clocks and every MMA about 115, and a k-block 440 to 800 clocks whatever the tile's width (its products of 256 columns occupy the tensor
    // pipe for 512).
    {
      const bool leader = elect_one();
      if (leader) {
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
      }
      int stage = 0;
      uint32_t phase = 0, armed = 0, armed_parity = 0;
      bool ok = true;
      // rows of B per load and MMA (a narrow tile loads as many and uses fewer)
      const int b_rows = (WIDE ? 256 : plan.bn) / CG, b2_rows = WIDE ? (plan.bn - 256) / CG : 0;
      // the transaction bytes of both CTAs' loads are counted by the leader's barrier
      const uint32_t full0 = CG == 2 ? cluster_map_u32(smem_u32(full), 0) : smem_u32(full);
      while (ok && walk.step(plan, a.out.N, kGroup, u)) {
        const int m0 = (u.m * CG + (int)rank) * kLM, w1 = WIDE ? min(u.width, 256) : u.width, nb = u.n0 + (int)rank * (w1 / CG),
                  nb2 = u.n0 + w1 + (int)rank * ((u.width - w1) / CG);
        for (int kb = u.kb0; kb < u.kb1; ++kb) {
          if (!mbar_wait_bounded(&empty[stage], phase ^ 1, abort_flag, a.status, 500 + stage)) {
            ok = false;
            break;
          }
          if (rank == 0) {
            armed |= 1u << stage;
            armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
          }
          if (leader) {
            uint8_t* sa = smem + stage * stage_bytes;
            uint8_t* sb = sa + kLStageA;
            if (rank == 0) mbar_arrive_expect_tx(&full[stage], CG * stage_bytes);
            const int k0 = kb * kLK;
            auto load = [&](void* dst, const CUtensorMap* m, int c0, int c1) {
              if constexpr (CG == 2) tma_load_2d_pair(dst, m, full0 + 8 * stage, c0, c1);
              else tma_load_2d(dst, m, &full[stage], c0, c1);
            };
            if constexpr (!A_MN) load(sa, &tmA, k0, m0);
            else {
#pragma unroll
              for (int j = 0; j < kLM / 64; ++j) load(sa + j * (kLK * 128), &tmA, m0 + 64 * j, k0);
            }
            if constexpr (!B_MN) {
              load(sb, &tmB, k0, nb);
              if (WIDE) load(sa + plan.b2_offset, &tmB2, k0, nb2);
            } else {
              for (int j = 0; j * 64 < b_rows; ++j) load(sb + j * (kLK * 128), &tmB, nb + 64 * j, k0);
              if (WIDE)
                for (int j = 0; j * 64 < b2_rows; ++j) load(sa + plan.b2_offset + j * (kLK * 128), &tmB, nb2 + 64 * j, k0);
            }
          }
          __syncwarp();
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
      }
      if (*abort_flag) {                                // copies in flight land before this CTA's shared memory is released
        for (int s = 0; s < stages; ++s) {
          if (!(armed & (1u << s))) continue;
          const uint32_t par = (armed_parity >> s) & 1u;
          for (uint32_t i = 0; i < (1u << 16); ++i)
            if (mbar_try_wait(&full[s], par)) break;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (rank == 0) {
      const bool leader = elect_one();
      // lower words of the operand descriptors at stage 0; a stage further on is lstep (16-byte units), the second MMA's columns b2step
      const uint32_t la0 = desc_lo(smem_u32(smem), A_MN ? kLK * 128 : 16), lb0 = desc_lo(smem_u32(smem) + kLStageA, B_MN ? kLK * 128 : 16);
      const uint32_t lstep = stage_bytes >> 4, b2step = (plan.b2_offset - kLStageA) >> 4;
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      while (ok && walk.step(plan, a.out.N, kGroup, u)) {
        const uint32_t idesc = lin_idesc(kLM * CG, WIDE ? min(u.width, 256) : u.width, A_MN, B_MN);
        const uint32_t idesc2 = WIDE ? lin_idesc(kLM * CG, u.width - 256, A_MN, B_MN) : 0u;
        const bool second = WIDE && u.width > 256;
        if (!mbar_wait_bounded<CG == 2>(&tempty[acc], acc_phase ^ 1, abort_flag, a.status, 600 + acc)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * 256;
        for (int kb = u.kb0; kb < u.kb1; ++kb) {
          if (!mbar_wait_bounded(&full[stage], phase, abort_flag, a.status, 700 + stage)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (leader) {
            const uint32_t la = la0 + stage * lstep, lb = lb0 + stage * lstep, acc0 = kb > u.kb0 ? 1u : 0u;
            auto slices = [&](uint32_t d, uint32_t b, uint32_t id) {
#pragma unroll
              for (int k = 0; k < kLK / 16; ++k) {
                const uint64_t da = desc_pack(la + (A_MN ? k * 128 : k * 2)), db = desc_pack(b + (B_MN ? k * 128 : k * 2));
                if constexpr (CG == 2) umma_bf16_ss_pair(d, da, db, id, k ? 1u : acc0);
                else umma_bf16_ss(d, da, db, id, k ? 1u : acc0);
              }
            };
            slices(d_tmem, lb, idesc);
            if (WIDE && second) slices(d_tmem + 256, lb + b2step, idesc2);
            if constexpr (CG == 2) umma_commit_pair(&empty[stage]);
            else umma_commit(&empty[stage]);
          }
          __syncwarp();
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        if (leader) {
          if constexpr (CG == 2) umma_commit_pair(&tfull[acc]);
          else umma_commit(&tfull[acc]);
        }
        __syncwarp();
        if (++acc == accs) { acc = 0; acc_phase ^= 1; }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue
    // Four warps share a quarter of the rows (the TMEM lanes a warp may read) and take patches of 32 columns in turn. A warp waits most of the time,
    // for TMEM, shared memory and the exponential unit, about 10 clocks per instruction: with 8 warps of 64 columns the drain of a tile outlasted its
    // products where an activation was applied (16384 x 1152 -> 4608, gelu_tanh and z: 168 us against 112 plain).
    const int quarter = warp & 3, side = (warp - 2) >> 2;
    uint8_t* stg = epi + (warp - 2) * kLStage;
    int acc = 0;
    uint32_t acc_phase = 0;
    while (walk.step(plan, a.out.N, kGroup, u)) {
      const int row0 = (u.m * CG + (int)rank) * kLM + quarter * 32;
      const int cols = min(u.width, a.out.N - u.n0);
      if (RES) {                                        // the residual's rows come into L2 while the product is computed
        const uint8_t* line = reinterpret_cast<const uint8_t*>(a.out.res + (int64_t)min(row0 + lane, a.out.M - 1) * a.out.ldres + u.n0);
        for (int o = side * 128; o < cols * 2; o += 512) asm volatile("prefetch.global.L2 [%0];" ::"l"(line + o));
      }
      if (!mbar_wait_bounded(&tfull[acc], acc_phase, abort_flag, a.status, 800 + acc)) break;
      tc_fence_after();
      // the warp's last sums are in registers: the accumulator may be overwritten as far as it goes
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2) arrive_relaxed(cluster_map_u32(smem_u32(&tempty[acc]), 0));
          else mbar_arrive(&tempty[acc]);
        }
      };
      const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * 256;
      if (side * 32 >= cols) release();
#pragma unroll 1
      for (int c = side * 32; c < cols; c += 128) {
        __align__(8) uint32_t r[32];
        tmem_ld_32x32(t_row + c, r);
        early_patch<ACT, RES>(a.out, stg, lane, row0, u.n0 + c, u.n0 + cols);
        tmem_wait_ld();
        if (c + 128 >= cols) release();
        if constexpr (SPLIT) {
          const int64_t tiles = (int64_t)plan.num_m * plan.full_n + (a.out.N % plan.bn ? plan.num_m : 0);
          float4* w = reinterpret_cast<float4*>(plan.ws) + (((u.part * tiles + u.tile) * (CG * 4) + rank * 4 + quarter) * (plan.bn / 4) + c / 4) * 32 + lane;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            w[j * 32] = make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]), __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3]));
        } else {
          finish_patch<FWD, ACT, RES>(a.out, stg, lane, row0, u.n0 + c, u.n0 + cols, reinterpret_cast<float2*>(r));
        }
      }
      if (++acc == accs) { acc = 0; acc_phase ^= 1; }
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

// The parts of every tile added in their order, and the epilogue: a warp per patch.
constexpr int kJoinWarps = 4;
template <bool FWD, int ACT, bool RES>
__global__ void __launch_bounds__(32 * kJoinWarps) linear_join_kernel(const __grid_constant__ LinArgs a, int cg, int patches) {
  __shared__ __align__(16) uint8_t stage[kJoinWarps][kLStage];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int id = blockIdx.x * kJoinWarps + wid;
  if (id >= patches) return;
  const LinPlan& p = a.plan;
  const int blocks = cg * 4, per_tile_row = (a.out.N + 31) / 32;
  const int mb = id / per_tile_row, col0 = (id - mb * per_tile_row) * 32;      // 32-row block, first column
  const int row0 = mb * 32, m = mb / blocks, block = mb - m * blocks;
  const int n = col0 / p.bn, c = col0 - n * p.bn, whole = p.num_m * p.full_n;
  int tile;
  if (n >= p.full_n) tile = whole + m;
  else {
    const int group = 16 / cg, g = m / group, first = g * group, gm = p.num_m - first < group ? p.num_m - first : group;
    tile = g * group * p.full_n + n * gm + (m - first);
  }
  const int64_t tiles = (int64_t)whole + (a.out.N % p.bn ? p.num_m : 0), part = tiles * blocks * (p.bn / 4) * 32;
  const float4* w = reinterpret_cast<const float4*>(p.ws) + (((int64_t)tile * blocks + block) * (p.bn / 4) + c / 4) * 32 + lane;
  early_patch<ACT, RES>(a.out, stage[wid], lane, row0, col0, a.out.N);
  float2 acc[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = make_float2(0.f, 0.f);
#pragma unroll 2
  for (int s = 0; s < p.splits; ++s) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 v = w[s * part + j * 32];
      acc[2 * j] = add2(acc[2 * j], make_float2(v.x, v.y));
      acc[2 * j + 1] = add2(acc[2 * j + 1], make_float2(v.z, v.w));
    }
  }
  finish_patch<FWD, ACT, RES>(a.out, stage[wid], lane, row0, col0, a.out.N, acc);
}

// ------------------------------------------------------------------------------------------ rows of any start
// Eight elements from p, of which `n` belong to the row: read as the five aligned words that hold them (a word is read only if it has an element of the
// row, so it lies in the same page) and shifted by two bytes where the row starts on an odd element. Elements from `n` on are foreign.
struct Shifted {
  uint32_t w[5];
  bool odd;
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = 0u;
    odd = false;
  }
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int n) {
    odd = reinterpret_cast<uintptr_t>(p) & 2;
    const uint32_t* q = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(3));
    const int have = min(n, 8) + odd;
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = 2 * i < have ? q[i] : 0u;
  }
  __device__ __forceinline__ void get(Raw<__nv_bfloat16, 8>& r) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = odd ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
  }
};
// Rows of any pitch and start into rows on 16 bytes, for TMA, which does not read the columns from N on. 9000 x 1001: 8 us (the library's strided
// copy took 24).
constexpr int kPadRows = 4;                              // rows in flight per thread
__global__ void __launch_bounds__(256) linear_pad_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, __nv_bfloat16* __restrict__ y, int64_t ldy,
                                                         int M, int N) {
  const int col = (blockIdx.x * 32 + (threadIdx.x & 31)) * 8;
  if (col >= N) return;
  const int64_t step = (int64_t)gridDim.y * 8;
  for (int64_t row = (int64_t)blockIdx.y * 8 + (threadIdx.x >> 5); row < M; row += kPadRows * step) {
    Shifted v[kPadRows];
#pragma unroll
    for (int u = 0; u < kPadRows; ++u) {
      v[u].zero();
      if (row + u * step < M) v[u].load(x + (row + u * step) * ldx + col, N - col);
    }
#pragma unroll
    for (int u = 0; u < kPadRows; ++u) {
      if (row + u * step >= M) break;
      Raw<__nv_bfloat16, 8> r;
      v[u].get(r);
      r.store(y + (row + u * step) * ldy + col);
    }
  }
}

// ------------------------------------------------------------------------------------------ dz and db
// A block owns a strip of LANES * 8 columns and every blocks-th group of rows, and sums its columns in a fixed order. Few rows (CLUSTER): the eight
// blocks of a strip are a cluster and add their sums through distributed shared memory in rank order, so db needs no second launch. Many rows:
// sums per block go to partial [blocks][N] and linear_db_kernel adds them; clusters of eight would leave SMs idle then (a GPC's 16 or 18 SMs hold
// two of them: half of the machine's time at 16384 x 4608).
constexpr int kStripBlocks = 8;
// z and dz have rows on 16 bytes (the caller's buffers); dy may lie anywhere (VEC false, see Shifted).
template <bool VEC, int LANES, bool CLUSTER, int ACT>
__global__ void __launch_bounds__(256, ACT == kActNone ? 4 : 3) linear_dz_kernel(const __nv_bfloat16* __restrict__ dy, int64_t ldy,
                                                                                const __nv_bfloat16* __restrict__ z, int64_t ldz,
                                                                                __nv_bfloat16* __restrict__ dz, int64_t lddz, void* __restrict__ db,
                                                                                int db_f32, float* __restrict__ partial, int M, int N) {
  constexpr int V = 8, COLS = LANES * V, ROWS = 256 / LANES;
  __shared__ float part[ROWS][COLS + 4];
  __shared__ float total[CLUSTER ? COLS : 1];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  const int col = blockIdx.x * COLS + lane * V;
  constexpr int W = V / 2;
  float2 acc[W];
#pragma unroll
  for (int j = 0; j < W; ++j) acc[j] = make_float2(0.f, 0.f);
  if (col < N) {
    constexpr int U = 4;                                 // rows in flight per thread
    const int64_t step = (int64_t)ROWS * gridDim.y;
    for (int64_t row = (int64_t)blockIdx.y * ROWS + sub; row < M; row += U * step) {
      Raw<__nv_bfloat16, V> rg[U], rz[U];
      Shifted sg[VEC ? 1 : U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        rz[u].zero();
        if constexpr (VEC) rg[u].zero();
        else sg[u].zero();
        if (row + u * step < M) {
          if constexpr (VEC) rg[u].load(dy + (row + u * step) * ldy + col);
          else sg[u].load(dy + (row + u * step) * ldy + col, N - col);
          if (ACT != kActNone) rz[u].load(z + (row + u * step) * ldz + col);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float g[V], p[V], out[V];
        if constexpr (!VEC) sg[u].get(rg[u]);
        rg[u].get(g);
        if (ACT != kActNone) rz[u].get(p);
#pragma unroll
        for (int j = 0; j < W; ++j) {
          float2 v = make_float2(g[2 * j], g[2 * j + 1]);
          if (ACT != kActNone) v = activate_grad<ACT>(make_float2(p[2 * j], p[2 * j + 1]), v);
          if (!VEC && col + 2 * j >= N) v.x = 0.f;       // behind the last column lie the next row's dy and a z that was never written
          if (!VEC && col + 2 * j + 1 >= N) v.y = 0.f;
          acc[j] = add2(acc[j], v);                      // rows past the end were loaded as zeros: their gradient is zero
          out[2 * j] = v.x;
          out[2 * j + 1] = v.y;
        }
        if (dz != nullptr && row + u * step < M) store_vec<__nv_bfloat16, V>(dz + (row + u * step) * lddz + col, out);
      }
    }
  }
  if (db == nullptr) return;
#pragma unroll
  for (int j = 0; j < W; ++j) {
    part[sub][lane * V + 2 * j] = acc[j].x;
    part[sub][lane * V + 2 * j + 1] = acc[j].y;
  }
  __syncthreads();
  const int oc = blockIdx.x * COLS + threadIdx.x;
  if (threadIdx.x < COLS) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) s += part[i][threadIdx.x];
    if constexpr (CLUSTER) total[threadIdx.x] = s;
    else if (oc < N) partial[(int64_t)blockIdx.y * N + oc] = s;
  }
  if constexpr (CLUSTER) {
    cluster_sync();
    if (blockIdx.y == 0 && threadIdx.x < COLS && oc < N) {
      float v[kStripBlocks], s = 0.f;
#pragma unroll
      for (int k = 0; k < kStripBlocks; ++k)
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[k]) : "r"(cluster_map_u32(smem_u32(&total[threadIdx.x]), k)));
#pragma unroll
      for (int k = 0; k < kStripBlocks; ++k) s += v[k];
      if (db_f32) reinterpret_cast<float*>(db)[oc] = s;
      else reinterpret_cast<__nv_bfloat16*>(db)[oc] = __float2bfloat16_rn(s);
    }
    cluster_sync();                                     // no block leaves while its sums are being read
  }
}

// db from partial [P][N]: 32 columns per block, its 32 warps take every 32nd row, fixed order.
__global__ void __launch_bounds__(1024) linear_db_kernel(const float* __restrict__ partial, void* __restrict__ db, int db_f32, int P, int N) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < N) {
#pragma unroll 4
    for (int q = wid; q < P; q += 32) s += partial[(int64_t)q * N + c];
  }
  part[wid][lane] = s;
  __syncthreads();
  s = warp_sum(part[lane][wid]);
  const int oc = blockIdx.x * 32 + wid;
  if (lane != 0 || oc >= N) return;
  if (db_f32) reinterpret_cast<float*>(db)[oc] = s;
  else reinterpret_cast<__nv_bfloat16*>(db)[oc] = __float2bfloat16_rn(s);
}

// ------------------------------------------------------------------------------------------ host
// Function attributes belong to a device: remembered per device. Threads may launch at once (a backward runs beside a forward).
using DeviceSet = std::atomic<uint64_t>;
template <typename F>
static bool allow_smem(F kern, int bytes, DeviceSet& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return true;
}

template <typename K>
static int lin_run(K kern, DeviceSet& done, int cg, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb2, const LinArgs& a, cudaStream_t stream) {
  if (!allow_smem(kern, kLSmem, done)) return -2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.plan.workers * cg);
  cfg.blockDim = dim3(kLThreads);
  cfg.dynamicSmemBytes = a.plan.stages * a.plan.stage_bytes + kLSmemFixed;
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cg; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = cg == 2 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, ta, tb, tb2, a) == cudaSuccess ? 0 : -3;
}
template <bool A_MN, bool B_MN, bool SPLIT, bool FWD, int ACT, bool RES>
static int lin_launch(int cg, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb2, const LinArgs& a, cudaStream_t stream) {
  static DeviceSet single{0}, pair{0}, wide{0};
  if (cg == 1) return lin_run(linear_kernel<1, false, A_MN, B_MN, SPLIT, FWD, ACT, RES>, single, 1, ta, tb, tb2, a, stream);
  if (a.plan.bn <= 256) return lin_run(linear_kernel<2, false, A_MN, B_MN, SPLIT, FWD, ACT, RES>, pair, 2, ta, tb, tb2, a, stream);
  return lin_run(linear_kernel<2, true, A_MN, B_MN, SPLIT, FWD, ACT, RES>, wide, 2, ta, tb, tb2, a, stream);
}
template <bool FWD, int ACT, bool RES>
static int lin_join(int cg, const LinArgs& a, cudaStream_t stream) {
  const int patches = a.plan.num_m * cg * 4 * ((a.out.N + 31) / 32);
  linear_join_kernel<FWD, ACT, RES><<<(patches + kJoinWarps - 1) / kJoinWarps, 32 * kJoinWarps, 0, stream>>>(a, cg, patches);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

struct LinCut { int cg, bn, splits; };
static int64_t lin_ws_floats(int M, int N, const LinCut& c) {
  if (c.splits < 2) return 0;
  const int64_t num_m = (M + kLM * c.cg - 1) / (kLM * c.cg), num_n = (N + c.bn - 1) / c.bn;
  return c.splits * num_m * num_n * kLM * c.cg * c.bn;
}

// Time of one k-block of a tile, in ns. Alone the products bound it (256 columns 302, 192 230, 128 and fewer about 200 with the loop around them);
// with every SM at it the operands, which come from L2 at 10 to 13 TB/s: 256 columns 420, 192 360, 128 260 (16384 x 4608 x 1152). `loaded`: columns
// that the TMA boxes fetch, more than `bn` where B is stored [K][N] and half a tile is no multiple of 64. `skewed`: rows of 128 bytes that a CTA
// fetches from matrices whose rows do not start on 128 bytes, each from two lines: 1.75 ns (products of 1000 x 1000 over 3000 and 6000 rows: 485
// ns a k-block for 128 columns, 660 for 256, against 230 where the rows have 1024 elements).
static double lin_kb_ns(int bn, int loaded, int skewed, double busy) {
  const double alone = bn * 1.18 > 200 ? bn * 1.18 : 200, crowded = 120 + 0.6 * (bn + loaded), lines = 1.75 * skewed;
  const double t = crowded > alone ? alone + (crowded - alone) * busy : alone;
  return t > lines ? t : lines;
}
// Units of whole tiles go round the workers; those of narrow tiles go one by one to the worker that is free first.
static void lin_plan(LinPlan& p, int N, int num_tiles_m, int most) {
  p.full_n = N / p.bn;
  p.num_m = num_tiles_m;
  const int rest = N - p.full_n * p.bn, whole = p.num_m * p.full_n * p.splits, narrow = rest ? p.num_m * p.splits : 0;
  p.workers = whole + narrow < most ? whole + narrow : most;
  const int ahead = whole % p.workers;                   // workers [0, ahead) have one whole unit more
  const int behind = ahead ? p.workers - ahead : 0;
  const int fit = rest ? (int)(lin_kb_ns(p.bn, p.bn, 0, 0) / lin_kb_ns((rest + 31) / 32 * 32, 0, 0, 0) + 0.1) : 0;       // narrow units in the time of a whole one
  const int catch_up = narrow < behind * fit ? narrow : behind * fit, left = narrow - catch_up;
  int at = 0;
  for (int w = 0; w < p.workers; ++w) {
    p.narrow_begin[w] = at;
    if (w >= ahead && behind) at += catch_up / behind + (w - ahead < catch_up % behind ? 1 : 0);
    at += left / p.workers + (w < left % p.workers ? 1 : 0);
  }
  p.narrow_begin[p.workers] = at;
}
// A product as the estimate sees it: B stored [K][N], matrices whose rows are no multiple of 128 bytes, what the epilogue takes (lin_drain).
struct LinKind { int b_mn, skew_a, skew_b, drain; };
// Time in which 128 columns of a tile are drained, in tenths of a us: 9 for the sums (every SM writes at the same time), 3 for a residual, 8 for z,
// which is a second result, and what the activation takes beyond its wait for memory.
static int lin_drain(int act, bool res, bool pre) {
  const int cost[kActKinds] = {0, 4, 1, 1, 0};           // in the order of ActKind
  return 9 + cost[act] + (res ? 3 : 0) + (act != kActNone && pre ? 8 : 0);
}
// The longest worker's units, in us (kb deep, `splits` parts).
static double lin_makespan(int cg, int bn, int splits, int num_m, int N, int kb, const LinKind& kind, int tenths) {
  const int most = sm_count() / cg, full_n = N / bn, rest = N - full_n * bn, whole = num_m * full_n * splits, narrow = rest ? num_m * splits : 0;
  const int workers = whole + narrow < most ? whole + narrow : most;
  const double depth = (double)((kb + splits - 1) / splits);
  // a tile is not done before its sums are drained: see lin_drain, hidden under the next tile's products where there are two
  // accumulators; 0.5 us pass between two tiles
  auto unit = [&](int w, int running) {
    const int loaded = kind.b_mn ? (w + 64 * cg - 1) / (64 * cg) * 64 * cg : w, skewed = (kind.skew_a ? kLM : 0) + (kind.skew_b ? loaded / cg : 0);
    const double drain = 0.1 * tenths * w / 128, mma = 0.5 + depth * lin_kb_ns(w, loaded, skewed, (double)running * cg / sm_count()) * 1e-3;
    return bn > 256 ? 1.1 * mma + drain : mma > drain ? mma : drain;        // 1.1: 4096 x 2048 x 2048 takes 32.9 us on 512 columns, 30.4 on 256
  };
  const int rounds = whole / workers, ahead = whole % workers, behind = ahead ? workers - ahead : 0;
  double t = rounds * unit(bn, workers) + (ahead ? unit(bn, ahead + (narrow < behind ? narrow : behind)) : 0);
  if (narrow) {
    const double tn = unit((rest + 31) / 32 * 32, workers);
    const int fit = full_n ? (int)(unit(bn, workers) / tn + 0.1) : 0, left = narrow - (narrow < behind * fit ? narrow : behind * fit);
    t += tn * ((left + workers - 1) / workers);
  }
  return t + (bn > 256 ? 0 : 0.1 * tenths * (full_n ? bn : rest) / 128);
}

// How a product is cut: CTAs per tile, tile width and parts along K. The shortest of the candidates by the estimate: tile widths that divide N
// evenly into 1, 2, ... columns of tiles, one CTA or a pair, and parts along K where the tiles leave workers idle. The parts cost a second
// launch and their sums in memory: 5.5 us and 4 bytes per sum and part at 4 TB/s (1152 x 1152 in 3 parts: 8.0 us).
static LinCut lin_find_cut(int M, int N, int K, const LinKind& kind) {
  const int kb = (K + kLK - 1) / kLK;
  LinCut best{1, 128, 1};
  double least = 1e30;
  for (int cg = 1; cg <= (M > kLM ? 2 : 1); ++cg) {
    const int num_m = (M + kLM * cg - 1) / (kLM * cg), most = sm_count() / cg;
    const int widest = cg == 2 ? 512 : 256;              // at least four stages of operands fit shared memory
    int last = 0;
    for (int n = (N + widest - 1) / widest; n <= (N + 127) / 128; ++n) {
      const int bn = ((N + n - 1) / n + 31) / 32 * 32;
      if (bn == last) continue;
      last = bn;
      const int tiles = num_m * ((N + bn - 1) / bn);
      for (int splits = 1; splits == 1 || (splits <= 8 && splits * 2 <= kb); ++splits) {
        if (splits > 1 && tiles * (splits - 1) >= 2 * most) break;
        double t = (cg == 2 ? 1.2 : 0.0) + lin_makespan(cg, bn, splits, num_m, N, kb, kind, splits > 1 ? lin_drain(0, false, false) : kind.drain);
        if (cg == 1) t *= 1.08;                          // a single CTA reads 1.5 times the operands per product
        if (splits > 1) t += 5.5 + 4e-6 * splits * (double)M * N / 4.0;
        if (t < least) {
          least = t;
          best = {cg, bn, splits};
        }
      }
    }
  }
  return best;
}
// The cut of a size is found once per thread and place in a small table (the search takes the host 0.4 to 4 us, beside 20 us for a small call).
static LinCut lin_cut(int M, int N, int K, const LinKind& kind) {
  struct Found { int M, N, K, kind; LinCut cut; };
  static thread_local Found table[64];
  const int bits = kind.drain * 8 + kind.b_mn * 4 + kind.skew_a * 2 + kind.skew_b;
  Found& f = table[((unsigned)M * 2654435761u ^ (unsigned)N * 40503u ^ (unsigned)K * 9176u ^ (unsigned)bits * 97u) >> 7 & 63];
  if (f.M != M || f.N != N || f.K != K || f.kind != bits) f = Found{M, N, K, bits, lin_find_cut(M, N, K, kind)};
  return f.cut;
}
static LinKind lin_kind(bool b_mn, int64_t lda, int64_t ldb, int act, bool res, bool pre) {
  return LinKind{b_mn ? 1 : 0, lda % 64 != 0, ldb % 64 != 0, lin_drain(act, res, pre)};
}

// out [M, N] = op(A) op(B), K deep: A stored [M][K] or (a_mn) [K][M], B stored [N][K] or (b_mn) [K][N]. ws: lin_ws_floats of the same sizes.
static int lin_gemm(const void* A, const void* B, LinArgs a, int K, int64_t lda, int64_t ldb, bool a_mn, bool b_mn, bool fwd, int act, float* ws,
                    int64_t ws_floats, cudaStream_t stream) {
  LinOut& o = a.out;
  if (o.M <= 0 || o.N <= 0) return 0;
  if (K <= 0 || o.M > kLMostSize || o.N > kLMostSize || K > kLMostSize || (lda & 7) || (ldb & 7) || (reinterpret_cast<uintptr_t>(A) & 15) || (reinterpret_cast<uintptr_t>(B) & 15)) return -10;
  const LinCut cut = lin_cut(o.M, o.N, K, lin_kind(b_mn, lda, ldb, fwd ? act : 0, o.res != nullptr, o.pre != nullptr));
  if (lin_ws_floats(o.M, o.N, cut) > (ws == nullptr ? 0 : ws_floats) || sm_count() / cut.cg > kMaxWorkers) return -10;
  LinPlan& p = a.plan;
  p.bn = cut.bn;
  p.splits = cut.splits;
  p.ws = ws;
  p.kb = (K + kLK - 1) / kLK;
  if (p.splits > p.kb) return -10;
  lin_plan(p, o.N, (o.M + kLM * cut.cg - 1) / (kLM * cut.cg), sm_count() / cut.cg);
  const int first = p.bn < 256 ? p.bn : 256, b_rows = first / cut.cg, b2_rows = (p.bn - first) / cut.cg;
  auto rows = [&](int r) { return (b_mn ? (r + 63) / 64 * 64 : r) * kLK * 2; };        // column blocks of 64 where B is stored [K][N]
  p.b2_offset = kLStageA + rows(b_rows);
  p.stage_bytes = p.b2_offset + rows(b2_rows);
  p.stages = (kLSmem - kLSmemFixed) / p.stage_bytes;
  if (p.stages > kLMaxStages) p.stages = kLMaxStages;
  CUtensorMap ta, tb, tb2;
  uint64_t dims[2], str[1] = {(uint64_t)lda * 2};
  uint32_t box[2];
  if (!a_mn) { dims[0] = K; dims[1] = o.M; box[0] = kLK; box[1] = kLM; }
  else       { dims[0] = o.M; dims[1] = K; box[0] = 64; box[1] = kLK; }
  if (make_tmap_bf16(&ta, A, 2, dims, str, box)) return -11;
  str[0] = (uint64_t)ldb * 2;
  if (!b_mn) { dims[0] = K; dims[1] = o.N; box[0] = kLK; box[1] = b_rows; }
  else       { dims[0] = o.N; dims[1] = K; box[0] = 64; box[1] = kLK; }
  if (make_tmap_bf16(&tb, B, 2, dims, str, box)) return -12;
  tb2 = tb;
  if (!b_mn && b2_rows > 0) {
    box[1] = b2_rows;
    if (make_tmap_bf16(&tb2, B, 2, dims, str, box)) return -12;
  }
  auto at16 = [](const void* q, int64_t ld) { return q == nullptr || (!(reinterpret_cast<uintptr_t>(q) & 15) && ld % 8 == 0); };
  o.vec = o.N % 8 == 0 && at16(o.C, o.ldc) && at16(o.res, o.ldres);
  if (o.pre != nullptr && (!at16(o.pre, o.ldpre) || o.ldpre < (o.N + 7) / 8 * 8)) return -10;
  const bool split = p.splits > 1;
  if (!fwd) {
    int rc;
    if (a_mn) rc = split ? lin_launch<true, true, true, false, 0, false>(cut.cg, ta, tb, tb2, a, stream) : lin_launch<true, true, false, false, 0, false>(cut.cg, ta, tb, tb2, a, stream);
    else rc = split ? lin_launch<false, true, true, false, 0, false>(cut.cg, ta, tb, tb2, a, stream) : lin_launch<false, true, false, false, 0, false>(cut.cg, ta, tb, tb2, a, stream);
    return rc || !split ? rc : lin_join<false, 0, false>(cut.cg, a, stream);
  }
  if (split)
    if (int rc = lin_launch<false, false, true, false, 0, false>(cut.cg, ta, tb, tb2, a, stream)) return rc;
#define LLMT_LIN(ACT, RES)                                                                              \
  if (act == ACT && (o.res != nullptr) == RES)                                                          \
    return split ? lin_join<true, ACT, RES>(cut.cg, a, stream) : lin_launch<false, false, false, true, ACT, RES>(cut.cg, ta, tb, tb2, a, stream);
  LLMT_LIN(0, false) LLMT_LIN(1, false) LLMT_LIN(2, false) LLMT_LIN(3, false) LLMT_LIN(4, false)
  LLMT_LIN(0, true) LLMT_LIN(1, true) LLMT_LIN(2, true) LLMT_LIN(3, true) LLMT_LIN(4, true)
#undef LLMT_LIN
  return -4;
}

// Blocks per strip of the form without clusters; 0: few rows and strips, clusters.
static int dz_blocks(int M, int N) {
  if (M <= 2048 && (N + 63) / 64 * kStripBlocks <= 2 * sm_count()) return 0;
  const int strips = (N + 255) / 256, fill = sm_count() * 3 / strips, rows = (M + 31) / 32;      // at least 32 rows per block
  return fill < 1 ? 1 : fill < rows ? fill : rows;
}

template <bool VEC, int LANES, bool CLUSTER, int ACT>
static int dz_launch(const void* dy, int64_t ldy, const void* z, int64_t ldz, void* dz, int64_t lddz, void* db, int db_f32, float* partial, int blocks,
                     int M, int N, cudaStream_t stream) {
  constexpr int COLS = LANES * 8;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((N + COLS - 1) / COLS, blocks);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = 1; at.val.clusterDim.y = kStripBlocks; at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = CLUSTER ? 1 : 0;
  using B = __nv_bfloat16;
  return cudaLaunchKernelEx(&cfg, linear_dz_kernel<VEC, LANES, CLUSTER, ACT>, reinterpret_cast<const B*>(dy), ldy, reinterpret_cast<const B*>(z), ldz,
                            reinterpret_cast<B*>(dz), lddz, db, db_f32, partial, M, N) == cudaSuccess ? 0 : -3;
}
template <int ACT>
static int dz_dispatch(bool vec, int blocks, const void* dy, int64_t ldy, const void* z, int64_t ldz, void* dz, int64_t lddz, void* db, int db_f32,
                       float* partial, int M, int N, cudaStream_t stream) {
  if (blocks == 0)
    return vec ? dz_launch<true, 8, true, ACT>(dy, ldy, z, ldz, dz, lddz, db, db_f32, nullptr, kStripBlocks, M, N, stream)
               : dz_launch<false, 8, true, ACT>(dy, ldy, z, ldz, dz, lddz, db, db_f32, nullptr, kStripBlocks, M, N, stream);
  return vec ? dz_launch<true, 32, false, ACT>(dy, ldy, z, ldz, dz, lddz, db, db_f32, partial, blocks, M, N, stream)
             : dz_launch<false, 32, false, ACT>(dy, ldy, z, ldz, dz, lddz, db, db_f32, partial, blocks, M, N, stream);
}

}  // namespace llmt

using namespace llmt;

// Workspace of a product out [M, N] of depth K whose operands' rows lie lda and ldb elements apart, in floats (0: none is needed): of llmt_linear_dx
// (dz, W) or llmt_linear_dw (dz, x) (`gradient`; act, res and pre 0), or of llmt_linear_act (x, W) with that activation, with a residual (`res`) and
// with z (`pre`).
extern "C" int llmt_linear_max_size() { return kLMostSize; }
extern "C" int64_t llmt_linear_ws_floats(int M, int N, int K, int64_t lda, int64_t ldb, int gradient, int act, int res, int pre) {
  if (act < 0 || act >= kActKinds || M <= 0 || N <= 0 || K <= 0 || M > kLMostSize || N > kLMostSize || K > kLMostSize) return 0;   // refused by the launch
  return lin_ws_floats(M, N, lin_cut(M, N, K, lin_kind(gradient != 0, lda, ldb, act, res != 0, pre != 0)));
}

// How a product with the same arguments is cut: out receives the CTAs of a tile, its columns and the parts along K. Sizes as llmt_linear_act takes them.
extern "C" void llmt_linear_cut(int M, int N, int K, int64_t lda, int64_t ldb, int gradient, int act, int res, int pre, int* out) {
  const LinCut c = lin_cut(M, N, K, lin_kind(gradient != 0, lda, ldb, act < 0 || act >= kActKinds ? 0 : act, res != 0, pre != 0));
  out[0] = c.cg;
  out[1] = c.bn;
  out[2] = c.splits;
}

// y [M][ldy] = x [M][ldx] (rows of N elements, any pitch and start) for TMA: y and its pitch on 16 bytes, at least N rounded up to a multiple of 8.
extern "C" int llmt_linear_pad(const void* x, int64_t ldx, void* y, int64_t ldy, int M, int N, cudaStream_t stream) {
  if (M < 0 || N < 0 || M > kLMostSize || N > kLMostSize || (ldy & 7) || ldy < (int64_t)(N + 7) / 8 * 8 || (reinterpret_cast<uintptr_t>(y) & 15) || (reinterpret_cast<uintptr_t>(x) & 1)) return -10;
  if (M == 0 || N == 0) return 0;
  const int strips = (N + 255) / 256, need = (M + 8 * kPadRows - 1) / (8 * kPadRows), fill = sm_count() * 16 / strips + 1;
  linear_pad_kernel<<<dim3(strips, need < fill ? need : fill), 256, 0, stream>>>(reinterpret_cast<const __nv_bfloat16*>(x), ldx, reinterpret_cast<__nv_bfloat16*>(y), ldy, M, N);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// y [M, N] = act(x [M, K] W [N, K]^T + bias) + res; pre (optional, read by llmt_linear_dz) receives x W^T + bias where there is an activation: rows on
// 16 bytes of at least N values rounded up to a multiple of 8.
extern "C" int llmt_linear_act(const void* x, const void* w, void* y, const void* bias, int bias_f32, const void* res, void* pre, int act, int M, int N,
                               int K, int64_t ldx, int64_t ldw, int64_t ldy, int64_t ldres, int64_t ldpre, float* ws, int64_t ws_floats, int* status,
                               cudaStream_t stream) {
  if (act < 0 || act >= kActKinds) return -10;
  LinArgs a{};
  LinOut& o = a.out;
  o.M = M; o.N = N;
  o.C = reinterpret_cast<__nv_bfloat16*>(y); o.ldc = ldy;
  o.bias = bias; o.bias_f32 = bias_f32;
  o.res = reinterpret_cast<const __nv_bfloat16*>(res); o.ldres = ldres;
  o.pre = reinterpret_cast<__nv_bfloat16*>(pre); o.ldpre = ldpre;
  a.status = status;
  return lin_gemm(x, w, a, K, ldx, ldw, false, false, true, act, ws, ws_floats, stream);
}
// dx [M, K] = dz [M, N] W [N, K]
extern "C" int llmt_linear_dx(const void* dz, const void* w, void* dx, int M, int N, int K, int64_t lddz, int64_t ldw, int64_t lddx, float* ws,
                              int64_t ws_floats, int* status, cudaStream_t stream) {
  LinArgs a{};
  a.out.M = M; a.out.N = K;
  a.out.C = reinterpret_cast<__nv_bfloat16*>(dx); a.out.ldc = lddx;
  a.status = status;
  return lin_gemm(dz, w, a, N, lddz, ldw, false, true, false, 0, ws, ws_floats, stream);
}
// dW [N, K] = dz [M, N]^T x [M, K]
extern "C" int llmt_linear_dw(const void* dz, const void* x, void* dw, int M, int N, int K, int64_t lddz, int64_t ldx, int64_t lddw, float* ws,
                              int64_t ws_floats, int* status, cudaStream_t stream) {
  LinArgs a{};
  a.out.M = N; a.out.N = K;
  a.out.C = reinterpret_cast<__nv_bfloat16*>(dw); a.out.ldc = lddw;
  a.status = status;
  return lin_gemm(dz, x, a, M, lddz, ldx, true, true, false, 0, ws, ws_floats, stream);
}
// Rows of `partial` ([rows][N] floats) that llmt_linear_dz needs for db; 0: none.
extern "C" int llmt_linear_db_partials(int M, int N) { return M > kLMostSize || N <= 0 || N > kLMostSize ? 0 : dz_blocks(M, N); }
// dz = dy act'(z) (act 0: dz = dy; dz nullptr: not written), db = column sums of dz in fp32 before rounding (nullptr: not computed). z and dz have
// rows on 16 bytes of at least N values rounded up to a multiple of 8.
extern "C" int llmt_linear_dz(const void* dy, int64_t ldy, const void* z, int64_t ldz, int act, void* dz, int64_t lddz, void* db, int db_f32,
                              float* partial, int P, int M, int N, cudaStream_t stream) {
  if (M < 0 || N <= 0 || M > kLMostSize || N > kLMostSize || act < 0 || act >= kActKinds || (act != 0 && z == nullptr)) return -10;
  const int blocks = dz_blocks(M, N);
  if (db != nullptr && blocks > 0 && (partial == nullptr || P < blocks)) return -10;
  auto at16 = [](const void* p, int64_t ld) { return p == nullptr || (!(reinterpret_cast<uintptr_t>(p) & 15) && ld % 8 == 0); };
  const int64_t N8 = (N + 7) / 8 * 8;
  if (act && (!at16(z, ldz) || ldz < N8)) return -10;
  if (dz != nullptr && (!at16(dz, lddz) || lddz < N8)) return -10;
  const bool vec = N % 8 == 0 && at16(dy, ldy);
  int rc = -4;
#define LLMT_DZ(ACT) \
  if (act == ACT) rc = dz_dispatch<ACT>(vec, blocks, dy, ldy, z, ldz, dz, lddz, db, db_f32, partial, M, N, stream);
  LLMT_DZ(0) LLMT_DZ(1) LLMT_DZ(2) LLMT_DZ(3) LLMT_DZ(4)
#undef LLMT_DZ
  if (rc || db == nullptr || blocks == 0) return rc;
  linear_db_kernel<<<(N + 31) / 32, 1024, 0, stream>>>(partial, db, db_f32, blocks, N);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
