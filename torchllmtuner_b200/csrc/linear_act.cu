// Linear layers with an epilogue: y = act(x W^T + b) + r, and what their gradients need (reference call sites: the biased projections, two-layer
// MLPs and mergers of llmtuner/models/qwen/qwen3_5/multimodal.py:47-290 and llmtuner/models/kimi/kimi_k3/multimodal.py:146-914).
//   z = x W^T + b,  y = act(z) + r;   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_rows dz,  dr = dy.
//
// The products run on tcgen05 with the roles of gemm.cu: one warp issues TMA loads, one the products, eight drain the accumulator; persistent
// workers, each one CTA (128-row tiles) or a pair of CTAs (256-row tiles, cta_group::2). The epilogue of the forward adds the bias, applies the
// activation and adds the residual in fp32 and rounds once; for the backward it also writes z (rounded to bf16: act' of the rounded z is off by
// at most |act''| |z| 2^-9, of the order of the rounding of dz itself). The bias gradient is summed in fp32 from dz before it is rounded.
#include "activations.cuh"
#include "common.cuh"
#include "kernels.h"
#include "vec_io.cuh"

namespace llmt {

int sm_count();
int make_tmap_bf16(CUtensorMap* out, const void* base, int rank, const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box);

constexpr int kLM = 128;                 // rows of a CTA's tile
constexpr int kLK = 64;                  // 64 bf16: one 128-byte swizzle row
constexpr int kLEpiWarps = 8;
constexpr int kLThreads = 64 + 32 * kLEpiWarps;
constexpr int kLMaxStages = 8;
constexpr int kLStageA = kLM * kLK * 2;
constexpr int kLSmem = 227 * 1024;
constexpr int kLSmemFixed = kLEpiWarps * 4096 + 1024 /*alignment*/ + 512 /*barriers*/;

struct LinArgs {
  int M, N, K;
  int bn;                                // tile width over the whole worker, a multiple of 32, at most 256
  int num_m, full_n, tiles;              // tile rows; whole tile columns; tiles (a narrower last column comes last)
  int kb, stages, stage_bytes;
  __nv_bfloat16* C;
  int64_t ldc;
  // forward epilogue
  const void* bias;
  int bias_f32, act;
  const __nv_bfloat16* res;
  int64_t ldres;
  __nv_bfloat16* pre;
  int64_t ldpre;
  int vec;                               // every row of C, res and pre starts on 16 bytes and N is a multiple of 8
  int* status;
};

__device__ __forceinline__ uint32_t lin_idesc(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

struct LinTile { int m, n0, width; };    // tile row, first column, columns computed (a multiple of 32)
__device__ __forceinline__ LinTile lin_tile(const LinArgs& a, int t, int group) {
  const int whole = a.num_m * a.full_n;
  if (t >= whole) {
    const int n0 = a.full_n * a.bn;
    return {t - whole, n0, (a.N - n0 + 31) & ~31};
  }
  // super-rows of `group` tile rows are swept column by column, so concurrent tiles cover a near-square patch and share operands in L2
  const int per = group * a.full_n, g = t / per, first = g * group;
  const int gm = a.num_m - first < group ? a.num_m - first : group;
  const int r = t - g * per;
  return {first + r % gm, (r / gm) * a.bn, a.bn};
}

template <int CG, bool A_MN, bool B_MN, bool EPI>
__global__ void __launch_bounds__(kLThreads, 1) linear_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                                                              const __grid_constant__ LinArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + a.stages * a.stage_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(epi + kLEpiWarps * 4096);
  uint64_t* empty = full + kLMaxStages;
  uint64_t* tfull = empty + kLMaxStages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
  const int unit = blockIdx.x / CG, units = gridDim.x / CG;
  constexpr int kGroup = 16 / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], CG * 32 * kLEpiWarps);
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

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      tma_prefetch_desc(&tmA);
      tma_prefetch_desc(&tmB);
      int stage = 0;
      uint32_t phase = 0, armed = 0, armed_parity = 0;
      bool ok = true;
      const int b_rows = a.bn / CG;                     // rows of B per load (a narrow tile loads as many and uses fewer)
      for (int t = unit; t < a.tiles && ok; t += units) {
        const LinTile tile = lin_tile(a, t, kGroup);
        const int m0 = (tile.m * CG + (int)rank) * kLM, nb = tile.n0 + (int)rank * (tile.width / CG);
        for (int kb = 0; kb < a.kb; ++kb) {
          if (!mbar_wait_bounded(&empty[stage], phase ^ 1, abort_flag, a.status, 500 + stage)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + stage * a.stage_bytes;
          uint8_t* sb = sa + kLStageA;
          if (rank == 0) {
            mbar_arrive_expect_tx(&full[stage], CG * a.stage_bytes);
            armed |= 1u << stage;
            armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
          }
          const int k0 = kb * kLK;
          const uint32_t bar = CG == 2 ? cluster_map_u32(smem_u32(&full[stage]), 0) : 0u;
          auto load = [&](void* dst, const CUtensorMap* m, int c0, int c1) {
            if constexpr (CG == 2) tma_load_2d_pair(dst, m, bar, c0, c1);
            else tma_load_2d(dst, m, &full[stage], c0, c1);
          };
          if constexpr (!A_MN) load(sa, &tmA, k0, m0);
          else {
#pragma unroll
            for (int j = 0; j < kLM / 64; ++j) load(sa + j * (kLK * 128), &tmA, m0 + 64 * j, k0);
          }
          if constexpr (!B_MN) load(sb, &tmB, k0, nb);
          else
            for (int j = 0; j * 64 < b_rows; ++j) load(sb + j * (kLK * 128), &tmB, nb + 64 * j, k0);
          if (++stage == a.stages) { stage = 0; phase ^= 1; }
        }
      }
      if (*abort_flag) {                                // copies in flight land before this CTA's shared memory is released
        for (int s = 0; s < a.stages; ++s) {
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
    if (lane == 0 && rank == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = unit; t < a.tiles && ok; t += units) {
        const uint32_t idesc = lin_idesc(kLM * CG, lin_tile(a, t, kGroup).width, A_MN, B_MN);
        if (!mbar_wait_bounded<CG == 2>(&tempty[acc], acc_phase ^ 1, abort_flag, a.status, 600 + acc)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * 256;
        for (int kb = 0; kb < a.kb; ++kb) {
          if (!mbar_wait_bounded(&full[stage], phase, abort_flag, a.status, 700 + stage)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * a.stage_bytes), sb = sa + kLStageA;
          const uint32_t la = desc_lo(sa, A_MN ? kLK * 128 : 16), lb = desc_lo(sb, B_MN ? kLK * 128 : 16);
          const uint32_t acc0 = kb ? 1u : 0u;
#pragma unroll
          for (int k = 0; k < kLK / 16; ++k) {
            const uint64_t da = desc_pack(la + (A_MN ? k * 128 : k * 2));
            const uint64_t db = desc_pack(lb + (B_MN ? k * 128 : k * 2));
            if constexpr (CG == 2) umma_bf16_ss_pair(d_tmem, da, db, idesc, k ? 1u : acc0);
            else umma_bf16_ss(d_tmem, da, db, idesc, k ? 1u : acc0);
          }
          if constexpr (CG == 2) umma_commit_pair(&empty[stage]);
          else umma_commit(&empty[stage]);
          if (++stage == a.stages) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        if constexpr (CG == 2) umma_commit_pair(&tfull[acc]);
        else umma_commit(&tfull[acc]);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue
    // A warp turns 32 rows x 32 columns (fp32) around in shared memory, so that global accesses run along rows. Two warps share a quarter of
    // the rows and take alternate chunks of columns.
    const int quarter = warp & 3, side = (warp - 2) >> 2;
    uint8_t* stg = epi + (warp - 2) * 4096;
    const int rr0 = lane >> 3, cc = lane & 7;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int t = unit; t < a.tiles; t += units) {
      const LinTile tile = lin_tile(a, t, kGroup);
      const int row0 = (tile.m * CG + (int)rank) * kLM + quarter * 32;
      const int cols = min(tile.width, a.N - tile.n0);
      if (EPI && a.res != nullptr) {                    // the residual's rows come into L2 while the product is computed
        const int pr = min(row0 + lane, a.M - 1);
        const uint8_t* line = reinterpret_cast<const uint8_t*>(a.res + (int64_t)pr * a.ldres + tile.n0);
        for (int o = side * 128; o < cols * 2; o += 256) asm volatile("prefetch.global.L2 [%0];" ::"l"(line + o));
      }
      if (!mbar_wait_bounded(&tfull[acc], acc_phase, abort_flag, a.status, 800 + acc)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * 256;
#pragma unroll 1
      for (int c = side * 32; c < cols; c += 64) {
        uint32_t r[32];
        tmem_ld_32x32(t_row + c, r);
        const int col0 = tile.n0 + c;
        if (a.vec) {
          const int col = col0 + cc * 4;
          const bool col_ok = col < a.N;
          uint2 old[8];
          float bias[4] = {0.f, 0.f, 0.f, 0.f};
          if constexpr (EPI) {
            if (a.bias != nullptr && col_ok) {
              if (a.bias_f32) load_vec<float, 4>(reinterpret_cast<const float*>(a.bias) + col, bias);
              else load_vec<__nv_bfloat16, 4>(reinterpret_cast<const __nv_bfloat16*>(a.bias) + col, bias);
            }
            if (a.res != nullptr) {                     // clamped instead of skipped: eight loads in flight together
              const int64_t at = col_ok ? col : tile.n0;
#pragma unroll
              for (int it = 0; it < 8; ++it)
                old[it] = *reinterpret_cast<const uint2*>(a.res + (int64_t)min(row0 + rr0 + it * 4, a.M - 1) * a.ldres + at);
            }
          }
          tmem_wait_ld();
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(stg + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
          __syncwarp();
#pragma unroll
          for (int it = 0; it < 8; ++it) {
            const int rr = it * 4 + rr0, row = row0 + rr;
            const uint4 v = *reinterpret_cast<const uint4*>(stg + rr * 128 + ((cc ^ (rr & 7)) << 4));
            float o[4] = {__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
            if constexpr (EPI) {
#pragma unroll
              for (int j = 0; j < 4; ++j) o[j] += bias[j];
              if (a.pre != nullptr && col_ok && row < a.M) store_vec<__nv_bfloat16, 4>(a.pre + (int64_t)row * a.ldpre + col, o);
              activate<4>(a.act, o);
              if (a.res != nullptr) {
                float q[4];
                unpack_bf16x2(old[it].x, q);
                unpack_bf16x2(old[it].y, q + 2);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] += q[j];
              }
            }
            if (col_ok && row < a.M) store_vec<__nv_bfloat16, 4>(a.C + (int64_t)row * a.ldc + col, o);
          }
        } else {                                        // rows off a 16-byte boundary: a lane per column, one row after another
          tmem_wait_ld();
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; ++j) reinterpret_cast<uint32_t*>(stg)[lane * 32 + ((j + lane) & 31)] = r[j];
          __syncwarp();
          const int col = col0 + lane;
          if (col < a.N) {
            float bias = 0.f;
            if constexpr (EPI) {
              if (a.bias != nullptr) bias = a.bias_f32 ? reinterpret_cast<const float*>(a.bias)[col] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.bias)[col]);
            }
#pragma unroll 4
            for (int rr = 0; rr < 32; ++rr) {
              const int row = row0 + rr;
              if (row >= a.M) break;
              float o[1] = {__uint_as_float(reinterpret_cast<uint32_t*>(stg)[rr * 32 + ((lane + rr) & 31)])};
              if constexpr (EPI) {
                o[0] += bias;
                if (a.pre != nullptr) a.pre[(int64_t)row * a.ldpre + col] = __float2bfloat16_rn(o[0]);
                activate<1>(a.act, o);
                if (a.res != nullptr) o[0] += __bfloat162float(a.res[(int64_t)row * a.ldres + col]);
              }
              a.C[(int64_t)row * a.ldc + col] = __float2bfloat16_rn(o[0]);
            }
          }
        }
      }
      tc_fence_before();
      if constexpr (CG == 2) mbar_arrive_cluster(cluster_map_u32(smem_u32(&tempty[acc]), 0));
      else mbar_arrive(&tempty[acc]);
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
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

// ------------------------------------------------------------------------------------------ dz and db
// A block owns a strip of columns and every eighth group of rows; the eight blocks of a cluster add their column sums through distributed
// shared memory in rank order, so db needs neither a second launch nor a workspace nor atomics.
constexpr int kStripBlocks = 8;
template <int V, int THREADS>
__global__ void __launch_bounds__(THREADS) linear_dz_kernel(const __nv_bfloat16* __restrict__ dy, int64_t ldy, const __nv_bfloat16* __restrict__ z,
                                                            int64_t ldz, int act, __nv_bfloat16* __restrict__ dz, int64_t lddz, void* __restrict__ db,
                                                            int db_f32, int M, int N) {
  constexpr int LANES = V == 8 ? 8 : 32, COLS = LANES * V, ROWS = THREADS / LANES;
  __shared__ float part[ROWS][COLS + 1];
  __shared__ float total[COLS];
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  const int col = blockIdx.x * COLS + lane * V;
  const uint32_t rank = blockIdx.y;
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  if (col < N) {
#pragma unroll 4
    for (int64_t row = (int64_t)rank * ROWS + sub; row < M; row += ROWS * kStripBlocks) {
      float g[V];
      load_vec<__nv_bfloat16, V>(dy + row * ldy + col, g);
      if (z != nullptr) {
        float p[V];
        load_vec<__nv_bfloat16, V>(z + row * ldz + col, p);
        activate_grad<V>(act, p, g);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += g[j];
      if (dz != nullptr) store_vec<__nv_bfloat16, V>(dz + row * lddz + col, g);
    }
  }
  if (db == nullptr) return;
#pragma unroll
  for (int j = 0; j < V; ++j) part[sub][lane * V + j] = acc[j];
  __syncthreads();
  if (threadIdx.x < COLS) {
    float s = 0.f;
#pragma unroll 8
    for (int i = 0; i < ROWS; ++i) s += part[i][threadIdx.x];
    total[threadIdx.x] = s;
  }
  cluster_sync();
  const int oc = blockIdx.x * COLS + threadIdx.x;
  if (rank == 0 && threadIdx.x < COLS && oc < N) {
    float s = total[threadIdx.x];
    for (int k = 1; k < kStripBlocks; ++k) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_map_u32(smem_u32(&total[threadIdx.x]), k)));
      s += v;
    }
    if (db_f32) reinterpret_cast<float*>(db)[oc] = s;
    else reinterpret_cast<__nv_bfloat16*>(db)[oc] = __float2bfloat16_rn(s);
  }
  cluster_sync();                                       // no block leaves while its sums are being read
}

// ------------------------------------------------------------------------------------------ host
// Function attributes belong to a device: remembered per device.
template <typename F>
static bool allow_smem(F kern, int bytes, uint64_t& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (dev < 64 && (done >> dev & 1)) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  if (dev < 64) done |= 1ull << dev;
  return true;
}

template <int CG, bool A_MN, bool B_MN, bool EPI>
static int lin_launch(const CUtensorMap& ta, const CUtensorMap& tb, const LinArgs& a, cudaStream_t stream) {
  static uint64_t done = 0;
  auto kern = linear_kernel<CG, A_MN, B_MN, EPI>;
  if (!allow_smem(kern, kLSmem, done)) return -2;
  const int most = sm_count() / CG;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((a.tiles < most ? a.tiles : most) * CG);
  cfg.blockDim = dim3(kLThreads);
  cfg.dynamicSmemBytes = a.stages * a.stage_bytes + kLSmemFixed;
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = CG; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = CG == 2 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, ta, tb, a) == cudaSuccess ? 0 : -3;
}

// C[M, N] = op(A) op(B) as in llmt_gemm_bf16 (tn, nn and tt layouts); e: the forward's epilogue, or nullptr.
static int lin_gemm(const void* A, const void* B, LinArgs a, int64_t lda, int64_t ldb, bool a_mn, bool b_mn, bool epi, cudaStream_t stream) {
  if (a.M <= 0 || a.N <= 0) return 0;
  if (a.K <= 0 || (lda & 7) || (ldb & 7) || (reinterpret_cast<uintptr_t>(A) & 15) || (reinterpret_cast<uintptr_t>(B) & 15)) return -10;
  if ((epi && (a_mn || b_mn)) || (a_mn && !b_mn)) return -4;
  const int cg = a.M > kLM ? 2 : 1;
  a.bn = a.N > 128 ? 256 : 128;
  a.num_m = (a.M + kLM * cg - 1) / (kLM * cg);
  a.full_n = a.N / a.bn;
  a.tiles = a.num_m * (a.full_n + (a.N % a.bn ? 1 : 0));
  a.kb = (a.K + kLK - 1) / kLK;
  const int b_rows = a.bn / cg;
  a.stage_bytes = kLStageA + (b_mn ? (b_rows + 63) / 64 * 64 : b_rows) * kLK * 2;
  a.stages = (kLSmem - kLSmemFixed) / a.stage_bytes;
  if (a.stages > kLMaxStages) a.stages = kLMaxStages;
  CUtensorMap ta, tb;
  uint64_t dims[2], str[1] = {(uint64_t)lda * 2};
  uint32_t box[2];
  if (!a_mn) { dims[0] = a.K; dims[1] = a.M; box[0] = kLK; box[1] = kLM; }
  else       { dims[0] = a.M; dims[1] = a.K; box[0] = 64; box[1] = kLK; }
  if (make_tmap_bf16(&ta, A, 2, dims, str, box)) return -11;
  str[0] = (uint64_t)ldb * 2;
  if (!b_mn) { dims[0] = a.K; dims[1] = a.N; box[0] = kLK; box[1] = b_rows; }
  else       { dims[0] = a.N; dims[1] = a.K; box[0] = 64; box[1] = kLK; }
  if (make_tmap_bf16(&tb, B, 2, dims, str, box)) return -12;
  auto at16 = [](const void* p, int64_t ld) { return p == nullptr || (!(reinterpret_cast<uintptr_t>(p) & 15) && ld % 8 == 0); };
  a.vec = a.N % 8 == 0 && at16(a.C, a.ldc) && at16(a.res, a.ldres) && at16(a.pre, a.ldpre) && !(reinterpret_cast<uintptr_t>(a.bias) & 15);
#define LLMT_LIN(AM, BMN, E) \
  if (a_mn == AM && b_mn == BMN && epi == E) \
    return cg == 2 ? lin_launch<2, AM, BMN, E>(ta, tb, a, stream) : lin_launch<1, AM, BMN, E>(ta, tb, a, stream);
  LLMT_LIN(false, false, true) LLMT_LIN(false, true, false) LLMT_LIN(true, true, false)
#undef LLMT_LIN
  return -4;
}

template <int V, int THREADS>
static int dz_launch(const void* dy, int64_t ldy, const void* z, int64_t ldz, int act, void* dz, int64_t lddz, void* db, int db_f32, int M, int N,
                     cudaStream_t stream) {
  constexpr int COLS = V == 8 ? 64 : 32;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((N + COLS - 1) / COLS, kStripBlocks);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = 1; at.val.clusterDim.y = kStripBlocks; at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  using B = __nv_bfloat16;
  return cudaLaunchKernelEx(&cfg, linear_dz_kernel<V, THREADS>, reinterpret_cast<const B*>(dy), ldy, reinterpret_cast<const B*>(z), ldz, act,
                            reinterpret_cast<B*>(dz), lddz, db, db_f32, M, N) == cudaSuccess ? 0 : -3;
}

}  // namespace llmt

using namespace llmt;

// y [M, N] = act(x [M, K] W [N, K]^T + bias) + res; pre (optional) receives x W^T + bias.
extern "C" int llmt_linear_act(const void* x, const void* w, void* y, const void* bias, int bias_f32, const void* res, void* pre, int act, int M, int N,
                               int K, int64_t ldx, int64_t ldw, int64_t ldy, int64_t ldres, int64_t ldpre, int* status, cudaStream_t stream) {
  if (act < 0 || act >= kActKinds) return -10;
  LinArgs a{};
  a.M = M; a.N = N; a.K = K;
  a.C = reinterpret_cast<__nv_bfloat16*>(y); a.ldc = ldy;
  a.bias = bias; a.bias_f32 = bias_f32; a.act = act;
  a.res = reinterpret_cast<const __nv_bfloat16*>(res); a.ldres = ldres;
  a.pre = reinterpret_cast<__nv_bfloat16*>(pre); a.ldpre = ldpre;
  a.status = status;
  return lin_gemm(x, w, a, ldx, ldw, false, false, true, stream);
}
// dx [M, K] = dz [M, N] W [N, K]
extern "C" int llmt_linear_dx(const void* dz, const void* w, void* dx, int M, int N, int K, int64_t lddz, int64_t ldw, int64_t lddx, int* status,
                              cudaStream_t stream) {
  LinArgs a{};
  a.M = M; a.N = K; a.K = N;
  a.C = reinterpret_cast<__nv_bfloat16*>(dx); a.ldc = lddx;
  a.status = status;
  return lin_gemm(dz, w, a, lddz, ldw, false, true, false, stream);
}
// dW [N, K] = dz [M, N]^T x [M, K]
extern "C" int llmt_linear_dw(const void* dz, const void* x, void* dw, int M, int N, int K, int64_t lddz, int64_t ldx, int64_t lddw, int* status,
                              cudaStream_t stream) {
  LinArgs a{};
  a.M = N; a.N = K; a.K = M;
  a.C = reinterpret_cast<__nv_bfloat16*>(dw); a.ldc = lddw;
  a.status = status;
  return lin_gemm(dz, x, a, lddz, ldx, true, true, false, stream);
}
// dz = dy act'(z) (z nullptr: dz = dy; dz nullptr: not written), db = column sums of dz in fp32 before rounding (nullptr: not computed).
extern "C" int llmt_linear_dz(const void* dy, int64_t ldy, const void* z, int64_t ldz, int act, void* dz, int64_t lddz, void* db, int db_f32, int M,
                              int N, cudaStream_t stream) {
  if (M < 0 || N <= 0 || act < 0 || act >= kActKinds) return -10;
  auto at16 = [](const void* p, int64_t ld) { return p == nullptr || (!(reinterpret_cast<uintptr_t>(p) & 15) && ld % 8 == 0); };
  const bool vec = N % 8 == 0 && at16(dy, ldy) && at16(z, ldz) && at16(dz, lddz);
  return vec ? dz_launch<8, 512>(dy, ldy, z, ldz, act, dz, lddz, db, db_f32, M, N, stream)
             : dz_launch<1, 512>(dy, ldy, z, ldz, act, dz, lddz, db, db_f32, M, N, stream);
}
