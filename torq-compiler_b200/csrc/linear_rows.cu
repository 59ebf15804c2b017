// Products of more rows than a decode step has with int8 weights: y[r][n] = scale[n] * sum_k x[r][k] w[n][k], x bf16, sums fp32.
//
// What bounds it: 2 rows N K operations at the rate of bf16 on the tensor cores, once there are a few hundred rows (4000 x 13824 x 1152:
// 127 G operations). Integers below 2^7 are exact in bf16, so the weights are widened on their way and only the sum is ever rounded.
// Which operand goes where follows from shared memory, whose 128 bytes a clock are the scarce thing. With the weights as A in TMEM they
// pass through it once, as bytes: copied in, read by the widening warps, who store the bf16 straight to TMEM; the instruction then reads
// only B, the activations, from shared memory. (Widened weights in shared memory would be written and read there at twice the bytes.) For
// a step of 64 along K a tile of 256 x 192 moves 40 KB in, 16 KB to the widening warps and 2 x 24 KB to the instructions, which take 768
// clocks over it. A result's row of TMEM is then a weight row, so its scale is one number a thread, and 32 lanes store 32 neighbouring
// outputs of one row: no alignment of N is needed.
//
// Roles: 16 warps widen, as teams of four that take 128 weight rows of a step by turns (a warp has 32 of them, as TMEM's lanes want it): eight
// warps took 1050 clocks over a step of 256 rows, most of it the latency of their own chain, where the instructions take 768; with 16 a step
// takes 770. Eight warps finish: they scale, round and turn patches of 32 x 32 in shared memory, so that they store 16 bytes a lane (stored 2
// bytes a lane straight from TMEM, a tile took longer than its products: 127 us against 102 for 4000 x 13824 x 1152). One or two multiply (one
// for each half, whose sums are its own), two copy (steps by turns).
// Blocks are persistent and take every grid-th tile. Tiles of the same weights lie one behind another, so weights and activations both
// come from L2 but for their first use. Where tiles are few, a cluster of up to eight blocks shares one, a part of K each, and adds the parts
// up over distributed shared memory in their order: 128 x 1152 x 6912 in 12.7 us (32 with a block to a tile).
// Measured from memory: 4000 x 13824 x 1152 104 us (1.22 PFLOP/s) in a loop of its own; 125 us where the plain form in fp32 runs in between
// and has used up the power budget.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "dependent_launch.cuh"
#include "kernels.h"
#include "tcgen05_ptx.cuh"
#include "tensor_map.h"
#include "widen.cuh"

namespace tb200 {
namespace {

constexpr int kWidenTeams = 4, kWidenWarps = 4 * kWidenTeams, kFinishWarps = 8, kThreads = (kWidenWarps + kFinishWarps + 4) * 32;
constexpr int kFinishRegs = 120, kWidenRegs = 56, kIssueRegs = 40, kLaunchRegs = 72;  // the last: what a launch of so many threads is given
static_assert(kFinishWarps * 32 * kFinishRegs + kWidenWarps * 32 * kWidenRegs + 128 * kIssueRegs <= kThreads * kLaunchRegs, "register split");
constexpr int kPatchPitch = 144, kPatch = 16 * kPatchPitch;  // 16 rows of 32 words, eight lanes of a 16-byte read on different banks
constexpr int kStepK = 64;  // a 128-byte row of activations, a 64-byte row of weights

struct RowsArgs {
  const uint16_t* scale;
  void* y;
  int y_f32, rows, N, steps, row_tiles, tiles;
  int splits;  // blocks of a cluster that share a tile, a part of K each (then a block has one tile)
  int* status;
  unsigned long long wait_ns;
};
struct RowsMaps {
  CUtensorMap x, w;
};

// HALVES x 128 weight rows by XN activation rows.
template <int HALVES, int XN>
struct Shape {
  static constexpr int stage_bytes = XN * 128 + HALVES * 8192;
  static constexpr int stages = std::min(8, (226 * 1024 - 1024 - kFinishWarps * kPatch) / stage_bytes);
  static constexpr int a_columns = 32 * HALVES;  // of TMEM, a step of widened weights
  static constexpr int a_stages = std::min(8, (512 - HALVES * XN) / a_columns);
  static constexpr int smem = 1024 + stages * stage_bytes + kFinishWarps * kPatch;
  static_assert(stage_bytes % 1024 == 0 && a_stages >= 2 && XN % 64 == 0 && XN <= 256, "tile");
  // A team sees every team_step-th step. It tells a stage's copies from the ones before by one bit, which takes that it sees all of that stage's, or
  // that the ones before have been multiplied when it comes to wait (it has waited for room of its last step, a_stages behind).
  static constexpr int team_step = kWidenTeams / HALVES;
  static_assert(stages % team_step == 0 || team_step + a_stages <= stages, "phases told apart");
};

template <int HALVES, int XN>
__global__ void __launch_bounds__(kThreads, 1) linear_rows_kernel(const RowsArgs a, const __grid_constant__ RowsMaps maps) {
  using S = Shape<HALVES, XN>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[S::stages], empty[S::stages], a_full[S::a_stages][HALVES], a_empty[S::a_stages][HALVES], acc_full[HALVES], acc_empty[HALVES];
  __shared__ uint32_t tmem_at;
  __shared__ int abort;
  const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_at)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 32) {
    for (int i = 0; i < S::stages; i++) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), HALVES);
    }
    for (int h = 0; h < HALVES; h++) {
      for (int i = 0; i < S::a_stages; i++) {
        mbar_init(smem_u32(&a_full[i][h]), 4);
        mbar_init(smem_u32(&a_empty[i][h]), 1);
      }
      mbar_init(smem_u32(&acc_full[h]), 1);
      mbar_init(smem_u32(&acc_empty[h]), kFinishWarps / HALVES);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    abort = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at, a_tmem = tmem + HALVES * XN;
  grid_dependency_wait();
  grid_dependency_release();

  // One wait that runs out ends all others: every role then runs through without waiting, and the results are not used.
  bool gave_up = false;
  auto wait = [&](uint64_t& bar, uint32_t parity, int code) {
    const uint32_t at = smem_u32(&bar);
    if (mbar_poll(at, parity, 16) || gave_up) return;
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_poll(at, parity, 64)) {
      if (globaltimer_ns() - t0 > a.wait_ns) *(volatile int*)&abort = code;
      if (*(volatile int*)&abort) {
        gave_up = true;
        return;
      }
    }
  };
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;  // of TMEM, this warp's
  // this block's tiles, and its steps of each
  const int rank = blockIdx.x % a.splits, first_tile = blockIdx.x / a.splits, stride = gridDim.x / a.splits;
  const int k0 = a.steps * rank / a.splits, steps = a.steps * (rank + 1) / a.splits - k0;
  auto cluster_sync = [&]() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  };

  if (warp < kWidenWarps) {
    // ------------------------------------------------ weights: bytes -> bf16 in TMEM
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWidenRegs));
    // a unit is 128 rows of a step: units go to the teams of four warps by turns
    const int own_row = (warp & 3) * 32 + lane;
    const uint32_t tiles = (a.tiles - first_tile + stride - 1) / stride, units = tiles * steps * HALVES;
#pragma unroll 1
    for (uint32_t unit = warp >> 2; unit < units; unit += kWidenTeams) {
      const uint32_t step = unit / HALVES, half = unit % HALVES, s = step % S::stages, as = step % S::a_stages;
      wait(full[s], (step / S::stages) & 1, 321);
      // rows of 64 bytes, whose 16-byte chunks the copy has exchanged by bits 1 and 2 of the row: eight lanes hit every bank once
      const uint32_t from = ring + s * S::stage_bytes + XN * 128 + (half * 128 + own_row) * 64;
      uint32_t v[32];
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const uint4 q = lds128(from + ((c ^ (own_row >> 1 & 3)) << 4));
        widen4(q.x, v[8 * c], v[8 * c + 1]);
        widen4(q.y, v[8 * c + 2], v[8 * c + 3]);
        widen4(q.z, v[8 * c + 4], v[8 * c + 5]);
        widen4(q.w, v[8 * c + 6], v[8 * c + 7]);
      }
      if (step >= S::a_stages) wait(a_empty[as][half], (step / S::a_stages - 1) & 1, 322);
      __syncwarp();
      tc_fence_after();
      tmem_st32(a_tmem + lanes + half * 32 + as * S::a_columns, v);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&a_full[as][half]));
    }
    if (a.splits > 1) {
      cluster_sync();
      cluster_sync();
    }
  } else if (warp < kWidenWarps + kFinishWarps) {
    // ------------------------------------------------ finished sums
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFinishRegs));
    constexpr int kColumns = HALVES == 2 ? XN : XN / 2;
    const int part = (warp >> 2) & 1, half = HALVES == 2 ? part : 0;
    const uint32_t from = tmem + lanes + part * kColumns, patch = ring + S::stages * S::stage_bytes + (warp - kWidenWarps) * kPatch;
    uint32_t tile = 0;
    for (int t = first_tile; t < a.tiles; t += stride, tile++) {
      const int n_tile = t / a.row_tiles, r_tile = t - n_tile * a.row_tiles;
      const int n0 = n_tile * (HALVES * 128) + half * 128 + (warp & 3) * 32;
      const int row0 = r_tile * XN + (HALVES == 2 ? 0 : part * kColumns), left = min(kColumns, a.rows - row0);  // <= 0: no row
      const float scale = n0 + lane < a.N ? __uint_as_float((uint32_t)__ldg(a.scale + n0 + lane) << 16) : 0.f;
      wait(acc_full[half], tile & 1, 323);
      __syncwarp();
      tc_fence_after();
      if (a.splits > 1) {
        // The parts of K meet over the cluster: of every four columns one block adds up what all have, in the order of K. What it is sent lies
        // in its ring, which nobody needs any more once all blocks of the cluster have multiplied.
        cluster_sync();
        const uint32_t box = ring + (warp - kWidenWarps) * (kColumns / 4) * 512 + lane * 16;
#pragma unroll 1
        for (int c = 0; c < kColumns; c += 16) {
          uint32_t v[16];
          tmem_ld16(from + c, v);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int g = c / 4 + j;
            uint32_t to;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(box + (g - g % a.splits + rank) * 512), "r"(g % a.splits));
            asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(v[4 * j]), "r"(v[4 * j + 1]), "r"(v[4 * j + 2]), "r"(v[4 * j + 3]) : "memory");
          }
        }
        tc_fence_before();
        cluster_sync();
#pragma unroll 1
        for (int g = rank; g < kColumns / 4; g += a.splits) {
          float f[4] = {};
          for (int i = 0; i < a.splits; i++) {
            const uint4 q = lds128(box + (g - rank + i) * 512);
            f[0] += __uint_as_float(q.x); f[1] += __uint_as_float(q.y); f[2] += __uint_as_float(q.z); f[3] += __uint_as_float(q.w);
          }
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int row = row0 + 4 * g + j;
            if (n0 + lane >= a.N || row >= a.rows) continue;
            const long long at = (long long)row * a.N + n0 + lane;
            if (a.y_f32) ((float*)a.y)[at] = f[j] * scale;
            else ((uint16_t*)a.y)[at] = __bfloat16_as_ushort(__float2bfloat16_rn(f[j] * scale));
          }
        }
        break;
      }
      uint32_t v[32];
      tmem_ld32_issue(from, v);
#pragma unroll 1
      for (int c = 0; c < kColumns; c += 32) {
        tmem_ld_wait32(v);
        float f[32];
#pragma unroll
        for (int j = 0; j < 32; j++) f[j] = __uint_as_float(v[j]) * scale;
        if (c + 32 < kColumns) {
          tmem_ld32_issue(from + c + 32, v);
        } else {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&acc_empty[half]));
        }
        const int rows = min(32, left - c);  // of this patch
        if (rows <= 0) continue;
        if (a.y_f32) {
#pragma unroll
          for (int h = 0; h < 32; h += 16) {
#pragma unroll
            for (int j = 0; j < 16; j++) sts32(patch + j * kPatchPitch + lane * 4, __float_as_uint(f[h + j]));
            __syncwarp();
            float* const to = (float*)a.y + (long long)(row0 + c + h) * a.N + n0;
            if (a.N % 4 == 0) {
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const int j = i * 4 + (lane >> 3), at = (lane & 7) * 4;
                const uint4 q = lds128(patch + j * kPatchPitch + at * 4);
                if (h + j < rows && n0 + at < a.N) *reinterpret_cast<uint4*>(to + (long long)j * a.N + at) = q;
              }
            } else {
              for (int j = 0; j < 16; j++)
                if (h + j < rows && n0 + lane < a.N) to[(long long)j * a.N + lane] = __uint_as_float(lds32(patch + j * kPatchPitch + lane * 4));
            }
            __syncwarp();
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; j++) {  // a word: two rows of one column
            uint32_t w;
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(f[2 * j + 1]), "f"(f[2 * j]));
            sts32(patch + j * kPatchPitch + lane * 4, w);
          }
          __syncwarp();
          uint16_t* const to = (uint16_t*)a.y + (long long)(row0 + c) * a.N + n0;
          if (a.N % 8 == 0) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const int j = i * 8 + (lane >> 2), at = (lane & 3) * 8;
              const uint4 q = lds128(patch + j * kPatchPitch + at * 4), r = lds128(patch + j * kPatchPitch + at * 4 + 16);
              const uint4 even = make_uint4(__byte_perm(q.x, q.y, 0x5410), __byte_perm(q.z, q.w, 0x5410), __byte_perm(r.x, r.y, 0x5410), __byte_perm(r.z, r.w, 0x5410));
              const uint4 odd = make_uint4(__byte_perm(q.x, q.y, 0x7632), __byte_perm(q.z, q.w, 0x7632), __byte_perm(r.x, r.y, 0x7632), __byte_perm(r.z, r.w, 0x7632));
              uint16_t* const row = to + (long long)(2 * j) * a.N + at;
              if (n0 + at < a.N) {
                if (2 * j < rows) *reinterpret_cast<uint4*>(row) = even;
                if (2 * j + 1 < rows) *reinterpret_cast<uint4*>(row + a.N) = odd;
              }
            }
          } else {
            for (int j = 0; j < 16; j++) {
              const uint32_t w = lds32(patch + j * kPatchPitch + lane * 4);
              if (n0 + lane < a.N) {
                if (2 * j < rows) to[(long long)(2 * j) * a.N + lane] = (uint16_t)w;
                if (2 * j + 1 < rows) to[(long long)(2 * j + 1) * a.N + lane] = (uint16_t)(w >> 16);
              }
            }
          }
          __syncwarp();
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    const int role = warp - kWidenWarps - kFinishWarps;
    if (role < HALVES) {
      // ------------------------------------------------ matrix instructions: a warp for each half, whose sums are its own
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(XN >> 3) << 17) | (8u << 24);
      const uint32_t sums = tmem + role * XN, widened = a_tmem + role * 32;
      uint32_t step = 0, tile = 0;
      for (int t = first_tile; t < a.tiles; t += stride, tile++) {
        if (tile) wait(acc_empty[role], (tile - 1) & 1, 324);
#pragma unroll 1
        for (int k = 0; k < steps; k++, step++) {
          const uint32_t s = step % S::stages, as = step % S::a_stages;
          wait(a_full[as][role], (step / S::a_stages) & 1, 326);  // whose warps have seen the step's copies arrive, the activations among them
          __syncwarp();
          tc_fence_after();
          mma_f16x4_ts_elect(sums, widened + as * S::a_columns, make_smem_desc(ring + s * S::stage_bytes, 128), 2, idesc, k ? 1u : 0u);
          mma_commit_elect(smem_u32(&a_empty[as][role]));
          mma_commit_elect(smem_u32(&empty[s]));
        }
        mma_commit_elect(smem_u32(&acc_full[role]));
      }
    } else if (role >= 2 && lane == 0) {
      // ------------------------------------------------ copies: two warps, every other step
      uint32_t step = 0;
      for (int t = first_tile; t < a.tiles; t += stride) {
        const int n_tile = t / a.row_tiles, r_tile = t - n_tile * a.row_tiles;
#pragma unroll 1
        for (int k = 0; k < steps; k++, step++) {
          if ((step & 1) != (uint32_t)(role & 1)) continue;
          const uint32_t s = step % S::stages, at = ring + s * S::stage_bytes, bar = smem_u32(&full[s]);
          if (step >= S::stages) wait(empty[s], (step / S::stages - 1) & 1, 327);
          if (gave_up) break;
          mbar_expect_tx(bar, S::stage_bytes);
          tma_load_2d(at, &maps.x, (k0 + k) * kStepK, r_tile * XN, bar);
          tma_load_2d(at + XN * 128, &maps.w, (k0 + k) * kStepK, n_tile * (HALVES * 128), bar);
        }
        if (gave_up) break;
      }
    }
    if (a.splits > 1) {
      cluster_sync();
      cluster_sync();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    if (*(volatile int*)&abort) {
      if (lane == 0) report_expired_wait(a.status, abort);
      __nanosleep(1000000);  // let what is in flight land after a failed wait
    }
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

bool encode_2d(CUtensorMap* map, const void* base, CUtensorMapDataType type, int bytes, uint64_t inner, uint64_t outer, uint32_t box_outer, CUtensorMapSwizzle swizzle) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {inner * bytes};
  cuuint32_t box[2] = {kStepK, box_outer};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <int HALVES, int XN>
cudaError_t run_rows(const LinearRowsArgs& l, int splits, int sms, cudaStream_t stream) {
  using S = Shape<HALVES, XN>;
  auto kernel = linear_rows_kernel<HALVES, XN>;
  static std::atomic<unsigned long long> attr_done;
  if (first_use_on_device(attr_done)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
    if (e != cudaSuccess) return e;
    mark_used_on_device(attr_done);
  }
  RowsMaps m{};
  if (!encode_2d(&m.x, l.x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, l.K, l.rows, XN, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_2d(&m.w, l.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, l.K, l.N, HALVES * 128, CU_TENSOR_MAP_SWIZZLE_64B))
    return cudaErrorInvalidValue;
  RowsArgs a{l.scale, l.y, l.y_f32, l.rows, l.N, ceil_div(l.K, kStepK), ceil_div(l.rows, XN), 0, splits, l.status, wait_limit_ns()};
  a.tiles = a.row_tiles * ceil_div(l.N, HALVES * 128);
  return launch_dependent_cluster(splits, kernel, dim3(splits > 1 ? a.tiles * splits : std::min(a.tiles, sms)), dim3(kThreads), S::smem, stream, true, a, m);
}

}  // namespace

// Shapes, with what a step of K and everything else of a tile took (microseconds). With 5 us for the launch these give 40 times (four shapes at ten
// sizes: 33 to 4000 rows, N of 1152 to 13824, K of 1152 to 6912) within 22 %, most of them too low by a tenth, and the shape they pick was the
// fastest at each of the ten. In the order of the list: 4000 x 13824 x 1152 105 / 122 / 143 / 230 us, 1000 x 13824 x 1152 (an earlier form, whole
// K) 41 / 35 / 41 / 64, 1000 x 1152 x 6912 29 / 35 / 25 / 33, 300 x 1536 x 1152 16.8 / 14.6 / 12.6 / 10.6.
struct RowsShape {
  int halves, xn;
  float step, tile;
};
constexpr RowsShape kShapes[] = {{2, 192, 0.43f, 5.0f}, {2, 128, 0.38f, 3.2f}, {1, 128, 0.23f, 1.7f}, {1, 64, 0.225f, 0.9f}};
constexpr float kMeet = 2.5f;  // what it takes a cluster to start and to add up its parts

// Blocks that fit at once in clusters of p: a cluster lies within one of the machine's groups of 16 to 20 processors. (128 x 1152 x 6912 as 18
// clusters of 8 took 21 us, in two goes, as 18 of 4 14.6, as 9 of 8 12.8.)
int cluster_blocks(int p, int sms) { return p == 8 ? sms * 3 / 4 : p == 4 ? sms * 7 / 8 : sms; }

cudaError_t launch_linear_rows(const LinearRowsArgs& a, int sms, cudaStream_t stream) {
  const int steps = ceil_div(a.K, kStepK);
  int best = 0, splits = 1;
  float least = INFINITY;
  for (int i = 0; i < 4; i++) {
    const RowsShape& s = kShapes[i];
    const long long tiles = (long long)ceil_div(a.N, s.halves * 128) * ceil_div(a.rows, s.xn);
    for (int p = 1; p <= 8 && (p == 1 || (tiles * p <= cluster_blocks(p, sms) && 2 * p <= steps)); p *= 2) {
      const float t = (float)((tiles * p + sms - 1) / sms) * (ceil_div(steps, p) * s.step + s.tile) + (p > 1 ? kMeet : 0.0f);
      if (t < least) least = t, best = i, splits = p;
    }
  }
  return best == 0 ? run_rows<2, 192>(a, splits, sms, stream) : best == 1 ? run_rows<2, 128>(a, splits, sms, stream)
       : best == 2 ? run_rows<1, 128>(a, splits, sms, stream) : run_rows<1, 64>(a, splits, sms, stream);
}

}  // namespace tb200
