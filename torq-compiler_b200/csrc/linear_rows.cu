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
// Roles: 8 warps widen (a warp has 32 weight rows, as TMEM's lanes want it), 8 warps scale, round and store what is finished (a tile's sums
// go to registers first, so that the next tile begins while they are stored), one warp multiplies, two copy (steps by turns).
// Blocks are persistent and take every grid-th tile. Tiles of the same weights lie one behind another, so weights and activations both
// come from L2 but for their first use.
#include <algorithm>
#include <atomic>

#include "dependent_launch.cuh"
#include "kernels.h"
#include "tcgen05_ptx.cuh"
#include "tensor_map.h"
#include "widen.cuh"

namespace tb200 {
namespace {

constexpr int kWidenWarps = 8, kFinishWarps = 8, kThreads = (kWidenWarps + kFinishWarps + 4) * 32;
constexpr int kFinishRegs = 152, kWidenRegs = 56, kIssueRegs = 56;
static_assert(256 * kFinishRegs + 256 * kWidenRegs + 128 * kIssueRegs <= kThreads * 96, "register split");
constexpr int kStepK = 64;  // a 128-byte row of activations, a 64-byte row of weights

struct RowsArgs {
  const uint16_t* scale;
  void* y;
  int y_f32, rows, N, steps, row_tiles, tiles;
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
  static constexpr int stages = std::min(8, 208 * 1024 / stage_bytes);
  static constexpr int a_columns = 32 * HALVES;  // of TMEM, a step of widened weights
  static constexpr int a_stages = std::min(8, (512 - HALVES * XN) / a_columns);
  static constexpr int smem = 1024 + stages * stage_bytes;
  static_assert(stage_bytes % 1024 == 0 && a_stages >= 2 && XN % 64 == 0 && XN <= 256, "tile");
};

template <int HALVES, int XN>
__global__ void __launch_bounds__(kThreads, 1) linear_rows_kernel(const RowsArgs a, const __grid_constant__ RowsMaps maps) {
  using S = Shape<HALVES, XN>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[S::stages], empty[S::stages], a_full[S::a_stages], a_empty[S::a_stages], acc_full, acc_empty;
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
      mbar_init(smem_u32(&empty[i]), 1);
    }
    for (int i = 0; i < S::a_stages; i++) {
      mbar_init(smem_u32(&a_full[i]), HALVES * 4);
      mbar_init(smem_u32(&a_empty[i]), 1);
    }
    mbar_init(smem_u32(&acc_full), 1);
    mbar_init(smem_u32(&acc_empty), kFinishWarps);
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

  if (warp < kWidenWarps) {
    // ------------------------------------------------ weights: bytes -> bf16 in TMEM
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWidenRegs));
    const int part = warp >> 2;  // two halves of the rows; or, with one half, every other step
    const int row = (HALVES == 2 ? part * 128 : 0) + (warp & 3) * 32 + lane;
    const uint32_t to = a_tmem + lanes + (HALVES == 2 ? part * 32 : 0);
    uint32_t step = 0;
    for (int t = blockIdx.x; t < a.tiles; t += gridDim.x) {
#pragma unroll 1
      for (int k = 0; k < a.steps; k++, step++) {
        if (HALVES == 1 && (step & 1) != (uint32_t)part) continue;
        const uint32_t s = step % S::stages, as = step % S::a_stages;
        wait(full[s], (step / S::stages) & 1, 321);
        // rows of 64 bytes, whose 16-byte chunks the copy has exchanged by bits 1 and 2 of the row: eight lanes hit every bank once
        const uint32_t from = ring + s * S::stage_bytes + XN * 128 + row * 64;
        uint32_t v[32];
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const uint4 q = lds128(from + ((c ^ (row >> 1 & 3)) << 4));
          widen4(q.x, v[8 * c], v[8 * c + 1]);
          widen4(q.y, v[8 * c + 2], v[8 * c + 3]);
          widen4(q.z, v[8 * c + 4], v[8 * c + 5]);
          widen4(q.w, v[8 * c + 6], v[8 * c + 7]);
        }
        if (step >= S::a_stages) wait(a_empty[as], (step / S::a_stages - 1) & 1, 322);
        __syncwarp();
        tc_fence_after();
        tmem_st32(to + as * S::a_columns, v);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&a_full[as]));
      }
    }
  } else if (warp < kWidenWarps + kFinishWarps) {
    // ------------------------------------------------ finished sums
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFinishRegs));
    constexpr int kColumns = HALVES == 2 ? XN : XN / 2;
    const int part = (warp >> 2) & 1;
    const uint32_t from = tmem + lanes + part * kColumns;
    uint32_t tile = 0;
    for (int t = blockIdx.x; t < a.tiles; t += gridDim.x, tile++) {
      const int n_tile = t / a.row_tiles, r_tile = t - n_tile * a.row_tiles;
      const int n = n_tile * (HALVES * 128) + (HALVES == 2 ? part * 128 : 0) + (warp & 3) * 32 + lane;
      const int row0 = r_tile * XN + (HALVES == 2 ? 0 : part * kColumns), left = min(kColumns, a.rows - row0);  // <= 0: no row
      const bool mine = n < a.N;
      const float scale = mine ? __uint_as_float((uint32_t)__ldg(a.scale + n) << 16) : 0.f;
      wait(acc_full, tile & 1, 323);
      __syncwarp();
      tc_fence_after();
      if (a.y_f32) {
        float* to = (float*)a.y + (long long)row0 * a.N + n;
#pragma unroll 1
        for (int c = 0; c < kColumns; c += 32) {
          uint32_t v[32];
          tmem_ld32_issue(from + c, v);
          tmem_ld_wait32(v);
#pragma unroll
          for (int j = 0; j < 32; j++, to += a.N)
            if (mine && c + j < left) *to = __uint_as_float(v[j]) * scale;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&acc_empty));
      } else {
        uint32_t p[kColumns / 2];
#pragma unroll
        for (int c = 0; c < kColumns; c += 16) {
          uint32_t v[16];
          tmem_ld16(from + c, v);
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float lo = __uint_as_float(v[2 * j]) * scale, hi = __uint_as_float(v[2 * j + 1]) * scale;
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p[c / 2 + j]) : "f"(hi), "f"(lo));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&acc_empty));
        uint16_t* to = (uint16_t*)a.y + (long long)row0 * a.N + n;
#pragma unroll
        for (int j = 0; j < kColumns; j++, to += a.N)
          if (mine && j < left) *to = (uint16_t)(p[j / 2] >> (16 * (j & 1)));
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    const int role = warp - kWidenWarps - kFinishWarps;
    if (role == 0) {
      // ------------------------------------------------ matrix instructions
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(XN >> 3) << 17) | (8u << 24);
      uint32_t step = 0, tile = 0;
      for (int t = blockIdx.x; t < a.tiles; t += gridDim.x, tile++) {
        if (tile) wait(acc_empty, (tile - 1) & 1, 324);
#pragma unroll 1
        for (int k = 0; k < a.steps; k++, step++) {
          const uint32_t s = step % S::stages, as = step % S::a_stages;
          wait(full[s], (step / S::stages) & 1, 325);
          wait(a_full[as], (step / S::a_stages) & 1, 326);
          __syncwarp();
          tc_fence_after();
          const uint64_t x = make_smem_desc(ring + s * S::stage_bytes, 128);
#pragma unroll
          for (int h = 0; h < HALVES; h++)
            mma_f16x4_ts_elect(tmem + h * XN, a_tmem + as * S::a_columns + h * 32, x, 2, idesc, k ? 1u : 0u);
          mma_commit_elect(smem_u32(&empty[s]));
          mma_commit_elect(smem_u32(&a_empty[as]));
        }
        mma_commit_elect(smem_u32(&acc_full));
      }
    } else if (role < 3 && lane == 0) {
      // ------------------------------------------------ copies: two warps, every other step
      uint32_t step = 0;
      for (int t = blockIdx.x; t < a.tiles; t += gridDim.x) {
        const int n_tile = t / a.row_tiles, r_tile = t - n_tile * a.row_tiles;
#pragma unroll 1
        for (int k = 0; k < a.steps; k++, step++) {
          if ((step & 1) != (uint32_t)(role - 1)) continue;
          const uint32_t s = step % S::stages, at = ring + s * S::stage_bytes, bar = smem_u32(&full[s]);
          if (step >= S::stages) wait(empty[s], (step / S::stages - 1) & 1, 327);
          if (gave_up) break;
          mbar_expect_tx(bar, S::stage_bytes);
          tma_load_2d(at, &maps.x, k * kStepK, r_tile * XN, bar);
          tma_load_2d(at + XN * 128, &maps.w, k * kStepK, n_tile * (HALVES * 128), bar);
        }
        if (gave_up) break;
      }
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
cudaError_t run_rows(const LinearRowsArgs& l, int sms, cudaStream_t stream) {
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
  RowsArgs a{l.scale, l.y, l.y_f32, l.rows, l.N, ceil_div(l.K, kStepK), ceil_div(l.rows, XN), 0, l.status, wait_limit_ns()};
  a.tiles = a.row_tiles * ceil_div(l.N, HALVES * 128);
  return launch_dependent(kernel, dim3(std::min(a.tiles, sms)), dim3(kThreads), S::smem, stream, a, m);
}

}  // namespace

cudaError_t launch_linear_rows(const LinearRowsArgs& a, int sms, cudaStream_t stream) {
  return run_rows<2, 192>(a, sms, stream);
}

}  // namespace tb200
