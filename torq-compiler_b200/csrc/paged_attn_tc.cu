// Attention of many rows over a paged cache on the tensor cores (paged.cuh, paged.h: tiles and the sharing-out of their work).
//
// A tile is 128 rows: up to 128 / group tokens with the query heads of one key/value head. Per block of 128 keys: S = Q K^T into TMEM
// (fp32), softmax in registers against a running maximum, P as bf16 back into TMEM, O += P V with P as the TMEM operand. S is double
// buffered, so the product of the next block runs while this block's softmax does; O (up to 256 columns) and both S fill TMEM.
// P is one bf16 a weight (half a step off, each by itself, while the row's sum is of the unrounded ones): results are off by 0.0021 to 0.0024, relative,
// where rounding the result alone gives 0.0017. A second term, as the kernel for few rows has it, would double the products with V and what the
// softmax, which bounds this kernel, has to convert and store.
//   p = 2^((s - m) scale log2 e), sums in fp32; m is the row's maximum, but follows it only when it has grown by more than 2^8 in
//   p (O and the sum are scaled then): a bound serves as well as the maximum itself, and most blocks leave O alone.
// Warps: eight for softmax (two to a row quarter, half a row's keys each); four that ask the copy engine for bf16 keys and values, or eight that
// widen int8 ones; and one each for matrix instructions, items, queries and the keys' places. Each key's place comes from the page table, so
// any page size and any sequence end fits; a unit is 128 keys x 64 dims in the 128-byte swizzle, zeros where a key is seen by no row of
// the tile. Keys are the K-major operand, values the same bytes read as MN-major. int8 caches are widened to bf16 (exact) on the way; the
// keys' scales meet the scores, the values' scales P.
// Work is shared out evenly: all tiles' key blocks in one row, every block of the grid takes an equal piece. A tile that falls to several
// leaves partial sums in memory, which the launch behind adds up in their order.
// What bounds it is the chain of the softmax, and the issue of copies and matrix instructions beside it; not the tensor cores. In a loop, the
// launch for the joins included: a prompt of 4096 tokens, 4 query heads of 256, 67 us (0.51 PFLOP/s of pairs that are seen; half of the blocks
// on the diagonal are not); 2000 tokens behind 7000, 32/8 heads of 128, 331 us on bf16 (0.79 PFLOP/s), 655 us on int8 (0.40), whose
// widening warps share the issue slots with the softmax.
#include <algorithm>

#include "dependent_launch.cuh"
#include "kernels.h"
#include "paged_row.cuh"
#include "paged_work.cuh"
#include "tcgen05_ptx.cuh"
#include "tensor_map.h"

namespace tb200 {

namespace {

// four warpgroups: two for softmax, one that widens int8 caches, one with a warp each for matrix instructions, items and the copy engine; the
// registers go where they are needed (of the 512 x 128 that a block starts with)
constexpr int kSoftmaxWarps = 8;
template <bool I8>
constexpr int kCopyWarpsOf = I8 ? 8 : 4;  // four widening warps took twice as long over a block as all else
template <bool I8>
constexpr int kThreadsOf = (kSoftmaxWarps + kCopyWarpsOf<I8> + 4) * 32;
// a block starts with 128 (bf16) or 96 (int8) registers a thread (int8, 1999 rows of five chunks, 32/8 heads of 128: 248 us so, 258 with 144 and 64)
constexpr int kSoftmaxRegs = 200, kSoftmaxRegsI8 = 152, kCopyRegsI8 = 56, kIssueRegs = 56;
static_assert(256 * kSoftmaxRegsI8 + 256 * kCopyRegsI8 + 128 * kIssueRegs <= kThreadsOf<true> * 96, "register split, int8");
static_assert(256 * kSoftmaxRegs + 256 * kIssueRegs <= kThreadsOf<false> * 128, "register split, bf16");
constexpr int kSoftmaxThreads = kSoftmaxWarps * 32;
constexpr int kUnit = 128 * 128;  // bytes of 128 rows of 64 bf16 values
constexpr int kMetaBlocks = 6, kItems = 4;
using TileScratch = RowsScratch<kSoftmaxThreads>;  // rows are computed once more by the softmax warps

struct alignas(16) Meta {
  float k_scale[kKeyBlock], v_scale[kKeyBlock];
  int slot[kKeyBlock];  // where the cache holds the key, -1 where no row of the tile sees it or nothing is held
  uint32_t holds[4];    // the keys with a slot, a bit each
  // column c holds key key0 + c; where that lies in front of a window's part of the keys, one of the first tokens. Rows see what lies in front of
  // `firsts` whatever their window (here, beside the slots, and not with the item: the softmax has no register left for it)
  int key0, firsts;
};
static_assert(sizeof(Meta) % 16 == 0, "what lies behind it in shared memory is read 8 bytes at a time");
struct Control {
  uint64_t full[16], empty[16], s_full[2], p_ready[2], pv_done, o_done, q_full, q_empty, item_full[kItems], item_empty[kItems], meta_full[kMetaBlocks], meta_empty[kMetaBlocks];
  Item items[kItems];
  uint32_t tmem;
  int abort;
  int stop;   // of the softmax warps: 1 when there is no more work, 2 when a wait ran out
  int again;  // a tile of this block alone has rows that came out non-finite
  float top[2][2][128];  // row maxima of the two halves, by parity of the block
  WorkShared work;
  Work share;  // for mend_tiles
};

// two fp32 operations in one instruction
__device__ __forceinline__ unsigned long long pack_f32(float x, float y) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack_f32(unsigned long long v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ unsigned long long add_f32x2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long mul_f32x2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long fma_f32x2(unsigned long long a, unsigned long long b, unsigned long long d) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(d));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float d) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(d));
  return r;
}
__device__ __forceinline__ bool pair_any(int id, bool x) {  // of 64 threads
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 p, %2, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, 64, p;\n\t"
      "selp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"((int)x)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void sts128(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Rows of the tiles that a block has done alone, and whose result is not finite, once more (rare: an infinity or a NaN among the values, a row without
// a key). By the softmax warps, which have written these results.
__device__ __noinline__ void mend_tiles(const AttnPagedArgs& a, const Control& control, TileScratch& sm, int t) {
  auto sync = [] { named_sync(5, kSoftmaxThreads); };
  const int group = a.n_q / a.v.n_kv, D = a.v.D;
  const Work& work = control.share;
  ItemCursor cursor(a, work, control.work);
  Item w;
  while (cursor.take(a, work, w)) {
    if (w.b1 - w.b0 != w.blocks) continue;  // the join's
    const int used = w.tokens * group;
    for (int r0 = 0; r0 < used; r0 += 32) {
      const int r = r0 + (t >> 3), tok = page_of(r, a.group_div);  // eight threads look at a row
      bool bad = false;
      if (r < used) {
        const uint16_t* const row = a.out + ((long long)(w.row0 + tok) * a.n_q + w.head * group + r - tok * group) * D;
        for (int d = (t & 7) * 8; d < D; d += 64) {
          const uint4 x = *reinterpret_cast<const uint4*>(row + d);
          for (uint32_t y : {x.x, x.y, x.z, x.w}) bad = bad || (y & 0x7f80u) == 0x7f80u || (y & 0x7f800000u) == 0x7f800000u;
        }
      }
      const uint32_t by8 = __ballot_sync(0xffffffffu, bad);
      sync();
      if ((t & 31) == 0) sm.any[t >> 5] = (by8 & 0xff ? 1u : 0u) | (by8 & 0xff00 ? 2u : 0u) | (by8 & 0xff0000 ? 4u : 0u) | (by8 >> 24 ? 8u : 0u);
      sync();
      uint32_t bits = 0;
      for (int i = 0; i < kSoftmaxWarps; i++) bits |= sm.any[i] << (4 * i);
      if (bits) attend_rows<kSoftmaxThreads>(a, sm, t, {w.row0, w.head, w.seq, w.first_pos}, r0, bits, 0, D, sync);
    }
  }
}

// How the copy engine sees the queries and a bf16 cache: boxes of 64 dims by the rows of a tile / by box_rows keys, and single keys.
struct TileMaps {
  CUtensorMap q, k, v, k_rows, v_rows;
};

// DC: units (64 dims) of a head. UNITS: ring of keys' and values' units in shared memory. (mend_tiles takes the arguments by address: from where the
// launch has put them the prompt of 4096 takes 67 us, by way of a copy on the stack 70.)
template <int DC, int UNITS, int AHEAD, bool I8>
__global__ void __launch_bounds__(kThreadsOf<I8>, 1) attn_paged_tile_kernel(const __grid_constant__ AttnPagedArgs a, const __grid_constant__ TileMaps maps) {
  constexpr int GROUPS = UNITS / DC;  // a block's keys, or its values, lie one behind another: a group
  constexpr int kCopyWarps = kCopyWarpsOf<I8>, kCopyThreads = kCopyWarps * 32, kThreads = kThreadsOf<I8>;
  extern __shared__ unsigned char smem_raw[];
  // [Q units][ring units] on 1024-byte boundaries, then the rest
  unsigned char* const base = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t q_smem = smem_u32(base), ring = q_smem + DC * kUnit;
  unsigned char* const raw = base + (DC + UNITS) * kUnit;  // int8 pieces on their way
  Meta* const meta = reinterpret_cast<Meta*>(raw + (I8 ? AHEAD * kUnit / 2 : 0));
  Control& c = *reinterpret_cast<Control*>(meta + kMetaBlocks);
  int* const first_tile = reinterpret_cast<int*>(base);  // while the work is shared out: tiles in front of each sequence

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PagedView& v = a.v;
  const int group = a.n_q / v.n_kv, D = v.D, tpt = a.tokens_per_tile;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&c.tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 32) {
    for (int i = 0; i < GROUPS; i++) {
      mbar_init(smem_u32(&c.full[i]), I8 ? kCopyWarps * DC : DC);
      mbar_init(smem_u32(&c.empty[i]), 1);
    }
    for (int i = 0; i < 2; i++) {  // a softmax warp may be one block ahead of another: a barrier for each buffer
      mbar_init(smem_u32(&c.s_full[i]), 1);
      mbar_init(smem_u32(&c.p_ready[i]), kSoftmaxWarps);
    }
    mbar_init(smem_u32(&c.pv_done), 1);
    mbar_init(smem_u32(&c.o_done), 1);
    for (int i = 0; i < kItems; i++) {
      mbar_init(smem_u32(&c.item_full[i]), 1);
      mbar_init(smem_u32(&c.item_empty[i]), kSoftmaxThreads + 96 + kCopyThreads);
    }
    for (int i = 0; i < kMetaBlocks; i++) {
      mbar_init(smem_u32(&c.meta_full[i]), 1);
      mbar_init(smem_u32(&c.meta_empty[i]), 1);
    }
    mbar_init(smem_u32(&c.q_full), 1);
    mbar_init(smem_u32(&c.q_empty), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    c.abort = 0;
    c.again = 0;
  }
  grid_dependency_wait();
  grid_dependency_release();

  if (tid == 0) a.joins[blockIdx.x].parts = 0;
  const Work work = share_out<kThreads>(a, c.work, first_tile);
  const bool works = work.works;
  if (tid == 0) c.share = work;  // (kept in a register it would cost the softmax one)
  // first_tile lies where queries and units will be: the copy engine's writes come behind every thread's accesses to it
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncthreads();  // the first item is known, and first_tile's room is free
  tc_fence_after();
  const uint32_t tmem = c.tmem;

  // One wait that runs out ends all others at once: every role then runs through without waiting, and the results are not used. (Kept short: it
  // stands in many places, and what bounds this kernel next to its copies is how many instructions its roles have in the cache.)
  bool gave_up = false;
  auto wait = [&](uint64_t& bar, uint32_t parity, int code) {
    const uint32_t at = smem_u32(&bar);
    if (mbar_poll(at, parity, 16) || gave_up) return;
    const unsigned long long t0 = globaltimer_ns();
    while (!mbar_poll(at, parity, 64)) {
      if (globaltimer_ns() - t0 > a.wait_ns) *(volatile int*)&c.abort = code;
      if (*(volatile int*)&c.abort) {
        gave_up = true;
        return;
      }
    }
  };

  // The roles take the block's items from a ring that a warp of its own fills. The reference stays valid until release_item.
  auto take_item = [&](uint32_t i) -> const Item& {
    wait(c.item_full[i % kItems], (i / kItems) & 1, 310);
    return c.items[i % kItems];
  };
  auto take_meta = [&](uint32_t block) -> const Meta& {  // it stays until the block's values have been multiplied
    wait(c.meta_full[block % kMetaBlocks], (block / kMetaBlocks) & 1, 312);
    return meta[block % kMetaBlocks];
  };
  auto release_item = [&](uint32_t i) { mbar_arrive(smem_u32(&c.item_empty[i % kItems])); };
  const uint32_t o_tmem = tmem + 256;
  if (warp >= kSoftmaxWarps && warp < kSoftmaxWarps + kCopyWarps) {
    // ------------------------------------------------ copies of int8 caches: widened on the way
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(I8 ? kCopyRegsI8 : kIssueRegs));
    if (I8 && works) {
    // A thread has the same piece of 16 bytes of two rows of every unit: what it asks for lands in room of its own, AHEAD units ahead of being
    // widened, so nothing but its own copies has to be waited for.
    const int t = tid - kSoftmaxThreads, piece = t & 3, row0 = t >> 2;
    const uint32_t own = smem_u32(raw) + t * 32;
    const long long row_bytes = (long long)v.n_kv * D;
    uint32_t unit = 0, block0 = 0;
    for (uint32_t items = 0;; items++) {
      const Item& w = take_item(items);
      if (__any_sync(0xffffffffu, gave_up || !w.tokens)) break;
      const int n = w.b1 - w.b0, units = 2 * DC * n;
      const long long head_bytes = (long long)w.head * D + piece * 16;
      release_item(items);
      auto ask = [&](int i) {  // unit i of the item: the keys of block 0, then those of block b and the values of b - 1, by turns
        if (i < units) {
          const int j = i + DC, b = j / (2 * DC), r = j - b * 2 * DC;  // (so that b = 0 begins with the keys of block 0 at r = DC)
          const bool keys = r >= DC ? b == 0 : b < n;
          const int block = keys ? b : b - 1, u = r >= DC ? r - DC : r;
          const Meta& m = take_meta(block0 + block);
          const char* const pages = (const char*)(keys ? a.k : a.vv) + head_bytes + u * 64;
          const bool in = u * 64 + piece * 16 < D;
          int slot[2];
#pragma unroll
          for (int k = 0; k < 2; k++) slot[k] = in ? m.slot[row0 + 64 * k] : -1;
          const uint32_t dst = own + (i % AHEAD) * (kUnit / 2);
#pragma unroll
          for (int k = 0; k < 2; k++) copy16(dst + k * 16, pages + max(slot[k], 0) * row_bytes, slot[k] >= 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll 1
      for (int i = 0; i < AHEAD; i++) ask(i);
#pragma unroll 1
      for (int i = 0; i < units; i++, unit++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
        const uint32_t part = unit / DC;
        if (part >= GROUPS) wait(c.empty[part % GROUPS], (part / GROUPS - 1) & 1, 301);
        const uint32_t dst = ring + (unit % UNITS) * kUnit + row0 * 128, from = own + (i % AHEAD) * (kUnit / 2);
        const uint32_t lo_at = ((2 * piece) ^ (row0 & 7)) << 4, hi_at = ((2 * piece + 1) ^ (row0 & 7)) << 4;  // a thread's rows are 64 apart
        uint4 x[2];
#pragma unroll
        for (int k = 0; k < 2; k++) x[k] = lds128(from + k * 16);
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const uint4 q = x[k];
          uint4 lo, hi;
          widen4(q.x, lo.x, lo.y); widen4(q.y, lo.z, lo.w);
          widen4(q.z, hi.x, hi.y); widen4(q.w, hi.z, hi.w);
          sts128(dst + k * 8192 + lo_at, lo);
          sts128(dst + k * 8192 + hi_at, hi);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&c.full[part % GROUPS]));
        ask(i + AHEAD);
      }
      block0 += n;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    }
    if (!I8 && works) {
    // bf16: by the copy engine, the units by turns to the warps (one warp's round of waiting for room and asking takes 0.3 us, which alone would
    // bound the copies at 52 GB/s an SM; two warps reached 100, four 128 on all SMs at once).
    // A run of R = box_rows keys to a lane: one box where all have a slot (they then follow one another) or none has (from outside the
    // cache: zeros). Runs with some, and all keys where pages end anywhere (no box), go four keys to a lane.
    const int own = warp - kSoftmaxWarps;
    const int R = a.box_rows ? a.box_rows : kKeyBlock, log_r = 31 - __clz(R), runs = a.box_rows ? kKeyBlock >> log_r : 0, none = v.pages * v.page_size;
    uint32_t unit0 = 0, block0 = 0;
    for (uint32_t items = 0;; items++) {
      const Item& w = take_item(items);
      if (__any_sync(0xffffffffu, gave_up || !w.tokens)) break;
      const int n = w.b1 - w.b0, units = 2 * DC * n, head = w.head;
      release_item(items);
#pragma unroll 1
      for (int i = (own - (int)unit0) & (kCopyWarps - 1); i < units; i += kCopyWarps) {
        const int j = i + DC, b = j / (2 * DC), r0 = j - b * 2 * DC;  // as for int8: K(0), K(1), V(0), K(2), V(1), ...
        const bool keys = r0 >= DC ? b == 0 : b < n;
        const int block = keys ? b : b - 1, u = r0 >= DC ? r0 - DC : r0;
        const uint32_t unit = unit0 + i, part = unit / DC, bar = smem_u32(&c.full[part % GROUPS]), dst = ring + unit % UNITS * kUnit;
        if (part >= GROUPS) wait(c.empty[part % GROUPS], (part / GROUPS - 1) & 1, 301);
        // (behind the wait for room: a warp passes over blocks, and a parity is told from the one before the last only while it is near)
        const Meta& m = take_meta(block0 + block);
        __syncwarp();
        if (lane == 0) mbar_expect_tx(bar, kUnit);
        // how many of this lane's run have a slot: whole words of the bits, or a part of one
        const int at = min(lane << log_r, kKeyBlock - 1);
        bool all_held = true, any_held = false;
        if (R >= 32) {
          for (int k = 0; k < R; k += 32) {
            const uint32_t word = m.holds[min((at + k) >> 5, 3)];
            all_held = all_held && word == 0xffffffffu;
            any_held = any_held || word;
          }
        } else {
          const uint32_t mask = (1u << R) - 1, word = m.holds[at >> 5] >> (at & 31) & mask;
          all_held = word == mask;
          any_held = word != 0;
        }
        const bool in_part = any_held && !all_held;
        const uint32_t parts = runs ? __ballot_sync(0xffffffffu, lane < runs && in_part) : 0xffffffffu;
        __syncwarp();
        if (lane < runs && !in_part) tma_load_3d(dst + (lane << log_r) * 128, keys ? &maps.k : &maps.v, u * 64, head, all_held ? m.slot[at] : none, bar);
        if (parts && (!runs || (parts >> (4 * lane >> log_r) & 1))) {
          const int4 x = *reinterpret_cast<const int4*>(&m.slot[4 * lane]);  // this lane's four, by themselves
          auto row = [&](int s) { return s < 0 ? -1 : s * v.n_kv + head; };
          tma_gather4(dst + lane * 512, keys ? &maps.k_rows : &maps.v_rows, u * 64, row(x.x), row(x.y), row(x.z), row(x.w), bar);
        }
      }
      unit0 += units;
      block0 += n;
    }
    }
  } else if (warp >= kSoftmaxWarps + kCopyWarps) {
    // ------------------------------------------------ matrix instructions
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (works && warp == kSoftmaxWarps + kCopyWarps) {
    // operands of 128-byte rows, 8-row groups 1024 bytes apart, 128-byte swizzle; values as MN-major: 64 dims, then the next unit
    auto desc = [](uint32_t at, uint32_t lead) {
      return (uint64_t)(((at & 0x3FFFF) >> 4) | (lead >> 4 << 16)) | (uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32;
    };
    const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kKeyBlock >> 3) << 17) | (8u << 24);
    const uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);
    // (what bounds this role is its own instructions, one behind another: descriptors and phases are stepped, not worked out)
    const uint64_t q0 = desc(q_smem, 16), k0 = desc(ring, 16), v0 = desc(ring, kUnit);
    uint32_t group_at = 0, turn = 0, blocks = 0;  // the group to be used next, its phase
    auto take_group = [&](int code) {
      wait(c.full[group_at], turn, code);
      tc_fence_after();
    };
    auto release_group = [&]() {
      mma_commit_elect(smem_u32(&c.empty[group_at]));
      if (++group_at == GROUPS) {
        group_at = 0;
        turn ^= 1;
      }
    };
    for (uint32_t items = 0;; items++) {
      const Item& w = take_item(items);
      const int n = w.b1 - w.b0;
      if (__any_sync(0xffffffffu, gave_up || !w.tokens)) break;
      release_item(items);
      wait(c.q_full, items & 1, 303);
      for (int b = 0; b <= n; b++) {
        if (b < n) {  // scores of block b
          const uint32_t s_tmem = tmem + ((blocks + b) & 1) * 128;
          const uint64_t kb = k0 + group_at * (DC * (kUnit >> 4));
          take_group(304);
          if (D == DC * 64) {
#pragma unroll
            for (int u = 0; u < DC; u++) mma_f16x4_elect(s_tmem, q0 + u * (kUnit >> 4), kb + u * (kUnit >> 4), idesc_s, u ? 1u : 0u);
          } else {
#pragma unroll 1
            for (int k = 0; k < (D >> 4); k++) {
              const uint32_t at = (k >> 2) * (kUnit >> 4) + (k & 3) * 2;
              mma_f16_elect(s_tmem, q0 + at, kb + at, idesc_s, k ? 1u : 0u);
            }
          }
          mma_commit_elect(smem_u32(&c.s_full[(blocks + b) & 1]));
          release_group();
          if (b == n - 1) mma_commit_elect(smem_u32(&c.q_empty));
        }
        if (b > 0) {  // sums of block b - 1: all dims in one instruction
          const uint32_t g = blocks + b - 1, p_tmem = tmem + (g & 1) * 128;
          const uint64_t vb = v0 + group_at * (DC * (kUnit >> 4));
          wait(c.p_ready[g & 1], (g >> 1) & 1, 305);
          take_group(306);
          // keys 0..63 of P lie in columns 0..31, keys 64..127 in columns 64..95
          mma_f16x4_ts_elect(o_tmem, p_tmem, vb, 2048 >> 4, idesc_o, b > 1 ? 1u : 0u);
          mma_f16x4_ts_elect(o_tmem, p_tmem + 64, vb + 4 * (2048 >> 4), 2048 >> 4, idesc_o, 1u);
          mma_commit_elect(smem_u32(&c.pv_done));
          release_group();
          mma_commit_elect(smem_u32(&c.meta_empty[g % kMetaBlocks]));
          if (b == n) mma_commit_elect(smem_u32(&c.o_done));
        }
      }
      blocks += n;
    }
    } else if (works && warp == kSoftmaxWarps + kCopyWarps + 2) {
      // ---------------------------------------------- queries, by the copy engine
      for (uint32_t items = 0;; items++) {
        const Item& w = take_item(items);
        if (__any_sync(0xffffffffu, gave_up || !w.tokens)) break;
        const int head = w.head, q_row = w.row0;
        release_item(items);
        if (items) wait(c.q_empty, (items - 1) & 1, 302);
        __syncwarp();
        if (lane == 0) {  // rows of the tile's tokens, in the tile's order; those behind the last token are somebody's or nobody's, and are not used
          const uint32_t bar = smem_u32(&c.q_full);
          mbar_expect_tx(bar, DC * 128 * tpt * group);
#pragma unroll 1
          for (int u = 0; u < DC; u++) tma_load_3d(q_smem + u * kUnit, &maps.q, u * 64, head * group, q_row, bar);
        }
      }
    } else if (works && warp == kSoftmaxWarps + kCopyWarps + 3) {
      // ---------------------------------------------- which keys, and where: four to a lane, a block's page ids asked for a block ahead
      uint32_t blocks = 0;
      for (uint32_t items = 0;; items++) {
        const Item& w = take_item(items);
        if (__any_sync(0xffffffffu, gave_up || !w.tokens)) break;
        const int b0 = w.b0, b1 = w.b1, head = w.head;
        const Keys keys_of(a, w);
        release_item(items);
        int next_page[4];
        auto ask_block = [&](int b) {
#pragma unroll
          for (int i = 0; i < 4; i++) next_page[i] = keys_of.ask(keys_of.at(b * kKeyBlock + 4 * lane) + i);
        };
        ask_block(b0);
        for (int b = b0; b < b1; b++, blocks++) {
          const int key0 = keys_of.at(b * kKeyBlock + 4 * lane);  // of this lane's four
          int slot[4];
          uint32_t held = 0;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            slot[i] = keys_of.slot(key0 + i, next_page[i]);
            held |= (slot[i] >= 0 ? 1u : 0u) << (4 * (lane & 7) + i);
          }
          if (b + 1 < b1) ask_block(b + 1);
          float ks[4] = {}, vs[4] = {};
          if (I8) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float* sc = a.scales + (long long)max(slot[i], 0) * 2 * v.n_kv + head;
              const float k1 = __ldg(sc), v1 = __ldg(sc + v.n_kv);
              // what makes a key's scores units of log2; it must not be zero where it meets a hidden key's -inf, and the smallest
              // number in its place leaves every finite score below 2^-20
              const float k2 = k1 * (a.scale * 1.4426950408889634f);
              ks[i] = slot[i] < 0 || k2 == 0.f ? __int_as_float(1) : k2;
              vs[i] = slot[i] < 0 ? 0.f : v1;
            }
          }
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) held |= __shfl_xor_sync(0xffffffffu, held, o);
          const uint32_t at = blocks % kMetaBlocks;
          if (blocks >= kMetaBlocks) wait(c.meta_empty[at], (blocks / kMetaBlocks - 1) & 1, 313);
          Meta& m = meta[at];
          *reinterpret_cast<int4*>(&m.slot[4 * lane]) = make_int4(slot[0], slot[1], slot[2], slot[3]);
          if (I8) {
            *reinterpret_cast<float4*>(&m.k_scale[4 * lane]) = make_float4(ks[0], ks[1], ks[2], ks[3]);
            *reinterpret_cast<float4*>(&m.v_scale[4 * lane]) = make_float4(vs[0], vs[1], vs[2], vs[3]);
          }
          if ((lane & 7) == 0) m.holds[lane >> 3] = held;
          if (lane == 0) {
            m.key0 = b * kKeyBlock + keys_of.shift;
            m.firsts = keys_of.front ? keys_of.front + keys_of.shift : keys_of.sinks;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&c.meta_full[at]));
        }
      }
    } else if (works && warp == kSoftmaxWarps + kCopyWarps + 1 && lane == 0) {
      // ---------------------------------------------- the block's items
      ItemCursor cursor(a, work, c.work);
      for (uint32_t i = 0;; i++) {
        if (i >= kItems) wait(c.item_empty[i % kItems], (i / kItems - 1) & 1, 311);
        if (gave_up) break;
        const bool more = cursor.take(a, work, c.items[i % kItems]);
        mbar_arrive(smem_u32(&c.item_full[i % kItems]));
        if (!more) break;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(I8 ? kSoftmaxRegsI8 : kSoftmaxRegs));
    if (works) {
    // ------------------------------------------------ softmax: thread = (row, half of the block's keys)
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int tok = page_of(row, a.group_div);
    const float cexp = a.scale * 1.4426950408889634f;
    uint32_t blocks = 0, items = 0;
    for (;; items++) {
      if (tid == 0) {  // one decides for all, who meet at barriers from here on
        const Item& w = take_item(items);
        c.stop = gave_up || *(volatile int*)&c.abort ? 2 : !w.tokens;
      }
      named_sync(5, kSoftmaxThreads);
      if (c.stop) break;
      const Item& w = c.items[items % kItems];
      const int tokens = w.tokens, used = tokens * group, n = w.b1 - w.b0, first_pos = w.first_pos;
      const bool warp_used = (warp & 3) * 32 < used;
      const int pos = (int)min((long long)first_pos + min(tok, tokens - 1), 0x7fffffffll);
      const int last_pos = (int)min((long long)first_pos + tokens - 1, 0x7fffffffll);
      const int near = a.window ? max(0, pos - a.window + 1) : 0;  // this row sees keys [near, pos] and those in front of `firsts`
      float m = -INFINITY, base = 0.f, sum = 0.f;  // base: what the exponents are taken from, m or (before there is one) zero
      for (int b = 0; b < n; b++, blocks++) {
        const uint32_t s_tmem = tmem + lanes + (blocks & 1) * 128 + half * 64;
        if (!warp_used) {  // rows of nobody: P keeps what it holds, and so does O
          wait(c.s_full[blocks & 1], (blocks >> 1) & 1, 307);
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&c.p_ready[blocks & 1]));
          continue;
        }
        const Meta& mt = take_meta(blocks);
        const int key0 = mt.key0 + half * 64;
        // whether some row of the tile does not see some key of this half
        const bool partial = (mt.holds[half * 2] & mt.holds[half * 2 + 1]) != 0xffffffffu || key0 + 63 > first_pos ||
                             (a.window && key0 < max(0, last_pos - a.window + 1) && key0 + 63 >= mt.firsts);
        wait(c.s_full[blocks & 1], (blocks >> 1) & 1, 307);
        tc_fence_after();
        // Of 32 scores, of columns 32 k on, those of keys this row does not see become -inf. The loops over them stay rolled up: a
        // processor's four quarters each run this beside other roles, and what does not fit their instruction buffers is waited for.
        auto hide = [&](int k, uint32_t (&s)[32]) {
          if (partial) {
            // bits of the keys this row sees: not behind its position, inside the window or among the first, and held
            auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
            auto upto = [](int n) { return n < 0 ? 0u : n >= 31 ? 0xffffffffu : (2u << n) - 1u; };
            const int k0 = key0 + 32 * k;
            const uint32_t see = upto(pos - k0) & (~below(near - k0) | below(mt.firsts - k0)) & mt.holds[half * 2 + k];
            if (__all_sync(0xffffffffu, see == 0xffffffffu)) return;  // most of a partial block is seen by all
#pragma unroll
            for (int i = 0; i < 32; i++) s[i] = see >> i & 1 ? s[i] : 0xff800000u;
          }
        };
        // four scores in units of log2
        auto scale4 = [&](const uint32_t (&s)[32], int i, const float* scale, float (&x)[4]) {
          const float4 by = I8 ? *reinterpret_cast<const float4*>(scale) : make_float4(cexp, cexp, cexp, cexp);
          x[0] = __uint_as_float(s[i]) * by.x; x[1] = __uint_as_float(s[i + 1]) * by.y;
          x[2] = __uint_as_float(s[i + 2]) * by.z; x[3] = __uint_as_float(s[i + 3]) * by.w;
        };
        float part;
        uint32_t p[32];  // two weights each; they take the place of the scores once these are not needed again
        for (bool follow = b == 0;;) {
          if (follow) {  // the row's maximum so far; m follows it where p would grow beyond 2^8, or had none yet
            float top = -INFINITY;
#pragma unroll 1
            for (int k = 0; k < 2; k++) {
              uint32_t s[32];
              tmem_ld32_issue(s_tmem + 32 * k, s);
              tmem_ld_wait32(s);
              hide(k, s);
              float tops[2] = {top, -INFINITY};
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                float x[4];
                scale4(s, i, mt.k_scale + half * 64 + 32 * k + i, x);
                tops[0] = max3(tops[0], x[0], x[1]);
                tops[1] = max3(tops[1], x[2], x[3]);
              }
              top = fmaxf(tops[0], tops[1]);
            }
            c.top[blocks & 1][half][row] = top;
            named_sync(1 + (warp & 3), 64);
            top = fmaxf(top, c.top[blocks & 1][half ^ 1][row]);
            float keep = 1.f;
            if (top > m && (b == 0 || !(top - m <= 8.f))) {
              keep = m == -INFINITY ? 0.f : exp2_fast(m - top);
              m = top;
              base = top;
            }
            if (b > 0) {
              sum *= keep;
              // these scores were issued behind the sums of the block before the last: its phase is over, the last one's is waited for
              wait(c.pv_done, (blocks - 1) & 1, 308);
              tc_fence_after();
#pragma unroll 1
              for (int i = 32 * half; i < D; i += 64) {  // columns behind D belong to nobody
                uint32_t o[32];
                tmem_ld32_issue(o_tmem + lanes + i, o);
                tmem_ld_wait32(o);
#pragma unroll
                for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
                tmem_st32(o_tmem + lanes + i, o);
              }
            }
          }
          // p = 2^(s c - base) in one multiply-add: how base was rounded is the same for every key of the row, so it cancels (where that factor
          // itself leaves fp32, at scores beyond 10^9, sums come out infinite or zero, which is caught at the end)
          const unsigned long long scale2 = pack_f32(cexp, cexp), base2 = pack_f32(-base, -base);
          unsigned long long parts2[2] = {0ull, 0ull};  // two pairs of running sums
          float most = -INFINITY;
          uint32_t both[I8 ? 1 : 2][32];  // (beside the widening warps there are no registers for 64 scores)
          if (!I8) {
            tmem_ld32_issue(s_tmem, both[0]);
            tmem_ld32_issue(s_tmem + 32, both[I8 ? 0 : 1]);
          }
#pragma unroll
          for (int k = 0; k < 2; k++) {
            uint32_t (&s)[32] = both[I8 ? 0 : k];
            if (I8) tmem_ld32_issue(s_tmem + 32 * k, s);
            tmem_ld_wait32(s);
            hide(k, s);
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              unsigned long long ks[2] = {scale2, scale2}, vs[2];
              if (I8) {
                const float4 x = *reinterpret_cast<const float4*>(mt.k_scale + half * 64 + 32 * k + i), y = *reinterpret_cast<const float4*>(mt.v_scale + half * 64 + 32 * k + i);
                ks[0] = pack_f32(x.x, x.y); ks[1] = pack_f32(x.z, x.w);
                vs[0] = pack_f32(y.x, y.y); vs[1] = pack_f32(y.z, y.w);
              }
#pragma unroll
              for (int j = 0; j < 2; j++) {
                float x, y;
                unpack_f32(fma_f32x2(pack_f32(__uint_as_float(s[i + 2 * j]), __uint_as_float(s[i + 2 * j + 1])), ks[j], base2), x, y);
                most = max3(most, x, y);
                unsigned long long e = pack_f32(exp2_fast(x), exp2_fast(y));
                parts2[j] = add_f32x2(parts2[j], e);
                if (I8) e = mul_f32x2(e, vs[j]);
                unpack_f32(e, x, y);
                p[16 * k + (i >> 1) + j] = pack_bf16(x, y);
              }
            }
          }
          {
            float x, y;
            unpack_f32(add_f32x2(parts2[0], parts2[1]), x, y);
            part = x + y;
          }
          if (follow) break;
          // where a weight came out beyond 2^8 (or is a row's first) the pair of warps goes over the block again, with the maximum
          follow = pair_any(1 + (warp & 3), row < used && (most > 8.f || (m == -INFINITY && most > -INFINITY)));
          if (!follow) break;
        }
        sum += part;
        tmem_st32(s_tmem, p);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&c.p_ready[blocks & 1]));
      }
      // ---- the item's rows: finished, or left for whoever finishes the tile
      wait(c.o_done, items & 1, 309);
      tc_fence_after();
      c.top[0][half][row] = sum;
      named_sync(5, kSoftmaxThreads);
      const float l = c.top[0][0][row] + c.top[0][1][row];
      named_sync(5, kSoftmaxThreads);
      const bool mine = row < used;
      const int my_row = w.row0 + tok, my_head = w.head * group + row - tok * group;
      uint16_t* const dst = a.out + ((long long)my_row * a.n_q + my_head) * D;
      bool finite = true;
      const bool whole = n == w.blocks;
      float* to = nullptr;  // partial sums: [four columns][row][4] and (base, l) of every row, in one of this block's two places
      if (!whole) {
        const int first = work_owner(w.w0, work.total, work.parts), here = (int)blockIdx.x;
        to = a.partial + (long long)attn_part(here, here == first && work.begin < w.w0) * attn_part_floats(D, 128);
        if (mine && half == 0) *reinterpret_cast<float2*>(to + D * 128 + row * 2) = make_float2(m == -INFINITY ? m : base, l);
        if (tid == 0 && here == first) write_join(a, work, w, first, used);
      }
      // no weights (no key seen, or none with a score above -inf): not finite, and seen to behind
      const float inv = l > 0.f ? 1.f / l : __int_as_float(0x7fc00000);
      if (warp_used) {
#pragma unroll 1
        for (int i = 32 * half; i < D; i += 64) {
          uint32_t o[32];
          tmem_ld32_issue(o_tmem + lanes + i, o);
          tmem_ld_wait32(o);
          if (!mine) continue;
          if (!whole) {
#pragma unroll
            for (int j = 0; j < 8; j++)
              if (i + 4 * j < D) reinterpret_cast<uint4*>(to)[((i >> 2) + j) * 128 + row] = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
            continue;
          }
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            if (i + j >= D) continue;
            uint32_t p[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const float x = __uint_as_float(o[j + 2 * k]) * inv, y = __uint_as_float(o[j + 2 * k + 1]) * inv;
              finite = finite && fabsf(x) <= 3.0e38f && fabsf(y) <= 3.0e38f;
              p[k] = pack_bf16(x, y);
            }
            *reinterpret_cast<uint4*>(dst + i + j) = make_uint4(p[0], p[1], p[2], p[3]);
          }
        }
      }
      if (whole && mine && !finite) c.again = 1;
      tc_fence_before();
      named_sync(5, kSoftmaxThreads);  // everybody has read O and the exchange
      release_item(items);
    }
    // All other roles are through, so no wait's limit runs while this goes on; and what was asked for has been copied and multiplied, so the
    // room of queries and units is free.
    if (c.again && c.stop == 1) mend_tiles(a, c, *reinterpret_cast<TileScratch*>(base), tid);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    __syncwarp();
    if (*(volatile int*)&c.abort) {
      if (lane == 0) report_expired_wait(a.status, c.abort);
      __nanosleep(1000000);  // let what is in flight land after a failed wait
    }
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// A bf16 tensor [outer][heads][D], fetched in boxes of 64 dims by box_heads by box_outer.
bool encode_heads(CUtensorMap* map, const void* base, uint64_t outer, int heads, int D, int box_heads, int box_outer) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, outer};
  cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)heads * D * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_outer};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// The same as rows of one head, one to a box (what a gather of four takes).
bool encode_rows(CUtensorMap* map, const void* base, uint64_t rows, int D) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)D, rows};
  cuuint64_t strides[1] = {(cuuint64_t)D * 2};
  cuuint32_t box[2] = {64, 1};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DC, int UNITS, int AHEAD, bool I8>
cudaError_t run_tile(const AttnPagedArgs& a, cudaStream_t stream) {
  constexpr int smem = 1024 + (DC + UNITS) * kUnit + (I8 ? AHEAD * kUnit / 2 : 0) + kMetaBlocks * (int)sizeof(Meta) + (int)sizeof(Control);
  static_assert((DC + UNITS) * kUnit >= (int)sizeof(TileScratch), "room for rows that are computed once more");
  static_assert(smem <= 227 * 1024, "shared memory");
  static_assert(UNITS % DC == 0, "a block's units lie one behind another");
  static_assert((DC + UNITS) * kUnit >= (4096 + 1) * 4, "room for the sequences' first tiles");
  auto kernel = attn_paged_tile_kernel<DC, UNITS, AHEAD, I8>;
  static std::atomic<unsigned long long> attr_done;
  if (first_use_on_device(attr_done)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    mark_used_on_device(attr_done);
  }
  TileMaps m{};
  const uint64_t slots = (uint64_t)a.v.pages * a.v.page_size;
  const int group = a.n_q / a.v.n_kv, run = std::max(a.box_rows, 1);
  if (!encode_heads(&m.q, a.q, a.v.rows, a.n_q, a.v.D, group, a.tokens_per_tile)) return cudaErrorInvalidValue;
  if (!I8 && (!encode_heads(&m.k, a.k, slots, a.v.n_kv, a.v.D, 1, run) || !encode_heads(&m.v, a.vv, slots, a.v.n_kv, a.v.D, 1, run) ||
              !encode_rows(&m.k_rows, a.k, slots * a.v.n_kv, a.v.D) || !encode_rows(&m.v_rows, a.vv, slots * a.v.n_kv, a.v.D)))
    return cudaErrorInvalidValue;
  return launch_dependent(kernel, dim3(a.grid), dim3(kThreadsOf<I8>), smem, stream, a, m);
}

}  // namespace

cudaError_t launch_attn_paged_tile(AttnPagedArgs a, cudaStream_t stream) {
  a.box_rows = a.window && a.sinks ? kSpanAlign : 128;  // (with first tokens in front of the window's, keys lie one behind another in sixteens)
  while (a.box_rows > 4 && a.v.page_size % a.box_rows) a.box_rows /= 2;
  if (a.box_rows < 8) a.box_rows = 0;
  const int units = (a.v.D + 63) / 64;
  if (a.scales)
    return units == 1 ? run_tile<1, 8, 4, true>(a, stream) : units == 2 ? run_tile<2, 8, 4, true>(a, stream)
         : units == 3 ? run_tile<3, 6, 4, true>(a, stream) : run_tile<4, 8, 2, true>(a, stream);
  return units == 1 ? run_tile<1, 8, 1, false>(a, stream) : units == 2 ? run_tile<2, 8, 1, false>(a, stream)
       : units == 3 ? run_tile<3, 6, 1, false>(a, stream) : run_tile<4, 8, 1, false>(a, stream);
}

}  // namespace tb200
