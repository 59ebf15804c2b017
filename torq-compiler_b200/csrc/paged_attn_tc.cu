// Attention of many rows over a paged cache on the tensor cores (paged.cuh, paged.h: tiles and the sharing-out of their work).
//
// A tile is 128 rows: up to 128 / group tokens with the query heads of one key/value head. Per block of 128 keys: S = Q K^T into TMEM
// (fp32), softmax in registers against a running maximum, P as bf16 back into TMEM, O += P V with P as the TMEM operand. S is double
// buffered, so the product of the next block runs while this block's softmax does; O (up to 256 columns) and both S fill TMEM.
//   p = 2^((s - m) scale log2 e), sums in fp32; m is the row's maximum, but follows it only when it has grown by more than 2^8 in
//   p (O and the sum are scaled then): a bound serves as well as the maximum itself, and most blocks leave O alone.
// Warps: eight for softmax (two to a row quarter, half a row's keys each), four that copy, one that issues the matrix instructions.
// Copies gather: each key row's place comes from the page table, so any page size and any sequence end fits; a unit is 128 keys
// x 64 dims in the 128-byte swizzle, zeros where a key is seen by no row of the tile. Keys are the K-major operand, values the same
// bytes read as MN-major.  int8 caches are widened to bf16 (exact) on the way; the keys' scales meet the scores, the values' scales P.
// Work is shared out evenly: all tiles' key blocks in one row, every block of the grid takes an equal piece. A tile that falls to
// several leaves partial sums in memory, which the last one to arrive adds up in their order (results do not depend on who that is).
#include <algorithm>

#include "dependent_launch.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "paged_row.cuh"
#include "tcgen05_ptx.cuh"
#include "tensor_map.h"

namespace tb200 {

namespace {

// four warpgroups: two for softmax, one that widens int8 caches, one with a warp each for matrix instructions, items and the copy engine; the
// registers go where they are needed (of the 512 x 128 that a block starts with)
constexpr int kSoftmaxWarps = 8, kCopyWarps = 4, kThreads = 512;
constexpr int kCopyRegs = 104, kIssueRegs = 56;
constexpr int kSoftmaxRegsI8 = 176, kSoftmaxRegs = 200;  // a bf16 cache's copies leave more
static_assert(256 * kSoftmaxRegsI8 + 128 * kCopyRegs + 128 * kIssueRegs <= kThreads * 128, "register split, int8");
static_assert(256 * kSoftmaxRegs + 256 * kIssueRegs <= kThreads * 128, "register split, bf16");
constexpr int kCopyThreads = kCopyWarps * 32, kSoftmaxThreads = kSoftmaxWarps * 32;
constexpr int kUnit = 128 * 128;  // bytes of 128 rows of 64 bf16 values
constexpr int kMetaBlocks = 8, kItems = 4;
static_assert(kSoftmaxThreads == kRowThreads, "the plain row is computed by the softmax warps");

struct alignas(16) Meta {
  float k_scale[kKeyBlock], v_scale[kKeyBlock];
  uint32_t holds[4];  // a bit for each key of the block: it is seen by a row of the tile, and its page holds something
  int key0;
};
static_assert(sizeof(Meta) % 16 == 0 && sizeof(RowScratch) % 16 == 0, "what lies behind them in shared memory is read 16 and 8 bytes at a time");
// A piece of work of a block of the grid: key blocks b0 .. b1 - 1 of a tile of one key/value head.
struct Item {
  int seq, head, index;     // index: of the tile among all tiles
  int row0, tokens;         // the tile's rows of the chunk; tokens 0: there is no more work
  int first_pos;            // position of the first token
  int near_key, end_key, sink_blocks, near_block, blocks;  // tile_span
  int b0, b1;
  long long w0;             // where the tile's work begins
};
struct Control {
  uint64_t full[16], empty[16], s_full[2], p_ready[2], pv_done, o_done, q_full, q_empty, item_full[kItems], item_empty[kItems];
  Item items[kItems];
  uint32_t tmem, bad_rows[4], arrived;
  int abort, stop;
  float top[2][2][128];  // row maxima of the two halves, by parity of the block
  long long totals[kThreads / 32];
  int start_seq, start_tile, start_index, start_off;
};

// what a sequence brings
struct Span {
  int row0, n, ctx;
};
__device__ __forceinline__ Span span_of(const AttnPagedArgs& a, int s) {
  Span r;
  r.row0 = max(a.v.row_start[s], 0);
  r.n = max(0, min(a.v.row_start[s + 1], a.v.rows) - r.row0);
  if (a.max_new) r.n = min(r.n, a.max_new);
  r.ctx = max(a.v.context[s], 0);
  return r;
}
__device__ __forceinline__ int tiles_of(const AttnPagedArgs& a, const Span& s) {
  return s.n * (a.n_q / a.v.n_kv) > a.few_rows ? (s.n + a.tokens_per_tile - 1) / a.tokens_per_tile : 0;
}

// The keys of an item, and where the cache holds them. Page ids are asked for a block ahead of their use, without a branch (a branch would wait
// for each); slots have 32 bits (the planner refuses more), -1 where no token of the tile sees the key or nothing is held.
struct Keys {
  const int32_t* pages_of;
  int near_key, end_key, sinks, sink_blocks, near_block, last, pages, page_size;
  PageDivisor div;
  __device__ __forceinline__ Keys(const AttnPagedArgs& a, const Item& w)
      : pages_of(a.v.table + (long long)w.seq * a.v.max_pages), near_key(w.near_key), end_key(w.end_key), sinks(a.sinks), sink_blocks(w.sink_blocks),
        near_block(w.near_block), last(a.v.capacity - 1), pages(a.v.pages), page_size(a.v.page_size), div(a.v.div) {}
  __device__ __forceinline__ int first(int b) const { return (b < sink_blocks ? b : near_block + (b - sink_blocks)) * kKeyBlock; }
  __device__ __forceinline__ int ask(int key) const {
    int page;  // volatile: it is to be on its way now, not when it is used
    asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(page) : "l"(pages_of + page_of(min(key, last), div)));
    return page;
  }
  __device__ __forceinline__ bool seen(int key) const { return key < end_key && (key >= near_key || key < sinks); }  // by a token of the tile
  __device__ __forceinline__ int count_seen(int key, int n) const {  // of keys key .. key + n - 1
    const int upto = min(key + n, end_key), firsts = max(0, min(min(upto, sinks), near_key) - key);
    return firsts + max(0, upto - max(key, near_key));
  }
  __device__ __forceinline__ int slot(int key, int page) const {
    const bool there = seen(key) && page >= 0 && page < pages;
    return there ? page * page_size + (key - page_of(key, div) * page_size) : -1;
  }
};

// Running sum over the block's threads up to and including this one, and the sum of all, through c.totals.
__device__ long long block_scan(Control& c, long long x, long long& all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) c.totals[warp] = v;
  __syncthreads();
  long long before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; w++) {
    const long long y = c.totals[w];
    before += w < warp ? y : 0;
    all += y;
  }
  return before + v;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
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
// four int8 -> four bf16, exact: 0x4300 | low seven bits of the biased byte is 128 + those bits, and 128 or 256 comes off again
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u, low = u & 0x7f7f7f7fu, off = ~u & 0x80808080u;
  const uint32_t a0 = __byte_perm(low, 0x43434343u, 0x4140), a1 = __byte_perm(low, 0x43434343u, 0x4342);
  const uint32_t c0 = __byte_perm(off, 0x43434343u, 0x4140), c1 = __byte_perm(off, 0x43434343u, 0x4342);
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"(a0), "r"(c0));
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(a1), "r"(c1));
}
__device__ __forceinline__ void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void sts128(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// How the copy engine sees the queries and a bf16 cache: boxes of 64 dims by the rows of a tile / by box_rows keys, and single keys.
struct TileMaps {
  CUtensorMap q, k, v, k_rows, v_rows;
};

// DC: units (64 dims) of a head. UNITS: ring of keys' and values' units in shared memory.
template <int DC, int UNITS, bool I8>
__global__ void __launch_bounds__(kThreads, 1) attn_paged_tile_kernel(const AttnPagedArgs a, const __grid_constant__ TileMaps maps) {
  extern __shared__ unsigned char smem_raw[];
  // [Q units][ring units] on 1024-byte boundaries, then the rest
  unsigned char* const base = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t q_smem = smem_u32(base), ring = q_smem + DC * kUnit;
  Meta* const meta = reinterpret_cast<Meta*>(base + (DC + UNITS) * kUnit);
  RowScratch& plain = *reinterpret_cast<RowScratch*>(meta + kMetaBlocks);
  Control& c = *reinterpret_cast<Control*>(reinterpret_cast<unsigned char*>(&plain) + sizeof(RowScratch));
  int* const first_tile = reinterpret_cast<int*>(base);  // while the work is shared out: tiles in front of each sequence

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PagedView& v = a.v;
  const int group = a.n_q / v.n_kv, D = v.D, tpt = a.tokens_per_tile;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&c.tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 32) {
    for (int i = 0; i < UNITS; i++) {
      mbar_init(smem_u32(&c.full[i]), I8 ? kCopyThreads : 1);
      mbar_init(smem_u32(&c.empty[i]), 1);
    }
    for (int i = 0; i < 2; i++) {  // a softmax warp may be one block ahead of another: a barrier for each buffer
      mbar_init(smem_u32(&c.s_full[i]), 1);
      mbar_init(smem_u32(&c.p_ready[i]), kSoftmaxThreads);
    }
    mbar_init(smem_u32(&c.pv_done), 1);
    mbar_init(smem_u32(&c.o_done), 1);
    for (int i = 0; i < kItems; i++) {
      mbar_init(smem_u32(&c.item_full[i]), 1);
      mbar_init(smem_u32(&c.item_empty[i]), kSoftmaxThreads + 64 + (I8 ? kCopyThreads : 0));
    }
    mbar_init(smem_u32(&c.q_full), 1);
    mbar_init(smem_u32(&c.q_empty), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    c.abort = 0;
    c.bad_rows[0] = c.bad_rows[1] = c.bad_rows[2] = c.bad_rows[3] = 0;
  }
  grid_dependency_wait();
  grid_dependency_release();

  // ---- the work: tiles of the sequences, key blocks of the tiles ----
  long long all = 0;
  int run = 0;
  for (int s0 = 0; s0 < v.S; s0 += kThreads) {
    const int s = s0 + tid;
    const int upto = run + (int)block_scan(c, s < v.S ? tiles_of(a, span_of(a, s)) : 0, all);
    if (s < v.S) first_tile[s + 1] = upto;
    run += (int)all;
  }
  if (tid == 0) first_tile[0] = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = c.tmem;
  const int n_tiles = min(run, a.max_tiles);
  auto blocks_of = [&](int i, int& seq, int& tile) {
    int lo = 0, hi = v.S - 1;  // the last sequence with first_tile[seq] <= i
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first_tile[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    seq = lo;
    tile = i - first_tile[lo];
    const Span sp = span_of(a, seq);
    return tile_span(sp.ctx, sp.n, tile, tpt, a.window, a.sinks, v.capacity).blocks;
  };
  int seq0 = 0, tile0 = 0, n0 = tid < n_tiles ? blocks_of(tid, seq0, tile0) : 0;
  long long upto0 = block_scan(c, n0, all), per_head = all;
  if (n_tiles > kThreads) {
    long long mine = 0;
    for (int i = tid + kThreads; i < n_tiles; i += kThreads) mine += blocks_of(i, seq0, tile0);
    block_scan(c, mine, all);
    per_head += all;
  }
  const long long total = per_head * v.n_kv;
  const int parts = (int)max(1ll, min((long long)gridDim.x, total / kTileMinBlocks));
  const bool works = total > 0 && (int)blockIdx.x < parts;
  const long long begin = works ? work_begin(total, blockIdx.x, parts) : 0, end = works ? work_begin(total, blockIdx.x + 1, parts) : 0;
  if (works) {
    const long long rem = begin % per_head;
    long long before = 0;
    for (int i0 = 0; i0 < n_tiles && before <= rem; i0 += kThreads) {
      const int i = i0 + tid;
      if (n_tiles > kThreads) {
        n0 = i < n_tiles ? blocks_of(i, seq0, tile0) : 0;
        upto0 = block_scan(c, n0, all);
      }
      const long long upto = before + upto0;
      if (n0 && upto > rem && upto - n0 <= rem) {
        c.start_tile = tile0;
        c.start_seq = seq0;
        c.start_index = i;
        c.start_off = (int)(rem - (upto - n0));
      }
      before += n_tiles > kThreads ? all : per_head;
    }
  }
  __syncthreads();  // the start is known, and first_tile's room is free

  bool gave_up = false;
  auto wait = [&](uint64_t& bar, uint32_t parity, int code) {
    // one wait that ran out ends all others at once: every role then runs through without waiting, and the results are not used
    if (gave_up) return;
    const uint32_t at = smem_u32(&bar);
    if (mbar_poll(at, parity, 256)) return;
    const unsigned long long t0 = globaltimer_ns();
    for (;;) {
      if (mbar_poll(at, parity, 256)) return;
      if (*(volatile int*)&c.abort) break;
      if (globaltimer_ns() - t0 > a.wait_ns) {
        report_expired_wait(a.status, code);
        *(volatile int*)&c.abort = 1;
        break;
      }
    }
    gave_up = true;
  };

  // The roles take the block's items from a ring that a warp of its own fills. The reference stays valid until release_item.
  auto take_item = [&](uint32_t i) -> const Item& {
    wait(c.item_full[i % kItems], (i / kItems) & 1, 310);
    return c.items[i % kItems];
  };
  auto release_item = [&](uint32_t i) { mbar_arrive(smem_u32(&c.item_empty[i % kItems])); };
  const uint32_t o_tmem = tmem + 256;
  if (warp >= kSoftmaxWarps && warp < kSoftmaxWarps + kCopyWarps) {
    // ------------------------------------------------ copies of int8 caches: widened on the way
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(I8 ? kCopyRegs : kIssueRegs));
    if (I8 && works) {
    const int t = tid - kSoftmaxThreads;
    uint32_t unit = 0, blocks = 0;
    constexpr int kRows = 4, kPieces = 4, kRowStep = kCopyThreads / kPieces;  // pieces of 16 bytes: a thread has the same one of four rows
    const int piece = t % kPieces, row0 = t / kPieces;
    const long long row_bytes = (long long)v.n_kv * D;
    for (uint32_t items = 0;; items++) {
      const Item& w = take_item(items);
      if (__any_sync(0xffffffffu, gave_up || !w.tokens)) break;
      const int b0 = w.b0, b1 = w.b1, head = w.head;
      const Keys keys_of(a, w);
      release_item(items);
      int next_page[kRows], next_own;
      auto ask_block = [&](int b) {
        const int key0 = keys_of.first(b);
#pragma unroll
        for (int i = 0; i < kRows; i++) next_page[i] = keys_of.ask(key0 + row0 + kRowStep * i);
        next_own = keys_of.ask(key0 + t);
      };
      // where this thread's pieces of the keys and of the values of a block start, in bytes behind the cache; negative: zeros
      long long key_at[kRows], val_at[kRows];
      int own = 0;
      float own_k = 0.f, own_v = 0.f;
      auto turn = [&](int b) {  // the block that was asked for becomes the one to copy
        const int key0 = keys_of.first(b);
#pragma unroll
        for (int i = 0; i < kRows; i++) {
          const int slot = keys_of.slot(key0 + row0 + kRowStep * i, next_page[i]);
          val_at[i] = key_at[i];
          key_at[i] = slot < 0 ? -1 : slot * row_bytes + ((long long)head * D + piece * 16);
        }
        own = keys_of.slot(key0 + t, next_own);
        const float* sc = a.scales + (long long)max(own, 0) * 2 * v.n_kv + head;
        asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(own_k) : "l"(sc));
        asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(own_v) : "l"(sc + v.n_kv));
      };
      // groups of up to two units go through registers, the next group asked for before one is widened
      constexpr int G = DC > 1 ? 2 : 1;
      uint4 x[G][kRows], y[G][kRows];
      auto load = [&](uint4 (&to)[G][kRows], const void* pages, const long long (&at)[kRows], int u0) {
#pragma unroll
        for (int g = 0; g < G; g++) {
          if (u0 + g >= DC) continue;
          const bool in = u0 + g + 1 < DC || (u0 + g) * 64 + piece * 16 < D;
#pragma unroll
          for (int i = 0; i < kRows; i++) {
            to[g][i] = make_uint4(0, 0, 0, 0);
            if (in && at[i] >= 0)
              asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(to[g][i].x), "=r"(to[g][i].y), "=r"(to[g][i].z), "=r"(to[g][i].w)
                           : "l"((const char*)pages + at[i] + (u0 + g) * 64));
          }
        }
      };
      auto store = [&](const uint4 (&from)[G][kRows], int u0) {
#pragma unroll
        for (int g = 0; g < G; g++) {
          if (u0 + g >= DC) continue;
          if (unit >= UNITS) wait(c.empty[unit % UNITS], (unit / UNITS - 1) & 1, 301);
          const uint32_t dst = ring + (unit % UNITS) * kUnit;
#pragma unroll
          for (int i = 0; i < kRows; i++) {
            const int r = row0 + kRowStep * i;
            const uint4 q = from[g][i];
            uint4 lo, hi;
            widen4(q.x, lo.x, lo.y); widen4(q.y, lo.z, lo.w);
            widen4(q.z, hi.x, hi.y); widen4(q.w, hi.z, hi.w);
            sts128(dst + r * 128 + (((2 * piece) ^ (r & 7)) << 4), lo);
            sts128(dst + r * 128 + (((2 * piece + 1) ^ (r & 7)) << 4), hi);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          mbar_arrive(smem_u32(&c.full[unit % UNITS]));
          unit++;
        }
      };
      ask_block(b0);
      turn(b0);
      load(x, a.k, key_at, 0);
      for (int b = b0; b <= b1; b++) {
        const bool keys = b < b1, values = b > b0, more = b + 1 < b1;
        if (more) ask_block(b + 1);
        if (keys) {  // what this block's keys are, by one thread a key
          Meta& m = meta[blocks % kMetaBlocks];
          blocks++;
          const uint32_t bits = __ballot_sync(0xffffffffu, own >= 0);
          if (lane == 0) m.holds[t >> 5] = bits;
          if (t == 0) m.key0 = keys_of.first(b);
          m.k_scale[t] = own >= 0 ? own_k : 0.f;
          m.v_scale[t] = own >= 0 ? own_v : 0.f;
        }
        if (DC <= 2) {
          if (values) load(y, a.vv, val_at, 0);
          if (keys) {
            store(x, 0);
            turn(more ? b + 1 : b);
          }
          if (more) load(x, a.k, key_at, 0);
          if (values) store(y, 0);
        } else {
          if (keys) {
            load(y, a.k, key_at, 2);
            store(x, 0);
          }
          if (values) load(x, a.vv, val_at, 0);
          if (keys) store(y, 2);
          if (values) {
            load(y, a.vv, val_at, 2);
            store(x, 0);
          }
          if (keys) turn(more ? b + 1 : b);
          if (more) load(x, a.k, key_at, 0);
          if (values) store(y, 2);
        }
      }
    }
    }
  } else if (warp >= kSoftmaxWarps + kCopyWarps) {
    // ------------------------------------------------ matrix instructions
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (works && warp == kSoftmaxWarps + kCopyWarps) {
    const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);  // 8-row groups 1024 bytes apart, sm_100 descriptor, 128-byte swizzle
    const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kKeyBlock >> 3) << 17) | (8u << 24);
    uint32_t unit = 0, blocks = 0;
    auto lo_of = [](uint32_t at) { return ((at & 0x3FFFF) >> 4) | (64u << 16); };
    for (uint32_t items = 0;; items++) {
      const Item& w = take_item(items);
      const int n = w.b1 - w.b0;
      if (__any_sync(0xffffffffu, gave_up || !w.tokens)) break;
      release_item(items);
      wait(c.q_full, items & 1, 303);
      for (int b = 0; b <= n; b++) {
        if (b < n) {  // scores of block b
          const uint32_t s_tmem = tmem + ((blocks + b) & 1) * 128;
#pragma unroll
          for (int u = 0; u < DC; u++) {
            wait(c.full[unit % UNITS], (unit / UNITS) & 1, 304);
            tc_fence_after();
            const uint32_t qa = lo_of(q_smem + u * kUnit), kb = lo_of(ring + (unit % UNITS) * kUnit);
            const int steps = min(4, (D - u * 64) >> 4);
            for (int k = 0; k < steps; k++) mma_f16_elect(s_tmem, qa + 2 * k, hi, kb + 2 * k, hi, idesc_s, (u | k) ? 1u : 0u);
            mma_commit_elect(smem_u32(&c.empty[unit % UNITS]));
            unit++;
          }
          mma_commit_elect(smem_u32(&c.s_full[(blocks + b) & 1]));
          if (b == n - 1) mma_commit_elect(smem_u32(&c.q_empty));
        }
        if (b > 0) {  // sums of block b - 1
          const uint32_t g = blocks + b - 1, p_tmem = tmem + (g & 1) * 128;
          wait(c.p_ready[g & 1], (g >> 1) & 1, 305);
          tc_fence_after();
#pragma unroll
          for (int u = 0; u < DC; u++) {
            wait(c.full[unit % UNITS], (unit / UNITS) & 1, 306);
            tc_fence_after();
            const int width = min(64, D - u * 64);
            const uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(width >> 3) << 17) | (8u << 24);
            const uint32_t vb = lo_of(ring + (unit % UNITS) * kUnit);
#pragma unroll
            for (int k = 0; k < 8; k++)  // keys 0..63 of P lie in columns 0..31, keys 64..127 in columns 64..95
              mma_f16_ts_elect(o_tmem + u * 64, p_tmem + (k < 4 ? k * 8 : 64 + (k - 4) * 8), vb + k * (2048 >> 4), hi, idesc_o, (b > 1 || k > 0) ? 1u : 0u);
            mma_commit_elect(smem_u32(&c.empty[unit % UNITS]));
            unit++;
          }
          mma_commit_elect(smem_u32(&c.pv_done));
          if (b == n) mma_commit_elect(smem_u32(&c.o_done));
        }
      }
      blocks += n;
    }
    } else if (works && warp == kSoftmaxWarps + kCopyWarps + 2) {
      // ---------------------------------------------- queries, and bf16 caches, by the copy engine: a lane asks for four rows of 128 bytes at once
      uint32_t unit = 0, blocks = 0;
      for (uint32_t items = 0;; items++) {
        const Item& w = take_item(items);
        if (__any_sync(0xffffffffu, gave_up || !w.tokens)) break;
        const int b0 = w.b0, b1 = w.b1, head = w.head, q_row = w.row0;
        const Keys keys_of(a, w);
        release_item(items);
        if (items) wait(c.q_empty, (items - 1) & 1, 302);
        __syncwarp();
        if (lane == 0) {  // rows of the tile's tokens, in the tile's order; those behind the last token are somebody's or nobody's, and are not used
          const uint32_t bar = smem_u32(&c.q_full);
          mbar_expect_tx(bar, DC * 128 * tpt * group);
          for (int u = 0; u < DC; u++) tma_load_3d(q_smem + u * kUnit, &maps.q, u * 64, head * group, q_row, bar);
        }
        if (I8) continue;
        auto begin_unit = [&]() {
          const uint32_t slot = unit % UNITS;
          if (unit >= UNITS) wait(c.empty[slot], (unit / UNITS - 1) & 1, 301);
          __syncwarp();
          if (lane == 0) mbar_expect_tx(smem_u32(&c.full[slot]), kUnit);
          __syncwarp();
          unit++;
          return slot;
        };
        auto tell = [&](int key0, uint32_t held) {  // the block's keys, before its first unit
          Meta& m = meta[blocks % kMetaBlocks];
          blocks++;
          if ((lane & 7) == 0) m.holds[lane >> 3] = held;
          if (lane == 0) m.key0 = key0;
          __syncwarp();
        };
        auto gather_bits = [&](uint32_t nibble) {  // four keys a lane -> the 32 of its eight lanes
          uint32_t held = nibble << (4 * (lane & 7));
          held |= __shfl_xor_sync(0xffffffffu, held, 1);
          held |= __shfl_xor_sync(0xffffffffu, held, 2);
          return held | __shfl_xor_sync(0xffffffffu, held, 4);
        };
        // four keys to a lane: where pages end anywhere, and for runs of keys that are seen in part
        auto gather = [&](const CUtensorMap* map, uint32_t slot, int u, int first, const int (&r)[4]) {
          tma_gather4(ring + slot * kUnit + first * 128, map, u * 64, r[0], r[1], r[2], r[3], smem_u32(&c.full[slot]));
        };
        if (!a.box_rows) {
          int next_page[4], key_row[4], val_row[4] = {};
          auto ask_block = [&](int b) {
#pragma unroll
            for (int i = 0; i < 4; i++) next_page[i] = keys_of.ask(keys_of.first(b) + 4 * lane + i);
          };
          ask_block(b0);
          for (int b = b0; b <= b1; b++) {
            if (b < b1) {
              const int key0 = keys_of.first(b);
              uint32_t nibble = 0;
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const int slot = keys_of.slot(key0 + 4 * lane + i, next_page[i]);
                key_row[i] = slot < 0 ? -1 : slot * v.n_kv + head;
                nibble |= (slot >= 0 ? 1u : 0u) << i;
              }
              if (b + 1 < b1) ask_block(b + 1);
              tell(key0, gather_bits(nibble));
              for (int u = 0; u < DC; u++) gather(&maps.k_rows, begin_unit(), u, 4 * lane, key_row);
            }
            if (b > b0)
              for (int u = 0; u < DC; u++) gather(&maps.v_rows, begin_unit(), u, 4 * lane, val_row);
#pragma unroll
            for (int i = 0; i < 4; i++) val_row[i] = key_row[i];
          }
        } else {
          // a run of box_rows keys to a lane: one box where all are seen (or none: from outside the cache, zeros), else four by four
          const int R = a.box_rows, runs = kKeyBlock / R, none = v.pages * v.page_size;
          int next_page, key_run = 0, val_run = 0;  // slot of a run's first key, or `none`
          uint32_t key_parts = 0, val_parts = 0;    // runs that are seen in part
          int key_first = 0, val_first = 0;
          auto copy_units = [&](const CUtensorMap* map, const CUtensorMap* rows, int run, uint32_t parts, int key0) {
            for (int u = 0; u < DC; u++) {
              const uint32_t slot = begin_unit();
              if (lane < runs && !(parts >> lane & 1)) tma_load_3d(ring + slot * kUnit + lane * R * 128, map, u * 64, head, run, smem_u32(&c.full[slot]));
              for (uint32_t left = parts; left; left &= left - 1) {
                const int g = __ffs(left) - 1, from = __shfl_sync(0xffffffffu, run, g);
                if (4 * lane < R) {
                  int r[4];
#pragma unroll
                  for (int i = 0; i < 4; i++) r[i] = keys_of.seen(key0 + g * R + 4 * lane + i) ? (from + 4 * lane + i) * v.n_kv + head : -1;
                  gather(rows, slot, u, g * R + 4 * lane, r);
                }
              }
            }
          };
          auto ask_block = [&](int b) { next_page = keys_of.ask(min(keys_of.first(b) + lane * R, keys_of.last)); };
          ask_block(b0);
          for (int b = b0; b <= b1; b++) {
            if (b < b1) {
              const int key0 = key_first = keys_of.first(b), mine = key0 + min(lane, runs - 1) * R;
              // the run of this lane, then the four keys of this lane
              const bool held = next_page >= 0 && next_page < v.pages && mine <= keys_of.last;
              const int seen = held ? keys_of.count_seen(mine, R) : 0;
              key_run = seen ? next_page * v.page_size + (mine - page_of(mine, v.div) * v.page_size) : none;
              key_parts = __ballot_sync(0xffffffffu, lane < runs && seen > 0 && seen < R);
              const uint32_t any = __ballot_sync(0xffffffffu, seen > 0);
              if (b + 1 < b1) ask_block(b + 1);
              uint32_t nibble = 0;
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const int k = 4 * lane + i;
                nibble |= ((any >> (k / R) & 1) && keys_of.seen(key0 + k) ? 1u : 0u) << i;
              }
              tell(key0, gather_bits(nibble));
              copy_units(&maps.k, &maps.k_rows, key_run, key_parts, key0);
            }
            if (b > b0) copy_units(&maps.v, &maps.v_rows, val_run, val_parts, val_first);
            val_run = key_run;
            val_parts = key_parts;
            val_first = key_first;
          }
        }
      }
    } else if (works && warp == kSoftmaxWarps + kCopyWarps + 1 && lane == 0) {
      // ---------------------------------------------- the block's items
      long long cur = begin;
      int head = (int)(begin / per_head), seq = c.start_seq, tile = c.start_tile, index = c.start_index, off = c.start_off;
      Span span = span_of(a, seq);
      int tiles = tiles_of(a, span);
      for (uint32_t i = 0;; i++) {
        if (i >= kItems) wait(c.item_empty[i % kItems], (i / kItems - 1) & 1, 311);
        if (gave_up) break;
        Item& w = c.items[i % kItems];
        if (cur >= end) {
          w.tokens = 0;
          mbar_arrive(smem_u32(&c.item_full[i % kItems]));
          break;
        }
        const TileSpan ts = tile_span(span.ctx, span.n, tile, tpt, a.window, a.sinks, v.capacity);
        const int b1 = (int)min((long long)ts.blocks, off + (end - cur));
        w.seq = seq; w.head = head; w.index = index;
        w.row0 = span.row0 + tile * tpt;
        w.tokens = min(tpt, span.n - tile * tpt);
        w.first_pos = (int)min((long long)span.ctx + tile * tpt, 0x7fffffffll);
        w.near_key = ts.near_key; w.end_key = ts.end_key; w.sink_blocks = ts.sink_blocks; w.near_block = ts.near_block; w.blocks = ts.blocks;
        w.b0 = off; w.b1 = b1;
        w.w0 = cur - off;
        mbar_arrive(smem_u32(&c.item_full[i % kItems]));
        cur += b1 - off;
        if (cur >= end) continue;
        off = 0;
        tile++;
        if (++index >= n_tiles) {  // the next head begins
          index = 0;
          head++;
          seq = -1;
          tile = tiles;
        }
        if (tile >= tiles) {
          tile = 0;
          do {
            if (++seq >= v.S) seq = 0;  // there is a tile, so a sequence with one
            span = span_of(a, seq);
            tiles = tiles_of(a, span);
          } while (!tiles);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(I8 ? kSoftmaxRegsI8 : kSoftmaxRegs));
    if (works) {
    // ------------------------------------------------ softmax: thread = (row, half of the block's keys)
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int tok = page_of(row, a.group_div), pieces = D >> 4;
    const float cexp = a.scale * 1.4426950408889634f;
    uint32_t blocks = 0, items = 0;
    for (;; items++) {
      if (tid == 0) {  // one decides for all, who meet at barriers from here on
        const Item& w = take_item(items);
        c.stop = gave_up || *(volatile int*)&c.abort || !w.tokens;
      }
      named_sync(5, kSoftmaxThreads);
      if (c.stop) break;
      const Item& w = c.items[items % kItems];
      const int tokens = w.tokens, used = tokens * group, n = w.b1 - w.b0, first_pos = w.first_pos;
      const bool warp_used = (warp & 3) * 32 < used;
      const int pos = (int)min((long long)first_pos + min(tok, tokens - 1), 0x7fffffffll);
      const int last_pos = (int)min((long long)first_pos + tokens - 1, 0x7fffffffll);
      const int near = a.window ? max(0, pos - a.window + 1) : 0;  // this row sees keys [near, pos] and those in front of sinks
      float m = -INFINITY, base = 0.f, sum = 0.f;  // base: m scaled, what the exponents are taken from
      for (int b = 0; b < n; b++, blocks++) {
        const uint32_t s_tmem = tmem + lanes + (blocks & 1) * 128 + half * 64;
        if (!warp_used) {  // rows of nobody: P keeps what it holds, and so does O
          wait(c.s_full[blocks & 1], (blocks >> 1) & 1, 307);
          mbar_arrive(smem_u32(&c.p_ready[blocks & 1]));
          continue;
        }
        wait(c.s_full[blocks & 1], (blocks >> 1) & 1, 307);
        tc_fence_after();
        uint32_t s0[32], s1[32];
        tmem_ld32_issue(s_tmem, s0);
        tmem_ld32_issue(s_tmem + 32, s1);
        const Meta& mt = meta[blocks % kMetaBlocks];
        const int key0 = mt.key0 + half * 64;
        const uint32_t holds0 = mt.holds[half * 2], holds1 = mt.holds[half * 2 + 1];
        const bool partial = (holds0 & holds1) != 0xffffffffu || key0 + 63 > first_pos ||
                             (a.window && key0 < max(0, last_pos - a.window + 1) && key0 + 63 >= a.sinks);
        tmem_ld_wait32(s0);
        tmem_ld_wait32(s1);
        if (I8) {
          auto scaled = [&](uint32_t (&s)[32], const float* k_scale) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 x = *reinterpret_cast<const float4*>(k_scale + i);
              float f[4];
              unpack_f32(mul_f32x2(pack_f32(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), pack_f32(x.x, x.y)), f[0], f[1]);
              unpack_f32(mul_f32x2(pack_f32(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])), pack_f32(x.z, x.w)), f[2], f[3]);
#pragma unroll
              for (int j = 0; j < 4; j++) s[i + j] = __float_as_uint(f[j]);
            }
          };
          scaled(s0, mt.k_scale + half * 64);
          scaled(s1, mt.k_scale + half * 64 + 32);
        }
        if (partial) {
          // bits of the keys this row sees: not behind its position, inside the window or among the first, and held
          auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
          const uint32_t see0 = below(pos - key0 + 1) & (~below(near - key0) | below(a.sinks - key0)) & holds0;
          const uint32_t see1 = below(pos - key0 - 31) & (~below(near - key0 - 32) | below(a.sinks - key0 - 32)) & holds1;
          const uint32_t none = __float_as_uint(-INFINITY);
#pragma unroll
          for (int i = 0; i < 32; i++) {
            s0[i] = see0 >> i & 1 ? s0[i] : none;
            s1[i] = see1 >> i & 1 ? s1[i] : none;
          }
        }
        float tops[4] = {__uint_as_float(s0[0]), __uint_as_float(s0[1]), __uint_as_float(s1[0]), __uint_as_float(s1[1])};
#pragma unroll
        for (int i = 2; i < 32; i += 2) {
          tops[i >> 1 & 1] = max3(tops[i >> 1 & 1], __uint_as_float(s0[i]), __uint_as_float(s0[i + 1]));
          tops[2 + (i >> 1 & 1)] = max3(tops[2 + (i >> 1 & 1)], __uint_as_float(s1[i]), __uint_as_float(s1[i + 1]));
        }
        float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]);
        c.top[blocks & 1][half][row] = top;
        named_sync(1 + (warp & 3), 64);
        top = fmaxf(top, c.top[blocks & 1][half ^ 1][row]);
        // follow the maximum when p could grow beyond 2^8, or when there was none yet
        const bool grows = row < used && top > m && !((top - m) * cexp <= 8.f);
        if (b == 0) {
          m = top;
          base = m == -INFINITY ? 0.f : m * cexp;
        } else if (__any_sync(0xffffffffu, grows)) {
          float keep = 1.f;
          if (grows) {
            const float to = top * cexp;
            keep = m == -INFINITY ? 0.f : exp2_fast(base - to);
            m = top;
            base = to;
          }
          sum *= keep;
          // these scores were issued behind the sums of the block before the last: its phase is over, the last one's is waited for
          wait(c.pv_done, (blocks - 1) & 1, 308);
          tc_fence_after();
          for (int i = half; i < pieces; i += 2) {
            uint32_t o[16];
            tmem_ld16(o_tmem + lanes + i * 16, o);
#pragma unroll
            for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
            tmem_st16(o_tmem + lanes + i * 16, o);
          }
          tmem_st_wait();
        }
        // p = 2^(s c - base) in one multiply-add: how base was rounded is the same for every key of the row, so it cancels (where that factor
        // itself leaves fp32, at scores beyond 10^9, sums come out infinite or zero, which is caught at the end)
        const unsigned long long scale2 = pack_f32(cexp, cexp), base2 = pack_f32(-base, -base);
        unsigned long long parts2[2] = {0ull, 0ull};  // two pairs of running sums
        auto weights = [&](const uint32_t (&s)[32], const float* v_scale, uint32_t to) {
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x, y;
            unpack_f32(fma_f32x2(pack_f32(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), scale2, base2), x, y);
            unsigned long long e = pack_f32(exp2_fast(x), exp2_fast(y));
            parts2[i >> 1 & 1] = add_f32x2(parts2[i >> 1 & 1], e);
            if (I8) {
              const float2 vs = *reinterpret_cast<const float2*>(v_scale + i);
              e = mul_f32x2(e, pack_f32(vs.x, vs.y));
            }
            unpack_f32(e, x, y);
            p[i >> 1] = pack_bf16(x, y);
          }
          tmem_st16(to, p);
        };
        weights(s0, mt.v_scale + half * 64, s_tmem);
        weights(s1, mt.v_scale + half * 64 + 32, s_tmem + 16);
        {
          float x, y;
          unpack_f32(add_f32x2(parts2[0], parts2[1]), x, y);
          sum += x + y;
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(smem_u32(&c.p_ready[blocks & 1]));
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
      bool finite = l != 0.f || m == -INFINITY;  // sums of a row are fit to be used
      auto store = [&](uint16_t* at, const float (&o)[16], float inv) {
        uint32_t p[8];
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const float x = o[j] * inv, y = o[j + 1] * inv;
          finite = finite && fabsf(x) <= 3.0e38f && fabsf(y) <= 3.0e38f;
          p[j >> 1] = pack_bf16(x, y);
        }
        uint4* to = reinterpret_cast<uint4*>(at);
        to[0] = make_uint4(p[0], p[1], p[2], p[3]);
        to[1] = make_uint4(p[4], p[5], p[6], p[7]);
      };
      bool done = true;
      if (n == w.blocks) {
        if (warp_used) {
          const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
          for (int i = half; i < pieces; i += 2) {
            uint32_t o[16];
            tmem_ld16(o_tmem + lanes + i * 16, o);
            float f[16];
#pragma unroll
            for (int j = 0; j < 16; j++) f[j] = l == 0.f ? 0.f : __uint_as_float(o[j]);
            if (mine) store(dst + i * 16, f, inv);
          }
        }
      } else {
        // partial sums: [four columns][row][4] and (base, l) of every row, in one of this block's two places
        const long long w0 = w.w0;
        const int first = work_owner(w0, total, parts), last = work_owner(w0 + w.blocks - 1, total, parts);
        auto place = [&](int part) { return part * 2 + (part == first && work_begin(total, part, parts) < w0 ? 1 : 0); };
        const long long floats = (long long)(D + 2) * 128;
        {
          float* const to = a.partial + place(blockIdx.x) * floats;
          if (warp_used) {
            for (int i = half; i < pieces; i += 2) {
              uint32_t o[16];
              tmem_ld16(o_tmem + lanes + i * 16, o);
              if (mine) {
                uint4* at = reinterpret_cast<uint4*>(to) + i * 4 * 128 + row;
#pragma unroll
                for (int j = 0; j < 4; j++) at[j * 128] = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
              }
            }
            if (mine && half == 0) *reinterpret_cast<float2*>(to + D * 128 + row * 2) = make_float2(m == -INFINITY ? m : base, l);
          }
        }
        __threadfence();
        named_sync(5, kSoftmaxThreads);
        uint32_t* const counter = a.counters + (long long)w.head * a.max_tiles + w.index;
        if (tid == 0) {
          c.arrived = atomicAdd(counter, 1u);
          if (c.arrived == (uint32_t)(last - first)) *counter = 0;  // as it was found
        }
        named_sync(5, kSoftmaxThreads);
        done = c.arrived == (uint32_t)(last - first);
        if (done) {
          __threadfence();
          // rows' maxima and sums first, `share` threads to a row; then every thread four values at a time, four of them from four parts in flight
          const int count = last - first + 1;
          int share = 2;
          while (share < 32 && used * share * 2 <= kSoftmaxThreads) share *= 2;
          const int sub = tid & (share - 1), r0 = tid / share;
          auto at_ml = [&](int f, int r) { return reinterpret_cast<const float2*>(a.partial + place(first + f) * floats + D * 128 + r * 2); };
          float top = -INFINITY, sums = 0.f;
          if (r0 < used) {
#pragma unroll 4
            for (int f = sub; f < count; f += share) top = fmaxf(top, __ldcg(at_ml(f, r0)).x);
          }
          for (int o = 1; o < share; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float from = top == -INFINITY ? 0.f : top;
          if (r0 < used) {
#pragma unroll 4
            for (int f = sub; f < count; f += share) {
              const float2 ml = __ldcg(at_ml(f, r0));
              sums += ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - from) * ml.y;
            }
          }
          for (int o = 1; o < share; o <<= 1) sums += __shfl_xor_sync(0xffffffffu, sums, o);
          if (r0 < used && sub == 0) {
            if (sums == 0.f && top != -INFINITY) atomicOr(&c.bad_rows[r0 >> 5], 1u << (r0 & 31));
            c.top[0][0][r0] = from;
            c.top[0][1][r0] = sums > 0.f ? 1.f / sums : (sums == 0.f ? 0.f : sums);
          }
          named_sync(5, kSoftmaxThreads);
          for (int i = tid; i < used * pieces; i += kSoftmaxThreads) {  // 16 columns of a row
            const int pc = i / used, r = i - pc * used;
            const float top_r = c.top[0][0][r], inv = c.top[0][1][r];
            float o[16] = {};
            for (int f0 = 0; f0 < count; f0 += 4) {
              float4 x[4][4];
              float mf[4];
#pragma unroll
              for (int f = 0; f < 4; f++) {
                const float* part = a.partial + place(first + min(f0 + f, count - 1)) * floats;
                mf[f] = f0 + f < count ? __ldcg(part + D * 128 + r * 2) : -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; j++) x[f][j] = __ldcg(reinterpret_cast<const float4*>(part) + (pc * 4 + j) * 128 + r);
              }
#pragma unroll
              for (int f = 0; f < 4; f++) {
                if (mf[f] == -INFINITY) continue;  // that part saw no key of this row
                const float y = exp2_fast(mf[f] - top_r);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                  o[4 * j] += y * x[f][j].x; o[4 * j + 1] += y * x[f][j].y; o[4 * j + 2] += y * x[f][j].z; o[4 * j + 3] += y * x[f][j].w;
                }
              }
            }
            const int tk = page_of(r, a.group_div);
            finite = true;
            store(a.out + ((long long)(w.row0 + tk) * a.n_q + w.head * group + r - tk * group) * D + pc * 16, o, inv);
            if (!finite) atomicOr(&c.bad_rows[r >> 5], 1u << (r & 31));
            finite = true;
          }
        }
      }
      if (done) {
        if (mine && !finite) atomicOr(&c.bad_rows[row >> 5], 1u << (row & 31));
        named_sync(5, kSoftmaxThreads);
        const uint32_t bad[4] = {c.bad_rows[0], c.bad_rows[1], c.bad_rows[2], c.bad_rows[3]};
        if (bad[0] | bad[1] | bad[2] | bad[3]) {  // rare: an infinity or a NaN among the values
          auto sync = [] { named_sync(5, kSoftmaxThreads); };
          for (int r = 0; r < used; r++) {
            if (!(bad[r >> 5] >> (r & 31) & 1)) continue;
            const int tk = page_of(r, a.group_div);
            const long long p = (long long)w.first_pos + tk;
            attend_row(a, plain, tid, w.row0 + tk, w.head * group + r - tk * group, w.seq, (int)min(p, 0x7fffffffll), sync);
          }
          if (tid < 4) c.bad_rows[tid] = 0;
        }
      }
      tc_fence_before();
      named_sync(5, kSoftmaxThreads);  // everybody has read O, the exchange and the flags
      release_item(items);
    }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    __syncwarp();
    if (*(volatile int*)&c.abort) __nanosleep(1000000);  // let what is in flight land after a failed wait
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

template <int DC, int UNITS, bool I8>
cudaError_t run_tile(const AttnPagedArgs& a, cudaStream_t stream) {
  constexpr int smem = 1024 + (DC + UNITS) * kUnit + kMetaBlocks * (int)sizeof(Meta) + (int)sizeof(RowScratch) + (int)sizeof(Control);
  static_assert(smem <= 227 * 1024, "shared memory");
  static_assert((DC + UNITS) * kUnit >= (4096 + 1) * 4, "room for the sequences' first tiles");
  auto kernel = attn_paged_tile_kernel<DC, UNITS, I8>;
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
  return launch_dependent(kernel, dim3(a.grid), dim3(kThreads), smem, stream, a, m);
}

}  // namespace

void attn_paged_shape(AttnPagedArgs& a, int sms) {
  const int group = a.n_q / a.v.n_kv;
  a.tokens_per_tile = 128 / group;
  a.group_div = page_divisor(group);
  a.max_tiles = a.v.rows / a.tokens_per_tile + std::min(a.v.S, a.v.rows);
  a.grid = sms;
  a.box_rows = 128;
  while (a.box_rows > 4 && a.v.page_size % a.box_rows) a.box_rows /= 2;
  if (a.box_rows < 8) a.box_rows = 0;
}
size_t attn_paged_counter_bytes(const AttnPagedArgs& a) { return (size_t)a.v.n_kv * a.max_tiles * 4; }
size_t attn_paged_partial_bytes(const AttnPagedArgs& a) { return (size_t)a.grid * 2 * (a.v.D + 2) * 128 * 4; }

cudaError_t launch_attn_paged_tile(AttnPagedArgs a, cudaStream_t stream) {
  a.wait_ns = wait_limit_ns();
  const int units = (a.v.D + 63) / 64;
  if (a.scales)
    return units == 1 ? run_tile<1, 8, true>(a, stream) : units == 2 ? run_tile<2, 8, true>(a, stream)
         : units == 3 ? run_tile<3, 9, true>(a, stream) : run_tile<4, 9, true>(a, stream);
  return units == 1 ? run_tile<1, 8, false>(a, stream) : units == 2 ? run_tile<2, 8, false>(a, stream)
       : units == 3 ? run_tile<3, 9, false>(a, stream) : run_tile<4, 9, false>(a, stream);
}

}  // namespace tb200
