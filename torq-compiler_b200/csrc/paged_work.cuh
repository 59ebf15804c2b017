// What the kernels of attn_paged share: how a block of the grid comes by its work, where its keys lie, and small arithmetic.
#pragma once
#include "kernels.h"
#include "paged.cuh"
#include "widen.cuh"

namespace tb200 {

// A piece of work of a block of the grid: key blocks b0 .. b1 - 1 of a tile of one key/value head.
struct Item {
  int seq, head;
  int row0, tokens;         // the tile's rows of the chunk; tokens 0: there is no more work
  int first_pos;            // position of the first token
  int near_key, end_key, front, shift, blocks;  // tile_span
  int b0, b1;
  long long w0;             // where the tile's work begins
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
// A kernel leaves the other kernel's sequences alone: those of few rows, or those of more.
__device__ __forceinline__ int tiles_of(const AttnPagedArgs& a, const Span& s) {
  const bool few = s.n * (a.n_q / a.v.n_kv) <= a.few_rows;
  return few == (a.takes_few != 0) ? (s.n + a.tokens_per_tile - 1) / a.tokens_per_tile : 0;
}

// The keys of an item, and where the cache holds them. Page ids are asked for a block ahead of their use, without a branch (a branch would wait
// for each); slots have 32 bits (the planner refuses more), -1 where no token of the tile sees the key or nothing is held.
struct Keys {
  const int32_t* pages_of;
  int near_key, end_key, sinks, front, shift, last, pages, page_size;
  PageDivisor div;
  __device__ __forceinline__ Keys(const AttnPagedArgs& a, const Item& w)
      : pages_of(a.v.table + (long long)w.seq * a.v.max_pages), near_key(w.near_key), end_key(w.end_key), sinks(a.sinks), front(w.front),
        shift(w.shift), last(a.v.capacity - 1), pages(a.v.pages), page_size(a.v.page_size), div(a.v.div) {}
  __device__ __forceinline__ int at(int place) const { return tile_key(front, shift, place); }
  __device__ __forceinline__ int ask(int key) const {
    int page;  // volatile: it is to be on its way now, not when it is used
    asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(page) : "l"(pages_of + page_of(min(key, last), div)));
    return page;
  }
  __device__ __forceinline__ bool seen(int key) const { return key < end_key && (key >= near_key || key < sinks); }  // by a token of the tile
  __device__ __forceinline__ int slot(int key, int page) const {
    const bool there = seen(key) && page >= 0 && page < pages;
    return there ? page * page_size + (key - page_of(key, div) * page_size) : -1;
  }
};

struct WorkShared {
  int totals[32];
  int start_seq, start_tile, start_index, start_off;
};
// Running sum over the block's threads up to and including this one, and the sum of all, through c.totals.
template <int THREADS>
__device__ __noinline__ int block_scan(WorkShared& c, int x, int& all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) c.totals[warp] = v;
  __syncthreads();
  const int y = lane < THREADS / 32 ? c.totals[lane] : 0;
  all = __reduce_add_sync(0xffffffffu, y);
  return v + __reduce_add_sync(0xffffffffu, lane < warp ? y : 0);
}

// All tiles of all heads, each with its key blocks, lie in one row, which the blocks of the grid share out evenly; this one has [begin, end).
struct Work {
  long long total, begin, end;
  int parts, n_tiles, head0;
  bool works;
};
// By all THREADS threads of the block. first_tile: room for S + 1 numbers, free again after the caller's next __syncthreads().
template <int THREADS>
__device__ __forceinline__ Work share_out(const AttnPagedArgs& a, WorkShared& c, int* first_tile) {
  const PagedView& v = a.v;
  const int tid = threadIdx.x;
  int all = 0, run = 0;
  for (int s0 = 0; s0 < v.S; s0 += THREADS) {
    const int s = s0 + tid, upto = run + block_scan<THREADS>(c, s < v.S ? tiles_of(a, span_of(a, s)) : 0, all);
    if (s < v.S) first_tile[s + 1] = upto;
    run += all;
  }
  if (tid == 0) first_tile[0] = 0;
  __syncthreads();
  Work w;
  w.n_tiles = min(run, a.max_tiles);
  int seq = 0, tile = 0;
  auto blocks_of = [&](int i) {
    int lo = 0, hi = v.S - 1;  // the last sequence with first_tile[seq] <= i
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first_tile[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    seq = lo;
    tile = i - first_tile[lo];
    const Span sp = span_of(a, seq);
    return kTileCost + tile_span(sp.ctx, sp.n, tile, a.tokens_per_tile, a.window, a.sinks, v.capacity).blocks;
  };
  int per_head = 0;  // the planner refuses what 32 bits do not hold
  for (int i0 = 0; i0 < w.n_tiles; i0 += THREADS) {
    block_scan<THREADS>(c, i0 + tid < w.n_tiles ? blocks_of(i0 + tid) : 0, all);
    per_head += all;
  }
  w.total = (long long)per_head * v.n_kv;
  w.parts = (int)max(1ll, min((long long)gridDim.x, w.total / a.min_blocks));
  w.works = w.total > 0 && (int)blockIdx.x < w.parts;
  w.begin = w.works ? work_begin(w.total, blockIdx.x, w.parts) : 0;
  w.end = w.works ? work_begin(w.total, blockIdx.x + 1, w.parts) : 0;
  w.head0 = w.works ? (int)(w.begin / per_head) : 0;
  const int rem = (int)(w.begin - (long long)w.head0 * per_head);
  for (int i0 = 0, before = 0; w.works && i0 < w.n_tiles && before <= rem; i0 += THREADS) {
    const int i = i0 + tid, n = i < w.n_tiles ? blocks_of(i) : 0, upto = before + block_scan<THREADS>(c, n, all);
    if (n && upto > rem && upto - n <= rem) {
      c.start_tile = tile;
      c.start_seq = seq;
      c.start_index = i;
      c.start_off = rem - (upto - n);
    }
    before += all;
  }
  return w;
}

// A block's items, one after another.
struct ItemCursor {
  long long cur;
  int head, seq, tile, index, off, tiles;
  Span span;
  __device__ __forceinline__ ItemCursor(const AttnPagedArgs& a, const Work& w, const WorkShared& c)
      : cur(w.begin), head(w.head0), seq(c.start_seq), tile(c.start_tile), index(c.start_index), off(c.start_off) {
    span = span_of(a, seq);
    tiles = tiles_of(a, span);
  }
  // the next one, or false (and one without tokens) when there are no more
  __device__ __forceinline__ bool take(const AttnPagedArgs& a, const Work& work, Item& w) {
    const int tpt = a.tokens_per_tile;
    while (cur < work.end) {
      const TileSpan ts = tile_span(span.ctx, span.n, tile, tpt, a.window, a.sinks, a.v.capacity);
      const int upto = (int)min((long long)ts.blocks + kTileCost, off + (work.end - cur));
      const bool any = upto > kTileCost;  // not only the front of a tile whose blocks are the next one's
      if (any) {
        w.seq = seq; w.head = head;
        w.row0 = span.row0 + tile * tpt;
        w.tokens = min(tpt, span.n - tile * tpt);
        w.first_pos = (int)min((long long)span.ctx + tile * tpt, 0x7fffffffll);
        w.near_key = ts.near_key; w.end_key = ts.end_key; w.front = ts.front; w.shift = ts.shift; w.blocks = ts.blocks;
        w.b0 = max(off - kTileCost, 0); w.b1 = upto - kTileCost;
        w.w0 = cur - off + kTileCost;
      }
      cur += upto - off;
      off = 0;
      if (cur < work.end) {
        tile++;
        if (++index >= work.n_tiles) {  // the next head begins
          index = 0;
          head++;
          seq = -1;
          tile = tiles;
        }
        if (tile >= tiles) {
          tile = 0;
          do {
            if (++seq >= a.v.S) seq = 0;  // there is a tile, so a sequence with one
            span = span_of(a, seq);
            tiles = tiles_of(a, span);
          } while (!tiles);
        }
      }
      if (any) return true;
    }
    w.tokens = 0;
    return false;
  }
};
// By the first block of those that share the tile.
__device__ __forceinline__ void write_join(const AttnPagedArgs& a, const Work& work, const Item& w, int first, int used) {
  AttnJoin& j = a.joins[first];
  j.first = first;
  j.second_place = work.begin < w.w0;
  j.row0 = w.row0; j.used = used; j.head = w.head; j.seq = w.seq; j.first_pos = w.first_pos;
  j.parts = work_owner(w.w0 + w.blocks - 1, work.total, work.parts) - first + 1;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace tb200
