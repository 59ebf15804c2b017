// A paged key/value cache and the ragged batch that works on it. Rows row_start[s] .. row_start[s + 1] - 1 of a chunk are the new
// tokens of sequence s, at positions context[s], context[s] + 1, ...; position p of a sequence lies at offset p % page_size of page
// table[s][p / page_size]. A page id outside [0, pages) holds nothing: what would be written there is dropped, its keys are not seen.
// The caches are [pages][page_size][n_kv * D] of one layer, bf16, or int8 with fp32 scales [pages][page_size][2 * n_kv] (of the
// keys, then of the values): a value is its integer times its scale.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <initializer_list>

#include "chunk_divide.h"

namespace tb200 {

// What an op reads while it writes must not lie under what it writes. The first `written` ranges are written, the others only read (those may
// lie over one another); a range of no bytes is nowhere.
struct ByteRange {
  const void* at;
  size_t bytes;
};
inline bool writes_lie_apart(std::initializer_list<ByteRange> ranges, int written) {
  const ByteRange* r = ranges.begin();
  for (int i = 0; i < written; i++)
    for (int j = i + 1; j < (int)ranges.size(); j++)
      if (r[i].bytes && r[j].bytes && (uintptr_t)r[i].at < (uintptr_t)r[j].at + r[j].bytes && (uintptr_t)r[j].at < (uintptr_t)r[i].at + r[i].bytes) return false;
  return true;
}

// n / d for 0 <= n < 2^31: with l = ceil(log2 d) and m = floor(2^32 * (2^l - d) / d) + 1, the quotient is (mulhi(n, m) + n) >> l (the
// round-up multiplier m + 2^32 exceeds 2^(32 + l) / d by less than 2^l / d, which no n below 2^32 turns into a step; n < 2^31 keeps
// the sum in 32 bits).
struct PageDivisor {
  uint32_t m = 0;
  int l = 0;
};
inline PageDivisor page_divisor(int d) {
  int l = 0;
  while ((1ll << l) < d) l++;
  return {(uint32_t)((((1ull << l) - (uint64_t)d) << 32) / (uint64_t)d + 1), l};
}
TB200_BOTH int page_of(int n, PageDivisor d) {
#ifdef __CUDA_ARCH__
  return (int)((__umulhi((uint32_t)n, d.m) + (uint32_t)n) >> d.l);
#else
  return (int)(((uint32_t)(((uint64_t)(uint32_t)n * d.m) >> 32) + (uint32_t)n) >> d.l);
#endif
}

struct PagedView {
  const int32_t* row_start;  // [S + 1], ascending
  const int32_t* context;    // [S]
  const int32_t* table;      // [S][max_pages]
  int rows, S, max_pages, page_size, pages, n_kv, D;
  int i8;                    // the caches hold int8
  int capacity;              // max_pages * page_size, at most 2^30
  PageDivisor div;
};

// ---- how attention cuts a chunk into tiles, and shares the tiles' work out ----
// A tile is up to tokens_per_tile new tokens of a sequence with the query heads of one key/value head; its work is the keys that one of its
// tokens may see, in blocks of kKeyBlock: those of the first tokens that stay visible, and right behind them those from the window's start on.
// (As a block of their own 4 first tokens cost a window of 512 over
// 8192 tokens, 16/2 heads of 64, 142.7 us instead of 94.0.)
constexpr int kKeyBlock = 128;
constexpr int kSpanAlign = 16;  // where both parts begin and the first one ends: keys that lie one behind another from such a place on still do
struct TileSpan {
  int front;     // places 0 .. front - 1 of the tile's keys are those keys
  int shift;     // place i from there on is key i + shift
  int blocks;    // in all; at least one, so that a tile that sees nothing is visited as well
  int near_key;  // keys in front of it are seen as first tokens only
  int end_key;   // one past the last key a token of the tile sees
};
TB200_BOTH long long span_min(long long a, long long b) { return a < b ? a : b; }
TB200_BOTH TileSpan tile_span(int ctx, int n, int tile, int tokens_per_tile, int window, int sinks, int capacity) {
  const long long first = (long long)ctx + (long long)tile * tokens_per_tile;
  const long long end = span_min((long long)ctx + span_min((long long)(tile + 1) * tokens_per_tile, n), capacity);
  long long near = window > 0 && first - window + 1 > 0 ? first - window + 1 : 0;
  near = span_min(near, end);
  TileSpan s;
  s.near_key = (int)near;
  s.end_key = (int)end;
  // from here on in 32 bits and without divisions: the capacity is at most 2^30
  const uint32_t front = ((uint32_t)sinks + kSpanAlign - 1) & ~(uint32_t)(kSpanAlign - 1);
  int base = s.near_key & (sinks > 0 ? -kSpanAlign : -kKeyBlock);  // the window's part
  s.front = 0;
  if (sinks > 0) {
    if (front <= (uint32_t)base) s.front = (int)front;
    else base = 0;  // no gap between the two
  }
  s.shift = base - s.front;
  // (a window that lies behind the table's end leaves the first tokens)
  const int places = s.near_key < s.end_key ? s.end_key - s.shift : s.front ? s.front : sinks < s.end_key ? sinks : s.end_key;
  s.blocks = (places + kKeyBlock - 1) / kKeyBlock;
  if (s.blocks < 1) s.blocks = 1;
  return s;
}
// A tile counts as its blocks and, in front of them, kTileCost more: what it takes to begin it and to store its rows.
constexpr int kTileCost = 1;
TB200_BOTH int tile_key(int front, int shift, int place) { return place < front ? place : place + shift; }
// `total` pieces of work in one row, shared out to `parts`: part i begins here
TB200_BOTH long long work_begin(long long total, int i, int parts) { return total * i / parts; }
TB200_BOTH int work_owner(long long w, long long total, int parts) {
  int c = (int)(w * parts / total);
  while (c + 1 < parts && work_begin(total, c + 1, parts) <= w) c++;
  while (c > 0 && work_begin(total, c, parts) > w) c--;
  return c;
}

}  // namespace tb200
