// A paged key/value cache and the ragged batch that works on it. Rows row_start[s] .. row_start[s + 1] - 1 of a chunk are the new
// tokens of sequence s, at positions context[s], context[s] + 1, ...; position p of a sequence lies at offset p % page_size of page
// table[s][p / page_size]. A page id outside [0, pages) holds nothing: what would be written there is dropped, its keys are not seen.
// The caches are [pages][page_size][n_kv * D] of one layer, bf16, or int8 with fp32 scales [pages][page_size][2 * n_kv] (of the
// keys, then of the values): a value is its integer times its scale.
#pragma once
#include <stdint.h>

#include "chunk_divide.h"

namespace tb200 {

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
  int capacity;              // max_pages * page_size, at most 2^30
  PageDivisor div;
};

}  // namespace tb200
