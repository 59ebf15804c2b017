// Device side of a paged cache (paged.h): which sequence a row belongs to, and where a position lies.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "paged.h"

namespace tb200 {

__device__ __forceinline__ float paged_bf2f(uint32_t bits) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// The sequence of row r, found by a warp: the number of sequences that end at or before it, 32 candidates at a time. What a
// row_start that does not ascend yields is still one of [0, S].
__device__ __forceinline__ int sequence_of_row(const PagedView& v, int r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = v.S;  // sequences before lo end at or before r; what is open are the n ends row_start[lo + 1 ..]
  while (n > 0) {
    const int step = (n + 31) / 32;  // a lane looks at the last end of a group of `step`
    const int below = __popc(__ballot_sync(0xffffffffu, lane * step < n && v.row_start[lo + min((lane + 1) * step, n)] <= r));
    const int skip = min(below * step, n);
    lo += skip;
    n = step == 1 ? 0 : min(step, n - skip);
  }
  return lo;
}

// Position of row r in sequence s, or -1 where the row belongs to no sequence (padding).
__device__ __forceinline__ int row_position(const PagedView& v, int s, int r) {
  if (s >= v.S) return -1;
  const int first = max(v.row_start[s], 0);
  if (r < first || r >= v.row_start[s + 1]) return -1;
  const long long p = (long long)max(v.context[s], 0) + (r - first);
  return (int)min(p, (long long)0x7fffffff);
}

// Slot (page * page_size + offset) of a position, or -1 where it holds nothing.
__device__ __forceinline__ long long slot_of(const PagedView& v, int s, int pos) {
  if (pos < 0 || pos >= v.capacity) return -1;
  const int i = page_of(pos, v.div);
  const int page = __ldg(v.table + (long long)s * v.max_pages + i);
  if (page < 0 || page >= v.pages) return -1;
  return (long long)page * v.page_size + (pos - i * v.page_size);
}

}  // namespace tb200
