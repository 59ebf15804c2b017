// One query head of one token against its keys, exactly as the mask says: keys it does not see are not touched. The plain form of
// attn_paged, which the kernels fall back to for a row whose sums are not finite (a matrix product multiplies what a hidden key's value
// holds by zero, and zero times infinity is not zero).
#pragma once
#include "kernels.h"
#include "paged.cuh"

namespace tb200 {

template <int THREADS>
struct RowScratch {
  float q[256], p[THREADS], red[8];
  long long slots[THREADS];
};

// By threads t = 0 .. THREADS - 1 (whole warps, 128 or 256) that `sync` synchronises. Writes dims d0 .. d1 - 1 of the row.
template <int THREADS, typename Sync>
__device__ __noinline__ void attend_row(const AttnPagedArgs& a, RowScratch<THREADS>& sm, int t, int row, int h, int seq, int pos, int d0, int d1, Sync sync) {
  constexpr int kDims = 256 / THREADS;  // a thread's: t, t + THREADS
  const PagedView& v = a.v;
  const int hk = h / (a.n_q / v.n_kv);
  const long long at_q = ((long long)row * a.n_q + h) * v.D;
  sync();
  for (int d = t; d < v.D; d += THREADS) sm.q[d] = paged_bf2f(a.q[at_q + d]) * a.scale;
  const int last = min(pos, v.capacity - 1), near = a.window ? max(0, pos - a.window + 1) : 0;
  float m = -INFINITY, sum = 0.f, o[kDims] = {};
  auto block_all = [&](float x, bool max_of) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, x, off);
      x = max_of ? fmaxf(x, y) : x + y;
    }
    sync();
    if ((t & 31) == 0) sm.red[t >> 5] = x;
    sync();
    x = sm.red[0];
    for (int w = 1; w < THREADS / 32; w++) x = max_of ? fmaxf(x, sm.red[w]) : x + sm.red[w];
    return x;
  };
  for (int j0 = 0; j0 <= last; j0 += THREADS) {
    if (j0 >= a.sinks && j0 + THREADS <= near) continue;
    const int j = j0 + t;
    const bool seen = j <= last && (j >= near || j < a.sinks);
    const long long slot = seen ? slot_of(v, seq, j) : -1;
    float s = -INFINITY, vs = 0.f;
    sync();  // q is there, and the last round's p and slots have been read
    if (slot >= 0) {
      s = 0.f;
      const long long at = (slot * v.n_kv + hk) * v.D;
      if (a.scales) {
#pragma unroll 1
        for (int d = 0; d < v.D; d++) s += sm.q[d] * (float)((const int8_t*)a.k)[at + d];
        s *= a.scales[slot * 2 * v.n_kv + hk];
        vs = a.scales[slot * 2 * v.n_kv + v.n_kv + hk];
      } else {
#pragma unroll 1
        for (int d = 0; d < v.D; d++) s += sm.q[d] * paged_bf2f(((const uint16_t*)a.k)[at + d]);
        vs = 1.f;
      }
    }
    const float top = fmaxf(m, block_all(s, true));
    const float p = slot >= 0 ? __expf(s - top) : 0.f, keep = m == top ? 1.f : __expf(m - top);
    m = top;
    sm.p[t] = p * vs;
    sm.slots[t] = slot;
    sum = sum * keep + block_all(p, false);
#pragma unroll
    for (int e = 0; e < kDims; e++) {
      const int d = t + e * THREADS;
      o[e] *= keep;
      if (d >= v.D) continue;
#pragma unroll 1
      for (int i = 0; i < THREADS; i++) {
        if (sm.slots[i] < 0) continue;
        const long long at = (sm.slots[i] * v.n_kv + hk) * v.D + d;
        o[e] += sm.p[i] * (a.scales ? (float)((const int8_t*)a.vv)[at] : paged_bf2f(((const uint16_t*)a.vv)[at]));
      }
    }
  }
#pragma unroll
  for (int e = 0; e < kDims; e++) {
    const int d = t + e * THREADS;
    if (d < v.D && d >= d0 && d < d1) a.out[at_q + d] = __bfloat16_as_ushort(__float2bfloat16_rn(sum == 0.f ? 0.f : o[e] / sum));
  }
  sync();
}

}  // namespace tb200
