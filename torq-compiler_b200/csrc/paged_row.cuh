// One query head of one token against its keys, exactly as the mask says: keys it does not see are not touched. The plain form of
// attn_paged, which the kernels fall back to for a row whose sums are not finite (a matrix product multiplies what a hidden key's value
// holds by zero, and zero times infinity is not zero).
#pragma once
#include "kernels.h"
#include "paged.cuh"

namespace tb200 {

constexpr int kRowThreads = 256;
struct RowScratch {
  float q[256], p[kRowThreads], red[kRowThreads / 32];
  long long slots[kRowThreads];
};

// By kRowThreads threads t = 0 .. kRowThreads - 1 (whole warps) that `sync` synchronises.
template <typename Sync>
__device__ __noinline__ void attend_row(const AttnPagedArgs& a, RowScratch& sm, int t, int row, int h, int seq, int pos, Sync sync) {
  const PagedView& v = a.v;
  const int hk = h / (a.n_q / v.n_kv);
  const long long at_q = ((long long)row * a.n_q + h) * v.D;
  sync();
  if (t < v.D) sm.q[t] = paged_bf2f(a.q[at_q + t]) * a.scale;
  const int last = min(pos, v.capacity - 1), near = a.window ? max(0, pos - a.window + 1) : 0;
  float m = -INFINITY, sum = 0.f, o = 0.f;
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
    for (int w = 1; w < kRowThreads / 32; w++) x = max_of ? fmaxf(x, sm.red[w]) : x + sm.red[w];
    return x;
  };
  for (int j0 = 0; j0 <= last; j0 += kRowThreads) {
    if (j0 >= a.sinks && j0 + kRowThreads <= near) continue;
    const int j = j0 + t;
    const bool seen = j <= last && (j >= near || j < a.sinks);
    const long long slot = seen ? slot_of(v, seq, j) : -1;
    float s = -INFINITY, vs = 0.f;
    sync();  // q is there, and the last round's p and slots have been read
    if (slot >= 0) {
      s = 0.f;
      const long long at = (slot * v.n_kv + hk) * v.D;
      if (a.scales) {
        for (int d = 0; d < v.D; d++) s += sm.q[d] * (float)((const int8_t*)a.k)[at + d];
        s *= a.scales[slot * 2 * v.n_kv + hk];
        vs = a.scales[slot * 2 * v.n_kv + v.n_kv + hk];
      } else {
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
    o *= keep;
    if (t < v.D)
      for (int i = 0; i < kRowThreads; i++) {
        if (sm.slots[i] < 0) continue;
        const long long at = (sm.slots[i] * v.n_kv + hk) * v.D + t;
        o += sm.p[i] * (a.scales ? (float)((const int8_t*)a.vv)[at] : paged_bf2f(((const uint16_t*)a.vv)[at]));
      }
  }
  if (t < v.D) a.out[at_q + t] = __bfloat16_as_ushort(__float2bfloat16_rn(sum == 0.f ? 0.f : o / sum));
  sync();
}

}  // namespace tb200
