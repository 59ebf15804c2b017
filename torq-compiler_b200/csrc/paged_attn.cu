// Attention of a chunk's queries over a paged cache (paged.cuh): o = softmax(scale * q k^T) v over the keys a token at position p sees,
// j <= p and (window == 0 or j > p - window or j < sinks), where their page holds something. A token that sees nothing gets zeros.
#include <algorithm>

#include "dependent_launch.cuh"
#include "kernels.h"
#include "paged.cuh"

namespace tb200 {

namespace {

// A block is one query head of one row: each thread has a key of its own for the scores, a dimension for the sums.
constexpr int kRowThreads = 128;
__global__ void __launch_bounds__(kRowThreads) attn_paged_row_kernel(const AttnPagedArgs a) {
  grid_dependency_wait();
  grid_dependency_release();
  const PagedView& v = a.v;
  __shared__ float qs[256], ps[kRowThreads], red[4];
  __shared__ long long slots[kRowThreads];
  const int row = blockIdx.x, h = blockIdx.y, t = threadIdx.x;
  const int seq = sequence_of_row(v, row);
  const int pos = row_position(v, seq, row);
  if (pos < 0 || (a.max_new && row - max(v.row_start[seq], 0) >= a.max_new)) return;
  const int hk = h / (a.n_q / v.n_kv);
  for (int d = t; d < v.D; d += kRowThreads) qs[d] = paged_bf2f(a.q[((long long)row * a.n_q + h) * v.D + d]) * a.scale;
  const int last = min(pos, v.capacity - 1), near = a.window ? max(0, pos - a.window + 1) : 0;
  float m = -INFINITY, sum = 0.f, o[2] = {0.f, 0.f};
  for (int j0 = 0; j0 <= last; j0 += kRowThreads) {
    if (j0 >= a.sinks && j0 + kRowThreads <= near) continue;
    const int j = j0 + t;
    const bool seen = j <= last && (j >= near || j < a.sinks);
    const long long slot = seen ? slot_of(v, seq, j) : -1;
    float s = -INFINITY, vs = 0.f;
    __syncthreads();
    if (slot >= 0) {
      s = 0.f;
      const long long at = (slot * v.n_kv + hk) * v.D;
      if (a.scales) {
        for (int d = 0; d < v.D; d++) s += qs[d] * (float)((const int8_t*)a.k)[at + d];
        s *= a.scales[slot * 2 * v.n_kv + hk];
        vs = a.scales[slot * 2 * v.n_kv + v.n_kv + hk];
      } else {
        for (int d = 0; d < v.D; d++) s += qs[d] * paged_bf2f(((const uint16_t*)a.k)[at + d]);
        vs = 1.f;
      }
    }
    float top = s;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if ((t & 31) == 0) red[t >> 5] = top;
    __syncthreads();
    top = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float p = slot >= 0 ? __expf(s - top) : 0.f, keep = m == top ? 1.f : __expf(m - top);
    m = top;
    float part = p;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) part += __shfl_xor_sync(0xffffffffu, part, off);
    __syncthreads();
    if ((t & 31) == 0) red[t >> 5] = part;
    ps[t] = p * vs;
    slots[t] = slot;
    __syncthreads();
    sum = sum * keep + red[0] + red[1] + red[2] + red[3];
    for (int e = 0; e < 2; e++) {
      const int d = t + e * kRowThreads;
      if (d >= v.D) break;
      float acc = o[e] * keep;
      for (int i = 0; i < kRowThreads; i++) {
        if (slots[i] < 0) continue;
        const long long at = (slots[i] * v.n_kv + hk) * v.D + d;
        acc += ps[i] * (a.scales ? (float)((const int8_t*)a.vv)[at] : paged_bf2f(((const uint16_t*)a.vv)[at]));
      }
      o[e] = acc;
    }
  }
  for (int e = 0; e < 2; e++) {
    const int d = t + e * kRowThreads;
    if (d < v.D) a.out[((long long)row * a.n_q + h) * v.D + d] = __bfloat16_as_ushort(__float2bfloat16_rn(sum == 0.f ? 0.f : o[e] / sum));
  }
}

}  // namespace

cudaError_t launch_attn_paged(const AttnPagedArgs& a, cudaStream_t stream) {
  return launch_dependent(attn_paged_row_kernel, dim3(a.v.rows, a.n_q), dim3(kRowThreads), 0, stream, a);
}

}  // namespace tb200
