// Writing a chunk's keys and values into a paged cache, and reading tokens back (paged.cuh says how the cache is laid out).
#include <algorithm>

#include "dependent_launch.cuh"
#include "kernels.h"
#include "paged.cuh"

namespace tb200 {

namespace {

// Eight values of a head, held by one lane: elements i .. i + 3 of its first and of its second half.
struct HalfPair {
  float a[4], b[4];
};
__device__ __forceinline__ void unpack(uint2 w, float (&f)[4]) {
  f[0] = __uint_as_float(w.x << 16); f[1] = __uint_as_float(w.x & 0xffff0000u);
  f[2] = __uint_as_float(w.y << 16); f[3] = __uint_as_float(w.y & 0xffff0000u);
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int L>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Head norm y = x * rsqrt(mean(x^2) + eps) * (1 + w) and rotation (y1, y2) -> (y1 cos - y2 sin, y2 cos + y1 sin) of queries and keys, all in
// fp32 and rounded once, to bf16 (queries, bf16 caches) or to the nearest integer times amax / 127 (int8 caches; amax is of the fp32 values
// of one token's head). Values go to their pages as they are, or rounded the same way. A head whose amax is below 1e-34 is all zeros,
// with scale zero; one that holds an infinity or a NaN gets scale NaN and reads back as NaN.
// The angle of a far position needs more than fp32: position * turns[i] with turns[i] = theta^(-2i / D) / 2 pi as a 64-bit fraction of a turn,
// whose wrap-around is the reduction to one turn; its upper 32 bits go to sincospi.
// L lanes hold a head (L the power of two from D / 8 on); a group of L lanes takes `per` heads of one row, one after another,
// so that a row's angles are worked out once for them.
template <int L>
__global__ void __launch_bounds__(256) rope_kv_paged_kernel(const RopePagedArgs a) {
  const PagedView& v = a.v;
  const int lane = threadIdx.x & 31, sub = lane % L, half = v.D >> 1;
  const bool active = sub * 4 < half;
  unsigned long long turns[4] = {};
  if (active) {
#pragma unroll
    for (int j = 0; j < 4; j++) turns[j] = a.turns[sub * 4 + j];
  }
  grid_dependency_wait();
  grid_dependency_release();
  const int heads = a.n_q + 2 * v.n_kv, groups = (heads + a.per - 1) / a.per;
  const long long item = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
  constexpr int kItems = 32 / L;
  // the items of a warp may lie in several rows: each row's sequence is found by the whole warp
  const long long first_item = item - lane / L;
  int row = (int)(item / groups), seq = 0, pos = -1;
#pragma unroll
  for (int k = 0; k < kItems; k++) {
    const int r = (int)min((first_item + k) / groups, (long long)v.rows - 1);
    const int s = sequence_of_row(v, r);
    if (k == lane / L) seq = s;
  }
  if (row < v.rows) pos = row_position(v, seq, row);
  const long long slot = pos >= 0 ? slot_of(v, seq, pos) : -1;
  float cs[4], sn[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int top = (int)(((unsigned long long)(unsigned)max(pos, 0) * turns[j]) >> 32);
    sincospif((float)top * 4.6566128730773926e-10f, &sn[j], &cs[j]);  // 2^-31: a turn is 2 in units of pi
  }
  const int h0 = (int)(item % groups) * a.per;
  for (int h = h0; h < h0 + a.per; h++) {  // every lane of the warp stays: the sums below are the warp's
    const bool on = active && pos >= 0 && h < heads;
    const bool is_q = h < a.n_q, is_k = !is_q && h < a.n_q + v.n_kv;
    HalfPair x = {};
    if (on) {
      const uint16_t* src = a.qkv + ((long long)row * heads + h) * v.D + sub * 4;
      unpack(__ldg(reinterpret_cast<const uint2*>(src)), x.a);
      unpack(__ldg(reinterpret_cast<const uint2*>(src + half)), x.b);
    }
    if (a.norms) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) ss += x.a[j] * x.a[j] + x.b[j] * x.b[j];
      ss = group_sum<L>(ss);
      if (on && (is_q || is_k)) {
        const float inv = rsqrtf(ss / (float)v.D + a.eps);
        const uint16_t* w = a.norms + (is_q ? 0 : v.D) + sub * 4;
        float wa[4], wb[4];
        unpack(__ldg(reinterpret_cast<const uint2*>(w)), wa);
        unpack(__ldg(reinterpret_cast<const uint2*>(w + half)), wb);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          x.a[j] = x.a[j] * inv * (1.0f + wa[j]);
          x.b[j] = x.b[j] * inv * (1.0f + wb[j]);
        }
      }
    }
    if (is_q || is_k) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float p = x.a[j], q = x.b[j];
        x.a[j] = p * cs[j] - q * sn[j];
        x.b[j] = q * cs[j] + p * sn[j];
      }
    }
    float amax = 0.f, bad = 0.f;
    if (a.scales) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        amax = fmaxf(amax, fmaxf(fabsf(x.a[j]), fabsf(x.b[j])));
        bad += (x.a[j] - x.a[j]) + (x.b[j] - x.b[j]);  // NaN where a value is not finite
      }
      amax = group_max<L>(amax);
      bad = group_sum<L>(bad);
    }
    if (!on) continue;
    if (is_q) {
      uint16_t* dst = a.q_out + ((long long)row * a.n_q + h) * v.D + sub * 4;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(x.a[0], x.a[1]), pack_bf16(x.a[2], x.a[3]));
      *reinterpret_cast<uint2*>(dst + half) = make_uint2(pack_bf16(x.b[0], x.b[1]), pack_bf16(x.b[2], x.b[3]));
      continue;
    }
    if (slot < 0) continue;
    const int hk = is_k ? h - a.n_q : h - a.n_q - v.n_kv;
    const long long at = (slot * v.n_kv + hk) * v.D + sub * 4;
    void* pages = is_k ? a.k : a.vv;
    if (!a.scales) {
      uint16_t* dst = (uint16_t*)pages + at;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(x.a[0], x.a[1]), pack_bf16(x.a[2], x.a[3]));
      *reinterpret_cast<uint2*>(dst + half) = make_uint2(pack_bf16(x.b[0], x.b[1]), pack_bf16(x.b[2], x.b[3]));
      continue;
    }
    const bool finite = bad == 0.f;
    const float scale = amax < 1e-34f ? 0.f : amax / 127.f;
    const float inv = finite && scale > 0.f ? 1.0f / scale : 0.f;
    auto quant = [&](const float (&f)[4]) {
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int q = finite ? max(-127, min(127, __float2int_rn(f[j] * inv))) : 0;
        w |= (uint32_t)(uint8_t)q << (8 * j);
      }
      return w;
    };
    int8_t* dst = (int8_t*)pages + at;
    *reinterpret_cast<uint32_t*>(dst) = quant(x.a);
    *reinterpret_cast<uint32_t*>(dst + half) = quant(x.b);
    if (sub == 0) a.scales[slot * 2 * v.n_kv + (is_k ? 0 : v.n_kv) + hk] = finite ? scale : __uint_as_float(0x7fc00000u);
  }
}

// k_out / v_out [rows][n_kv * D] bf16: the tokens' keys and values, int8 ones as bf16(integer * scale); zeros where a position holds
// nothing. A warp takes a row.
template <bool I8>
__global__ void __launch_bounds__(256) kv_read_paged_kernel(const ReadPagedArgs a) {
  grid_dependency_wait();
  grid_dependency_release();
  const PagedView& v = a.v;
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= v.rows) return;
  const int seq = sequence_of_row(v, row);
  const int pos = row_position(v, seq, row);
  if (pos < 0) return;
  const long long slot = slot_of(v, seq, pos);
  const int width = v.n_kv * v.D, chunks = width / 8, per_head = v.D / 8;
  for (int i = lane; i < 2 * chunks; i += 32) {
    const bool is_v = i >= chunks;
    const int c = is_v ? i - chunks : i;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (slot >= 0) {
      const long long at = slot * width + c * 8;
      const void* pages = is_v ? a.vv : a.k;
      if (!I8) {
        w = __ldg(reinterpret_cast<const uint4*>((const uint16_t*)pages + at));
      } else {
        const uint2 b = __ldg(reinterpret_cast<const uint2*>((const int8_t*)pages + at));
        const float s = __ldg(a.scales + slot * 2 * v.n_kv + (is_v ? v.n_kv : 0) + c / per_head);
        auto two = [&](uint32_t word, int j) {
          return pack_bf16((float)(int8_t)(word >> (8 * j)) * s, (float)(int8_t)(word >> (8 * j + 8)) * s);
        };
        w = make_uint4(two(b.x, 0), two(b.x, 2), two(b.y, 0), two(b.y, 2));
      }
    }
    *reinterpret_cast<uint4*>((is_v ? a.v_out : a.k_out) + (long long)row * width + c * 8) = w;
  }
}

}  // namespace

cudaError_t launch_rope_kv_paged(RopePagedArgs a, cudaStream_t stream) {
  const int heads = a.n_q + 2 * a.v.n_kv;
  // One head to a group until the machine is full (a group is at most a warp, an SM runs 64 of them): a single token's heads then run beside
  // one another; more rows share the work on their angles over up to eight heads.
  const long long warps = 64ll * current_sm_count();
  a.per = 1;
  while (a.per < 8 && a.per < heads && (long long)a.v.rows * heads / (2 * a.per) >= 2 * warps) a.per *= 2;
  const long long items = (long long)a.v.rows * ((heads + a.per - 1) / a.per);
  auto run = [&](auto kernel, int lanes) {
    const int per_block = 256 / lanes;
    return launch_dependent(kernel, dim3((unsigned)((items + per_block - 1) / per_block)), dim3(256), 0, stream, a);
  };
  const int need = a.v.D / 8;
  if (need <= 2) return run(rope_kv_paged_kernel<2>, 2);
  if (need <= 4) return run(rope_kv_paged_kernel<4>, 4);
  if (need <= 8) return run(rope_kv_paged_kernel<8>, 8);
  if (need <= 16) return run(rope_kv_paged_kernel<16>, 16);
  return run(rope_kv_paged_kernel<32>, 32);
}

cudaError_t launch_kv_read_paged(const ReadPagedArgs& a, cudaStream_t stream) {
  const dim3 grid((a.v.rows + 7) / 8);
  return a.scales ? launch_dependent(kv_read_paged_kernel<true>, grid, dim3(256), 0, stream, a)
                  : launch_dependent(kv_read_paged_kernel<false>, grid, dim3(256), 0, stream, a);
}

}  // namespace tb200
