// Writing a chunk's keys and values into a paged cache, and reading tokens back (paged.cuh says how the cache is laid out).
#include <algorithm>

#include "dependent_launch.cuh"
#include "kernels.h"
#include "paged.cuh"

namespace tb200 {

namespace {

__device__ __forceinline__ void unpack(uint4 w, float (&f)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; j++) {
    f[2 * j] = __uint_as_float(u[j] << 16);
    f[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack(const float (&f)[8]) {
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int L>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// The sequence of a row at or behind `first`, whose sequence is s: lanes may ask for different rows.
__device__ __forceinline__ int sequence_from(const PagedView& v, int s, int row) {
  while (s < v.S && v.row_start[s + 1] <= row) s++;
  return s;
}

// Head norm y = x * rsqrt(mean(x^2) + eps) * (1 + w) and rotation (y1, y2) -> (y1 cos - y2 sin, y2 cos + y1 sin) of queries and keys, all in
// fp32 and rounded once, to bf16 (queries, bf16 caches) or to the nearest integer times amax / 127 (int8 caches; amax is of the fp32 values
// of one token's head). Values go to their pages as they are, or rounded the same way. A head whose amax is below 1e-34 is all zeros,
// with scale zero; one that holds an infinity or a NaN gets scale NaN and reads back as NaN.
// The angle of a far position needs more than fp32: position * turns[i] with turns[i] = theta^(-2i / D) / 2 pi as a 64-bit fraction of a turn,
// whose wrap-around is the reduction to one turn; its upper 32 bits go to sincospi.
// L lanes hold a head (L the power of two from D / 16 on), eight neighbouring values of each half to a lane, so that every access has 16
// bytes; a group of L lanes takes `per` heads of one row, one after another, so that a row's angles are worked out once for them, and asks
// for the next head before it works on one.
template <int L>
__global__ void __launch_bounds__(256) rope_kv_paged_kernel(const RopePagedArgs a) {
  const PagedView& v = a.v;
  const int lane = threadIdx.x & 31, sub = lane % L, half = v.D >> 1;
  const bool active = sub * 8 < half;
  grid_dependency_wait();
  grid_dependency_release();
  const int heads = a.n_q + 2 * v.n_kv, groups = (heads + a.per - 1) / a.per;
  const long long item = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
  const int row = (int)min(item / groups, 0x7fffffffll), h0 = (int)(item % groups) * a.per, h1 = min(h0 + a.per, heads);
  const uint16_t* const src = a.qkv + (long long)row * heads * v.D + sub * 8;
  uint4 next_a = make_uint4(0, 0, 0, 0), next_b = next_a;
  auto ask = [&](int h) {
    if (active && row < v.rows && h < h1) {
      next_a = __ldg(reinterpret_cast<const uint4*>(src + h * v.D));
      next_b = __ldg(reinterpret_cast<const uint4*>(src + h * v.D + half));
    }
  };
  ask(h0);
  // the items of a warp may lie in several rows: the warp looks for the first one's sequence, and each goes on from there
  const int first = (int)min((item - lane / L) / groups, (long long)v.rows - 1);
  const int seq = sequence_from(v, sequence_of_row(v, first), min(row, v.rows - 1));
  const int pos = row < v.rows ? row_position(v, seq, row) : -1;
  const long long slot = pos >= 0 ? slot_of(v, seq, pos) : -1;
  float cs[8], sn[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int top = active ? (int)(((unsigned long long)(unsigned)max(pos, 0) * __ldg(a.turns + sub * 8 + j)) >> 32) : 0;
    sincospif((float)top * 4.6566128730773926e-10f, &sn[j], &cs[j]);  // 2^-31: a turn is 2 in units of pi
  }
  for (int i = 0; i < a.per; i++) {  // every lane of the warp stays: the sums below are the warp's
    const int h = h0 + i;
    const bool on = active && pos >= 0 && h < h1;
    const bool is_q = h < a.n_q, is_k = !is_q && h < a.n_q + v.n_kv;
    float xa[8], xb[8];
    unpack(next_a, xa);
    unpack(next_b, xb);
    ask(h + 1);
    if (a.norms) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j++) ss += xa[j] * xa[j] + xb[j] * xb[j];
      ss = group_sum<L>(ss);
      if (on && (is_q || is_k)) {
        const float inv = rsqrtf(ss / (float)v.D + a.eps);
        const uint16_t* w = a.norms + (is_q ? 0 : v.D) + sub * 8;
        float wa[8], wb[8];
        unpack(__ldg(reinterpret_cast<const uint4*>(w)), wa);
        unpack(__ldg(reinterpret_cast<const uint4*>(w + half)), wb);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          xa[j] = xa[j] * inv * (1.0f + wa[j]);
          xb[j] = xb[j] * inv * (1.0f + wb[j]);
        }
      }
    }
    if (is_q || is_k) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float p = xa[j], q = xb[j];
        xa[j] = p * cs[j] - q * sn[j];
        xb[j] = q * cs[j] + p * sn[j];
      }
    }
    uint32_t top = 0;  // bits of the largest magnitude; those of a NaN are above an infinity's, and these above every number's
    if (a.scales) {
      if (on) {
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, max(__float_as_uint(fabsf(xa[j])), __float_as_uint(fabsf(xb[j]))));
      }
      top = group_max<L>(top);
    }
    if (!on) continue;
    if (is_q) {
      uint16_t* dst = a.q_out + ((long long)row * a.n_q + h) * v.D + sub * 8;
      *reinterpret_cast<uint4*>(dst) = pack(xa);
      *reinterpret_cast<uint4*>(dst + half) = pack(xb);
      continue;
    }
    if (slot < 0) continue;
    const int hk = is_k ? h - a.n_q : h - a.n_q - v.n_kv;
    const long long at = (slot * v.n_kv + hk) * v.D + sub * 8;
    void* pages = is_k ? a.k : a.vv;
    if (!a.scales) {
      uint16_t* dst = (uint16_t*)pages + at;
      *reinterpret_cast<uint4*>(dst) = pack(xa);
      *reinterpret_cast<uint4*>(dst + half) = pack(xb);
      continue;
    }
    const bool finite = top < 0x7f800000u;
    const float amax = __uint_as_float(top), scale = amax < 1e-34f ? 0.f : amax / 127.f;
    const float inv = finite && scale > 0.f ? 1.0f / scale : 0.f;
    auto quant = [&](const float (&f)[8]) {
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int q = finite ? max(-127, min(127, __float2int_rn(f[j] * inv))) : 0;
        w[j >> 2] |= (uint32_t)(uint8_t)q << (8 * (j & 3));
      }
      return make_uint2(w[0], w[1]);
    };
    int8_t* dst = (int8_t*)pages + at;
    *reinterpret_cast<uint2*>(dst) = quant(xa);
    *reinterpret_cast<uint2*>(dst + half) = quant(xb);
    if (sub == 0) a.scales[slot * 2 * v.n_kv + (is_k ? 0 : v.n_kv) + hk] = finite ? scale : __uint_as_float(0x7fc00000u);
  }
}

// k_out / v_out [rows][n_kv * D] bf16: the tokens' keys and values, int8 ones as bf16(integer * scale); zeros where a position holds
// nothing. A warp takes `per` rows, whose slots its lanes look up side by side; a lane then takes 16 values of a head at a time, and asks for
// four such pieces before it stores one.
template <bool I8>
__global__ void __launch_bounds__(256) kv_read_paged_kernel(const ReadPagedArgs a) {
  grid_dependency_wait();
  grid_dependency_release();
  const PagedView& v = a.v;
  const int lane = threadIdx.x & 31;
  const long long first = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * a.per;
  if (first >= v.rows) return;
  const int row0 = (int)first, n = min(a.per, v.rows - row0);
  const int own = row0 + min(lane, n - 1);
  const int seq = sequence_from(v, sequence_of_row(v, row0), own), pos = row_position(v, seq, own);
  const int own_slot = pos < 0 ? -2 : (int)slot_of(v, seq, pos);  // -2: a row of nobody; slots are below 2^31
  const int width = v.n_kv * v.D, pieces = width / 16, per_head = v.D / 16, row_pieces = 2 * pieces;
  int r = 0, c = lane;
  while (__any_sync(0xffffffffu, r < n)) {
    uint4 w[4][2];
    uint16_t* to[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      while (r < n && c >= row_pieces) c -= row_pieces, r++;
      const int slot = __shfl_sync(0xffffffffu, own_slot, r & 31);
      const bool is_v = c >= pieces;
      const int at = is_v ? c - pieces : c;
      to[i] = r < n && slot != -2 ? (is_v ? a.v_out : a.k_out) + (long long)(row0 + r) * width + at * 16 : nullptr;
      w[i][0] = w[i][1] = make_uint4(0, 0, 0, 0);
      if (to[i] && slot >= 0) {
        const long long from = (long long)slot * width + at * 16;
        const void* pages = is_v ? a.vv : a.k;
        if (!I8) {
          w[i][0] = __ldg(reinterpret_cast<const uint4*>((const uint16_t*)pages + from));
          w[i][1] = __ldg(reinterpret_cast<const uint4*>((const uint16_t*)pages + from) + 1);
        } else {
          w[i][0] = __ldg(reinterpret_cast<const uint4*>((const int8_t*)pages + from));
          w[i][1].x = __float_as_uint(__ldg(a.scales + (long long)slot * 2 * v.n_kv + (is_v ? v.n_kv : 0) + at / per_head));
        }
      }
      c += 32;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (!to[i]) continue;
      if (I8) {
        const float s = __uint_as_float(w[i][1].x);
        auto two = [&](uint32_t word, int j) {
          return pack_bf16((float)(int8_t)(word >> (8 * j)) * s, (float)(int8_t)(word >> (8 * j + 8)) * s);
        };
        const uint4 q = w[i][0];
        w[i][0] = make_uint4(two(q.x, 0), two(q.x, 2), two(q.y, 0), two(q.y, 2));
        w[i][1] = make_uint4(two(q.z, 0), two(q.z, 2), two(q.w, 0), two(q.w, 2));
      }
      reinterpret_cast<uint4*>(to[i])[0] = w[i][0];
      reinterpret_cast<uint4*>(to[i])[1] = w[i][1];
    }
  }
}

}  // namespace

cudaError_t launch_rope_kv_paged(RopePagedArgs a, cudaStream_t stream) {
  const int heads = a.n_q + 2 * a.v.n_kv;
  int lanes = 1;
  while (lanes < a.v.D / 16) lanes *= 2;
  // One head to a group until the machine has 32 warps an SM: a single token's heads then run beside one another; more rows share the work on
  // their angles over up to eight heads.
  const long long enough = 32ll * current_sm_count() * (32 / lanes);
  a.per = 1;
  while (a.per < 8 && a.per < heads && (long long)a.v.rows * heads / (2 * a.per) >= enough) a.per *= 2;
  const long long items = (long long)a.v.rows * ((heads + a.per - 1) / a.per);
  auto run = [&](auto kernel) {
    const int per_block = 256 / lanes;
    return launch_dependent(kernel, dim3((unsigned)((items + per_block - 1) / per_block)), dim3(256), 0, stream, a);
  };
  switch (lanes) {
    case 1: return run(rope_kv_paged_kernel<1>);
    case 2: return run(rope_kv_paged_kernel<2>);
    case 4: return run(rope_kv_paged_kernel<4>);
    case 8: return run(rope_kv_paged_kernel<8>);
    default: return run(rope_kv_paged_kernel<16>);
  }
}

cudaError_t launch_kv_read_paged(ReadPagedArgs a, cudaStream_t stream) {
  a.per = (int)std::min(8ll, std::max(1ll, a.v.rows / (16ll * current_sm_count())));  // rows a warp, once there are 16 warps an SM
  const dim3 grid((unsigned)((a.v.rows + 8ll * a.per - 1) / (8ll * a.per)));
  return a.scales ? launch_dependent(kv_read_paged_kernel<true>, grid, dim3(256), 0, stream, a)
                  : launch_dependent(kv_read_paged_kernel<false>, grid, dim3(256), 0, stream, a);
}

}  // namespace tb200
