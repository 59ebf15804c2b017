// Writing a chunk's keys and values into a paged cache, and reading tokens back (paged.cuh says how the cache is laid out).
#include <algorithm>

#include "dependent_launch.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "widen.cuh"

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
// What bounds it: memory, once its instructions are few enough (an int8 cache and norms take the most of them). L lanes hold a head (L the
// power of two from D / 16 on), eight neighbouring values of each half to a lane, so that every access has 16 bytes. A warp takes the same
// `per` heads of 32 / L rows one after another: its branches are then the same for all lanes, a row's angles and the norm's weights are
// fetched once for several heads, and four heads are on their way while one is worked on (one ahead: 28.7 us against 22.7 for 16384 rows of 4/1 heads
// of 256 into bf16, 101 MB; 4001 rows of 32/8 heads of 128 with norms into int8, 90 MB, take 29 us, at 66 % of the issue slots).
constexpr int kAhead = 4;
template <int L>
__global__ void __launch_bounds__(128) rope_kv_paged_kernel(const RopePagedArgs a) {
  const PagedView& v = a.v;
  const int lane = threadIdx.x & 31, sub = lane % L, half = v.D >> 1;
  const bool active = sub * 8 < half;
  grid_dependency_wait();
  grid_dependency_release();
  const int heads = a.n_q + 2 * v.n_kv, groups = (heads + a.per - 1) / a.per;
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 5), first = unit / groups * (32 / L);
  if (first >= v.rows) return;
  const int h0 = (int)(unit % groups) * a.per, h1 = min(h0 + a.per, heads);
  const int row = (int)first + lane / L;
  const uint16_t* const src = a.qkv + (long long)row * heads * v.D + sub * 8;
  // heads on their way: a lane's pieces land in places of its own, so only its own copies are waited for
  __shared__ uint4 ring[kAhead][2][128];
  const bool reads = active && row < v.rows;
  auto ask = [&](int h) {
    if (h < h1) {
      const uint16_t* const from = reads ? src + h * v.D : a.qkv;
      const uint32_t to = (uint32_t)__cvta_generic_to_shared(&ring[(h - h0) % kAhead][0][threadIdx.x]);
      copy16(to, from, reads);
      copy16(to + sizeof(ring[0][0]), reads ? from + half : from, reads);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kAhead; i++) ask(h0 + i);
  const int seq = sequence_from(v, sequence_of_row(v, (int)first), min(row, v.rows - 1));
  const int pos = row < v.rows ? row_position(v, seq, row) : -1;
  const long long slot = pos >= 0 ? slot_of(v, seq, pos) : -1;
  const bool on = active && pos >= 0;
  float cs[8], sn[8];
  if (h0 < a.n_q + v.n_kv) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int top = active ? (int)(((unsigned long long)(unsigned)max(pos, 0) * __ldg(a.turns + sub * 8 + j)) >> 32) : 0;
      sincospif((float)top * 4.6566128730773926e-10f, &sn[j], &cs[j]);  // 2^-31: a turn is 2 in units of pi
    }
  }
  uint4 w_a = make_uint4(0, 0, 0, 0), w_b = w_a;  // the norm's weights
  for (int h = h0; h < h1; h++) {
    const bool is_q = h < a.n_q, is_k = !is_q && h < a.n_q + v.n_kv;
    float xa[8], xb[8];
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    unpack(ring[(h - h0) % kAhead][0][threadIdx.x], xa);
    unpack(ring[(h - h0) % kAhead][1][threadIdx.x], xb);
    ask(h + kAhead);
    if (is_q || is_k) {
      if (a.norms) {
        if (active && (h == h0 || h == a.n_q)) {
          const uint16_t* w = a.norms + (is_q ? 0 : v.D) + sub * 8;
          w_a = __ldg(reinterpret_cast<const uint4*>(w));
          w_b = __ldg(reinterpret_cast<const uint4*>(w + half));
        }
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) ss += xa[j] * xa[j] + xb[j] * xb[j];
        ss = group_sum<L>(ss);
        const float inv = rsqrtf(ss / (float)v.D + a.eps);
        float wa[8], wb[8];
        unpack(w_a, wa);
        unpack(w_b, wb);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          xa[j] = xa[j] * inv * (1.0f + wa[j]);
          xb[j] = xb[j] * inv * (1.0f + wb[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float p = xa[j], q = xb[j];
        xa[j] = p * cs[j] - q * sn[j];
        xb[j] = q * cs[j] + p * sn[j];
      }
    }
    if (is_q) {
      if (!on) continue;
      uint16_t* dst = a.q_out + ((long long)row * a.n_q + h) * v.D + sub * 8;
      *reinterpret_cast<uint4*>(dst) = pack(xa);
      *reinterpret_cast<uint4*>(dst + half) = pack(xb);
      continue;
    }
    const int hk = is_k ? h - a.n_q : h - a.n_q - v.n_kv;
    const long long at = (slot * v.n_kv + hk) * v.D + sub * 8;
    void* pages = is_k ? a.k : a.vv;
    if (!a.scales) {
      if (!on || slot < 0) continue;
      uint16_t* dst = (uint16_t*)pages + at;
      *reinterpret_cast<uint4*>(dst) = pack(xa);
      *reinterpret_cast<uint4*>(dst + half) = pack(xb);
      continue;
    }
    uint32_t top = 0;  // bits of the largest magnitude; those of a NaN are above an infinity's, and these above every number's
    if (on) {
#pragma unroll
      for (int j = 0; j < 8; j++) top = max(top, max(__float_as_uint(fabsf(xa[j])), __float_as_uint(fabsf(xb[j]))));
    }
    top = group_max<L>(top);
    if (!on || slot < 0) continue;
    const bool finite = top < 0x7f800000u;
    const float amax = __uint_as_float(top), scale = amax < 1e-34f ? 0.f : amax / 127.f;
    const float inv = finite && scale > 0.f ? 1.0f / scale : 0.f;
    // Nearest integers by an addition: 1.5 * 2^23 + n has n in its low byte. |x| inv is at most 127 (1 + 2^-22), which rounds to 127.
    auto quant = [&](const float (&f)[8]) {
      uint32_t b[8];
#pragma unroll
      for (int j = 0; j < 8; j++) b[j] = __float_as_uint(fmaf(finite ? f[j] : 0.f, inv, 12582912.0f));
      return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                        __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
    };
    int8_t* dst = (int8_t*)pages + at;
    *reinterpret_cast<uint2*>(dst) = quant(xa);
    *reinterpret_cast<uint2*>(dst + half) = quant(xb);
    if (sub == 0) a.scales[slot * 2 * v.n_kv + (is_k ? 0 : v.n_kv) + hk] = finite ? scale : __uint_as_float(0x7fc00000u);
  }
}

// k_out / v_out [rows][n_kv * D] bf16: the tokens' keys and values, int8 ones as bf16(integer * scale); zeros where a position holds
// nothing. A warp takes `per` rows, whose slots its lanes look up side by side; a lane then takes 16 values of a head at a time, and asks for
// four such pieces before it stores one. 20011 rows of a head of 256 from int8 (31 MB) take 12.3 us, of which 4.6 are any call's: the reads of
// a row's sequence, context and page stand in front of its values.
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
  // One head to a warp until the machine has 24 warps an SM: a single token's heads then run beside one another; more rows share the work on
  // their angles over up to eight heads.
  const int rows = 32 / lanes;
  const long long row_groups = (a.v.rows + rows - 1) / rows;
  a.per = 1;
  while (a.per < 8 && a.per < heads && row_groups * heads / (2 * a.per) >= 24ll * current_sm_count()) a.per *= 2;
  const long long warps = row_groups * ((heads + a.per - 1) / a.per);
  auto run = [&](auto kernel) { return launch_dependent(kernel, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, stream, a); };
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
