// attn_paged: which kernel takes which rows, the kernel for sequences of few rows (a decode step), and the launch that joins what several
// blocks have done of one tile. paged.h says how the work is cut, paged_attn_tc.cu has the kernel for many rows.
//
// Few rows (new tokens times query heads of a key/value head, at most 16): what bounds it is the cache's way from HBM, so every SM has its share
// of all keys in flight. A tile is up to 8 or 16 rows; each of a block's four warps takes 16 keys of it at a time, by itself: copies into a ring of
// its own, S^T = K Q^T (keys are the 16-row operand of mma.sync m16n8k16, rows the 8-column one), its own running maximum, O^T += V^T P^T. What
// is a column of S^T is a column of O^T, so a thread keeps the same two rows throughout; P^T changes its layout by movmatrix and enters in two
// bf16 terms (2^-17 of it is lost). int8 caches are widened in registers: keys 16 bytes to a thread, the order of the dims inside a step being
// free as long as the queries follow it; values 2 bytes a tile of 16 dims, dims 8 apart in steps of D / 8. Warps meet in shared memory, in their
// order. Tiles that several blocks share are joined by the launch behind. With it, from memory: one token behind 1024 (4/1 heads of 256) 17 us, 32
// sequences of up to 8000 tokens (32/8 heads of 128, int8) 86 us, at 52 % of the issue slots.
#include <algorithm>

#include "dependent_launch.cuh"
#include "kernels.h"
#include "paged_row.cuh"
#include "paged_work.cuh"

namespace tb200 {

namespace {

constexpr int kFewWarps = 4, kFewThreads = kFewWarps * 32, kChunk = 16;  // keys a warp takes at a time
constexpr int kFewRows = 16;                                               // rows that a tile's partial sums have room for

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {  // an 8 x 8 tile of 16-bit values, two of a row to a thread
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma_16x8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// How a head of D dims lies in shared memory: dims in steps of 16 (int8: keys in groups of 64, values in groups of 32, what is behind D being
// finite and unused), rows apart so that no bank is hit twice.
struct FewShape {
  int k_pitch, v_pitch, q_pitch, stages, smem, ring;
};
TB200_BOTH FewShape few_shape(int D, bool i8, int stages) {
  FewShape s;
  if (i8) {
    s.k_pitch = (D + 63) / 64 * 64;
    s.k_pitch += s.k_pitch % 128 == 0 ? 64 : 0;   // 64 modulo 128
    s.v_pitch = (D + 127) / 128 * 128 + 16;       // 16 modulo 128
  } else {
    s.k_pitch = s.v_pitch = (2 * D + 127) / 128 * 128 + 16;
  }
  s.q_pitch = ((D + 63) / 64 * 64) * 2 + 16;
  s.stages = stages;
  s.ring = kFewWarps * stages * kChunk * (s.k_pitch + s.v_pitch);  // 39936 at least, more than RowsScratch
  const int meet = kFewWarps * kFewRows * D * 4;  // the warps' sums take the rings' place
  s.ring = s.ring > meet ? s.ring : meet;
  s.ring = (s.ring + 15) / 16 * 16;
  s.smem = s.ring + kFewRows * s.q_pitch + kFewWarps * stages * kChunk * 8 + kFewWarps * kFewRows * 8;
  return s;
}

// NT: steps of 16 dims a head has at most. RT: groups of 8 rows of a tile.
template <int NT, int RT, int STAGES, bool I8>
__global__ void __launch_bounds__(kFewThreads) attn_paged_few_kernel(const __grid_constant__ AttnPagedArgs a) {
  extern __shared__ __align__(16) unsigned char sm[];
  __shared__ WorkShared shared;
  __shared__ uint32_t held_bits[kFewWarps][STAGES], bad;
  const PagedView& v = a.v;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tig = lane & 3;
  const int D = v.D, group = a.n_q / v.n_kv, steps = D >> 4;
  const FewShape sh = few_shape(D, I8, STAGES);
  unsigned char* const ring = sm + warp * (STAGES * kChunk * (sh.k_pitch + sh.v_pitch));
  unsigned char* const qs = sm + sh.ring;
  float2* const scales = reinterpret_cast<float2*>(qs + kFewRows * sh.q_pitch) + warp * STAGES * kChunk;  // of a chunk's keys and values
  float2* const meet = reinterpret_cast<float2*>(qs + kFewRows * sh.q_pitch) + kFewWarps * STAGES * kChunk;  // (base, sum) of every warp's rows
  grid_dependency_wait();
  grid_dependency_release();
  if (tid == 0) {
    a.joins[blockIdx.x].parts = 0;
    bad = 0;
  }
  const Work work = share_out<kFewThreads>(a, shared, reinterpret_cast<int*>(sm));
  __syncthreads();
  if (!work.works) return;
  const float cexp = a.scale * 1.4426950408889634f;
  const int row_bytes = D * (I8 ? 1 : 2), pieces = row_bytes >> 4;
  const unsigned slot_bytes = (unsigned)v.n_kv * row_bytes;
  const int lane_key = page_of(lane, a.piece_div), lane_piece = lane - lane_key * pieces, step_keys = page_of(32, a.piece_div), step_pieces = 32 - step_keys * pieces;
  ItemCursor cursor(a, work, shared);
  Item w;
  while (cursor.take(a, work, w)) {
    const int used = w.tokens * group;
    // queries, rows behind the last and dims behind D as zeros
    for (int i = tid; i < kFewRows * ((D + 63) / 64 * 8); i += kFewThreads) {
      const int r = i / ((D + 63) / 64 * 8), c = i - r * ((D + 63) / 64 * 8), tok = page_of(r, a.group_div);
      uint4 x = make_uint4(0, 0, 0, 0);
      if (r < used && c * 8 < D)
        x = __ldg(reinterpret_cast<const uint4*>(a.q + ((long long)(w.row0 + tok) * a.n_q + w.head * group + r - tok * group) * D) + c);
      *reinterpret_cast<uint4*>(qs + r * sh.q_pitch + c * 16) = x;
    }
    // chunks of 16 keys, by turns to the warps; those that no row sees are passed over
    const Keys keys(a, w);
    const int n_chunks = (w.b1 - w.b0) * (kKeyBlock / kChunk);
    static_assert(kSpanAlign % kChunk == 0, "a chunk's keys lie one behind another");
    auto key_of = [&](int ci) { return keys.at(w.b0 * kKeyBlock + ci * kChunk); };
    auto next_chunk = [&](int ci) {
      for (; ci < n_chunks; ci += kFewWarps) {
        const int k = key_of(ci);
        if (k < keys.end_key && (k + kChunk > keys.near_key || k < keys.sinks)) break;
      }
      return ci;
    };
    int asked = next_chunk(warp), asked_page = 0;  // the chunk whose page ids are on their way: one key to a lane
    auto ask = [&]() {
      if (asked < n_chunks) asked_page = keys.ask(key_of(asked) + (lane & 15));
    };
    int filled = 0;
    auto fill = [&]() {  // copies the chunk that was asked for into the next stage, and asks for the one behind it
      if (asked < n_chunks) {
        const int stage = filled % STAGES, slot = keys.slot(key_of(asked) + (lane & 15), asked_page);
        unsigned char* const kd = ring + stage * kChunk * (sh.k_pitch + sh.v_pitch);
        unsigned char* const vd = kd + kChunk * sh.k_pitch;
        const long long head_bytes = (long long)w.head * row_bytes;
        if (I8 && lane < kChunk) {
          const float* sc = a.scales + (long long)max(slot, 0) * 2 * v.n_kv + w.head;
          const uint32_t to = smem_at(scales + stage * kChunk + lane);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(sc), "r"(slot >= 0 ? 4 : 0) : "memory");
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + 4), "l"(sc + v.n_kv), "r"(slot >= 0 ? 4 : 0) : "memory");
        }
        const unsigned held = __ballot_sync(0xffffffffu, slot >= 0);  // the keys twice over
        if (lane == 0) held_bits[warp][stage] = held;
        // piece by piece, 32 at a time: a lane steps from (key, piece) to the one 32 further on
        int key = lane_key, c = lane_piece;
        uint32_t k_to = smem_at(kd + key * sh.k_pitch + c * 16), v_to = smem_at(vd + key * sh.v_pitch + c * 16);
        const char* const k_from = (const char*)a.k + head_bytes;
        const char* const v_from = (const char*)a.vv + head_bytes;
#pragma unroll 2
        for (int p0 = 0; p0 < kChunk * pieces; p0 += 32) {  // (every lane shuffles in every turn: 16 keys' pieces need not be a multiple of 32)
          const int s = __shfl_sync(0xffffffffu, slot, key & 15);
          if (key < kChunk) {
            const unsigned long long from = (unsigned long long)(unsigned)max(s, 0) * slot_bytes + (unsigned)(c * 16);
            copy16(k_to, k_from + from, s >= 0);
            copy16(v_to, v_from + from, s >= 0);
          }
          key += step_keys;
          c += step_pieces;
          k_to += step_keys * sh.k_pitch + step_pieces * 16;
          v_to += step_keys * sh.v_pitch + step_pieces * 16;
          if (c >= pieces) {
            c -= pieces;
            key++;
            k_to += sh.k_pitch - pieces * 16;
            v_to += sh.v_pitch - pieces * 16;
          }
        }
        asked = next_chunk(asked + kFewWarps);
        ask();
      }
      filled++;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    ask();
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; i++) fill();
    __syncthreads();  // the queries are there

    // this thread's rows, 2 tig and 2 tig + 1 of each group of 8
    int pos[RT][2], near[RT][2];
    float m[RT][2], base[RT][2], sum[RT][2];  // m: from where on a score moves base, the scaled score that exponents are taken from
    const int last_near = a.window ? max(0, (int)min((long long)w.first_pos + w.tokens - 1, 0x7fffffffll) - a.window + 1) : 0;
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int tok = min(page_of(8 * t + 2 * tig + j, a.group_div), w.tokens - 1);
        pos[t][j] = (int)min((long long)w.first_pos + tok, 0x7fffffffll);
        near[t][j] = a.window ? max(0, pos[t][j] - a.window + 1) : 0;
        m[t][j] = -INFINITY;
        base[t][j] = sum[t][j] = 0.f;
      }
    float o[NT][RT][4];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[i][t][j] = 0.f;

    int done = 0;
    for (int ci = next_chunk(warp); ci < n_chunks; ci = next_chunk(ci + kFewWarps), done++) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncwarp();
      const int stage = done % STAGES, key0 = key_of(ci);
      unsigned char* const kd = ring + stage * kChunk * (sh.k_pitch + sh.v_pitch);
      unsigned char* const vd = kd + kChunk * sh.k_pitch;
      float s[RT][4];
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[t][j] = 0.f;
      if (!I8) {
        const uint32_t k_at = smem_at(kd + (lane & 15) * sh.k_pitch + (lane >> 4) * 16);
        const uint32_t q_at = smem_at(qs + (lane & 7) * sh.q_pitch + (lane >> 3) * 16);
#pragma unroll
        for (int i = 0; i < NT; i += 2) {
          if (i >= steps) continue;
          uint32_t ka[4], kb[4];
          ldsm4(ka, k_at + i * 32);
          if (i + 1 < steps) ldsm4(kb, k_at + i * 32 + 32);
#pragma unroll
          for (int t = 0; t < RT; t++) {
            uint32_t q[4];
            ldsm4(q, q_at + t * 8 * sh.q_pitch + i * 32);
            mma_16x8(s[t], ka[0], ka[1], ka[2], ka[3], q[0], q[1]);
            if (i + 1 < steps) mma_16x8(s[t], kb[0], kb[1], kb[2], kb[3], q[2], q[3]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < (NT + 3) / 4; i++) {  // 64 dims: this thread's 16 of them, of keys g and g + 8
          if (i * 4 >= steps) continue;
          const uint4 lo = *reinterpret_cast<const uint4*>(kd + g * sh.k_pitch + i * 64 + tig * 16);
          const uint4 hi = *reinterpret_cast<const uint4*>(kd + (g + 8) * sh.k_pitch + i * 64 + tig * 16);
          const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            uint32_t a0[2], a1[2], a2[2], a3[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
              widen4(wl[j + k], a0[k], a2[k]);
              widen4(wh[j + k], a1[k], a3[k]);
            }
#pragma unroll
            for (int t = 0; t < RT; t++) {
              const uint4 q = *reinterpret_cast<const uint4*>(qs + (8 * t + g) * sh.q_pitch + (i * 64 + tig * 16 + j * 4) * 2);
              mma_16x8(s[t], a0[0], a1[0], a2[0], a3[0], q.x, q.y);
              mma_16x8(s[t], a0[1], a1[1], a2[1], a3[1], q.z, q.w);
            }
          }
        }
      }
      // s[t][0], [1]: key g, rows 2 tig, 2 tig + 1; s[t][2], [3]: key g + 8
      float2 sc[2] = {make_float2(1.f, 1.f), make_float2(1.f, 1.f)};
      if (I8) {
        sc[0] = scales[stage * kChunk + g];
        sc[1] = scales[stage * kChunk + g + 8];
      }
      // x = scores in units of log2; keys that a row does not see at -inf. Only chunks at an edge of what the tile sees need looking at key by key.
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          s[t][j] *= sc[0].x;
          s[t][2 + j] *= sc[1].x;
        }
      const bool edge = held_bits[warp][stage] != 0xffffffffu || key0 + kChunk - 1 > w.first_pos || (key0 < last_near && key0 + kChunk > a.sinks);
      if (edge) {
        const bool held_a = held_bits[warp][stage] >> g & 1, held_b = held_bits[warp][stage] >> (g + 8) & 1;
        const int ka = key0 + g, kb = ka + 8;
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
          for (int j = 0; j < 2; j++) {
            if (!(held_a && ka <= pos[t][j] && (ka >= near[t][j] || ka < a.sinks))) s[t][j] = -INFINITY;
            if (!(held_b && kb <= pos[t][j] && (kb >= near[t][j] || kb < a.sinks))) s[t][2 + j] = -INFINITY;
          }
      }
      // m follows a row's maximum only where a weight would grow beyond 2^8 (or is the row's first): a bound serves as well, and costs no shuffles
      bool grows = false;
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int j = 0; j < 2; j++) grows = grows || fmaxf(s[t][j], s[t][2 + j]) > m[t][j];
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int t = 0; t < RT; t++) {
          float keep[2];
#pragma unroll
          for (int j = 0; j < 2; j++) {
            float top = fmaxf(s[t][j], s[t][2 + j]);
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            keep[j] = 1.f;
            if (top > m[t][j]) {
              const float to = top * cexp;
              keep[j] = m[t][j] == -INFINITY ? 0.f : exp2_fast(base[t][j] - to);
              base[t][j] = to;
              m[t][j] = top + 8.f / cexp;
              sum[t][j] *= keep[j];
            }
          }
#pragma unroll
          for (int i = 0; i < NT; i++) {
            o[i][t][0] *= keep[0]; o[i][t][1] *= keep[1];
            o[i][t][2] *= keep[0]; o[i][t][3] *= keep[1];
          }
        }
      }
      uint32_t p_hi[RT][2], p_lo[RT][2];
#pragma unroll
      for (int t = 0; t < RT; t++) {
#pragma unroll
        for (int j = 0; j < 2; j++) {  // (a row without a key has base 0 and scores of -inf: weights of zero)
          const float x = exp2_fast(fmaf(s[t][j], cexp, -base[t][j])), y = exp2_fast(fmaf(s[t][2 + j], cexp, -base[t][j]));
          sum[t][j] += x + y;
          s[t][j] = I8 ? (x == 0.f ? 0.f : x * sc[0].y) : x;
          s[t][2 + j] = I8 ? (y == 0.f ? 0.f : y * sc[1].y) : y;
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint32_t hi = pack_bf16(s[t][2 * h], s[t][2 * h + 1]);
          const uint32_t lo = pack_bf16(s[t][2 * h] - __uint_as_float(hi << 16), s[t][2 * h + 1] - __uint_as_float(hi & 0xffff0000u));
          p_hi[t][h] = transpose8(hi);
          p_lo[t][h] = transpose8(lo);
        }
      }
      if (!I8) {
        const uint32_t v_at = smem_at(vd + ((lane & 7) + (lane >> 4) * 8) * sh.v_pitch + ((lane >> 3) & 1) * 16);
#pragma unroll
        for (int i = 0; i < NT; i++) {
          if (i >= steps) continue;
          uint32_t va[4];
          ldsm4_trans(va, v_at + i * 32);
#pragma unroll
          for (int t = 0; t < RT; t++) {
            mma_16x8(o[i][t], va[0], va[1], va[2], va[3], p_hi[t][0], p_hi[t][1]);
            mma_16x8(o[i][t], va[0], va[1], va[2], va[3], p_lo[t][0], p_lo[t][1]);
          }
        }
      } else {
        // dim D' / 8 * g + j (D' = D rounded up to 32) of keys 2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9, four j at a time: tiles 2 i, 2 i + 1 of 16 dims
        const int per = (D + 31) / 32 * 4;
        const unsigned char* const from = vd + 2 * tig * sh.v_pitch + g * per;
        auto four = [&](int i, const uint32_t (&x)[4]) {
          uint32_t a0, a1, a2, a3, b0, b1, b2, b3;
          widen4(__byte_perm(x[0], x[1], 0x5140), a0, a1);  // two keys' bytes side by side, then widened
          widen4(__byte_perm(x[0], x[1], 0x7362), b0, b1);
          widen4(__byte_perm(x[2], x[3], 0x5140), a2, a3);
          widen4(__byte_perm(x[2], x[3], 0x7362), b2, b3);
#pragma unroll
          for (int t = 0; t < RT; t++) {
            mma_16x8(o[2 * i][t], a0, a1, a2, a3, p_hi[t][0], p_hi[t][1]);
            mma_16x8(o[2 * i][t], a0, a1, a2, a3, p_lo[t][0], p_lo[t][1]);
            mma_16x8(o[2 * i + 1][t], b0, b1, b2, b3, p_hi[t][0], p_hi[t][1]);
            mma_16x8(o[2 * i + 1][t], b0, b1, b2, b3, p_lo[t][0], p_lo[t][1]);
          }
        };
        if (NT >= 8 && per % 16 == 0) {  // 16 bytes of a key at once
#pragma unroll
          for (int i = 0; i < NT / 2; i += 4) {
            if (4 * i >= per) continue;
            uint4 y[4];
#pragma unroll
            for (int k = 0; k < 4; k++) y[k] = *reinterpret_cast<const uint4*>(from + ((k & 1) + (k >> 1) * 8) * sh.v_pitch + 4 * i);
            four(i, {y[0].x, y[1].x, y[2].x, y[3].x});
            four(i + 1, {y[0].y, y[1].y, y[2].y, y[3].y});
            four(i + 2, {y[0].z, y[1].z, y[2].z, y[3].z});
            four(i + 3, {y[0].w, y[1].w, y[2].w, y[3].w});
          }
        } else {
#pragma unroll
          for (int i = 0; i < NT / 2; i++) {
            if (4 * i >= per) continue;
            uint32_t x[4];
#pragma unroll
            for (int k = 0; k < 4; k++) x[k] = *reinterpret_cast<const uint32_t*>(from + ((k & 1) + (k >> 1) * 8) * sh.v_pitch + 4 * i);
            four(i, x);
          }
        }
      }
      __syncwarp();
      fill();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // every warp is through with its ring
    // [warp][row][D], and (base, sum) of every warp's rows
    float* const parts = reinterpret_cast<float*>(sm);
#pragma unroll
    for (int t = 0; t < RT; t++) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) sum[t][j] += __shfl_xor_sync(0xffffffffu, sum[t][j], off);
        const int row = 8 * t + 2 * tig + j;
        if (g == 0) meet[warp * kFewRows + row] = make_float2(m[t][j] == -INFINITY ? m[t][j] : base[t][j], sum[t][j]);
        if (row < used) {
          float* const to = parts + (warp * kFewRows + row) * D;
          const int per = (D + 31) / 32 * 4;
#pragma unroll
          for (int i = 0; i < NT; i++) {
            const int d = I8 ? per * g + 2 * i : 16 * i + g, d2 = I8 ? d + 1 : d + 8;
            const bool in = I8 ? 2 * i < per : i < steps;
            if (in && d < D) to[d] = o[i][t][j];
            if (in && d2 < D) to[d2] = o[i][t][2 + j];
          }
        }
      }
    }
    __syncthreads();
    const bool whole = w.b1 - w.b0 == w.blocks;
    const int here = (int)blockIdx.x, first = whole ? here : work_owner(w.w0, work.total, work.parts);
    float* const to = a.partial + (long long)attn_part(here, here == first && work.begin < w.w0) * attn_part_floats(D, kFewRows);
    for (int i = tid; i < used * (D >> 2); i += kFewThreads) {  // four dims of a row, the warps in their order
      const int row = i / (D >> 2), q = i - row * (D >> 2);
      float top = -INFINITY, all = 0.f;
#pragma unroll
      for (int k = 0; k < kFewWarps; k++) top = fmaxf(top, meet[k * kFewRows + row].x);
      const float from = top == -INFINITY ? 0.f : top;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kFewWarps; k++) {
        const float2 ml = meet[k * kFewRows + row];
        if (ml.x == -INFINITY) continue;  // the warp saw no key of this row
        const float f = exp2_fast(ml.x - from);
        const float4 y = *reinterpret_cast<const float4*>(parts + (k * kFewRows + row) * D + q * 4);
        all += f * ml.y;
        x.x += f * y.x; x.y += f * y.y; x.z += f * y.z; x.w += f * y.w;
      }
      if (!whole) {
        reinterpret_cast<float4*>(to)[q * kFewRows + row] = x;
        if (q == 0) *reinterpret_cast<float2*>(to + D * kFewRows + row * 2) = make_float2(top, all);
        continue;
      }
      const float inv = all > 0.f ? 1.f / all : (all == 0.f ? 0.f : all);  // no weights: no key seen, or none with a score above -inf
      x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv;
      if (!(fabsf(x.x) <= 3.0e38f && fabsf(x.y) <= 3.0e38f && fabsf(x.z) <= 3.0e38f && fabsf(x.w) <= 3.0e38f) || all == 0.f)
        atomicOr(&bad, 1u << row);
      const int tok = page_of(row, a.group_div);
      *reinterpret_cast<uint2*>(a.out + ((long long)(w.row0 + tok) * a.n_q + w.head * group + row - tok * group) * D + q * 4) =
          make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
    }
    if (!whole && tid == 0 && here == first) write_join(a, work, w, first, used);
    __syncthreads();  // the rings are free again
    const uint32_t again = bad;
    if (again) {  // rare: an infinity or a NaN among the values, a row without a key (the rings have room for the scratch at every head size)
      attend_rows<kFewThreads>(a, *reinterpret_cast<RowsScratch<kFewThreads>*>(sm), tid, {w.row0, w.head, w.seq, w.first_pos}, 0, again, 0, D, [] { __syncthreads(); });
      if (tid == 0) bad = 0;
    }
  }
}

// Adds up the parts of the tiles that several blocks shared, in their order. A block has 32 rows of a tile of many rows, so that all of them run at
// once (of 16 rows, in 2.7 goes: 15.0 us instead of 10.7 for heads of 64, 19.6 instead of 16.6 for heads of 256, by the profiler), or the rows
// and 64 dims of a tile of few rows. What bounds it is the chain of reads (which tile, the parts' maxima, the parts), and how many loads of
// parts are under way at once: where rows are few the parts are spread over the threads that this leaves.
constexpr int kJoinRows = 32, kJoinDims = 64, kJoinThreads = 256, kJoinAhead = 3;
struct JoinSet {
  const float* partial;
  const AttnJoin* joins;
  int count, pitch;  // blocks that may have begun a shared tile; rows that partial sums have room for
  int join_rows;     // rows a block of the join takes
};
__global__ void __launch_bounds__(kJoinThreads, 4) attn_paged_join_kernel(const __grid_constant__ AttnPagedArgs a, const JoinSet many, const JoinSet few) {
  extern __shared__ __align__(16) unsigned char join_sm[];
  __shared__ float4 meet[kJoinThreads];
  __shared__ float invs[kJoinRows];
  __shared__ uint32_t bad;
  grid_dependency_wait();
  grid_dependency_release();
  constexpr int kChunks = 128 / kJoinRows;
  const bool is_many = (int)blockIdx.x < many.count * kChunks;
  const JoinSet set = is_many ? many : few;
  // tiles of many rows: 32 of them to a block, all dims one after another; tiles of few rows: 64 dims to a block
  const int rest = (int)blockIdx.x - many.count * kChunks, dim_blocks = (a.v.D + kJoinDims - 1) / kJoinDims;
  const int at = is_many ? blockIdx.x / kChunks : rest / dim_blocks, r0 = is_many ? blockIdx.x % kChunks * kJoinRows : 0;
  const int first_dim = is_many ? 0 : rest % dim_blocks * kJoinDims, end_dim = is_many ? a.v.D : min(a.v.D, first_dim + kJoinDims);
  const AttnJoin j = set.joins[at];
  const int pitch = set.join_rows, rows = min(pitch, j.used - r0);
  if (!j.parts || rows <= 0) return;
  const int tid = threadIdx.x, D = a.v.D, group = a.n_q / a.v.n_kv;
  float2* const ml = reinterpret_cast<float2*>(join_sm);  // [part][rows]: (base, sum), then (factor, -)
  auto part = [&](int f) { return set.partial + (long long)attn_part(j.first + f, f == 0 && j.second_place) * attn_part_floats(D, set.pitch); };
  if (tid == 0) bad = 0;
  // Tiles of many rows: a thread has four dims of every 64 of two rows (of a warp's lanes eight rows lie side by side, whose partial sums are
  // 128 bytes, and 16 dims, which the result has in 32). The first 64 are asked for before the rows' factors are known.
  const int many_r = (tid & 7) | (tid >> 2 & 8), many_q = (tid >> 3 & 3) | (tid >> 4 & 12);
  float4 x[2][kJoinAhead];
  auto ask = [&](int d) {
#pragma unroll
    for (int c = 0; c < 2; c++) {
#pragma unroll
      for (int f = 0; f < kJoinAhead; f++)
        x[c][f] = many_r + 16 * c < rows && d < D && f < j.parts ? __ldcg(reinterpret_cast<const float4*>(part(f)) + d / 4 * set.pitch + r0 + many_r + 16 * c)
                                                                 : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  if (is_many) ask(many_q * 4);
#pragma unroll 4
  for (int i = tid; i < j.parts * pitch; i += kJoinThreads) {  // (a power of two)
    const int f = i >> (31 - __clz(pitch)), r = i & (pitch - 1);
    ml[i] = r < rows ? __ldcg(reinterpret_cast<const float2*>(part(f) + D * set.pitch + (r0 + r) * 2)) : make_float2(-INFINITY, 0.f);
  }
  __syncthreads();
  {  // eight threads to a row: its maximum, and the sum against it
    const int r = tid >> 3, sub = tid & 7, parts = r < pitch ? j.parts : 0;
    float top = -INFINITY, sum = 0.f;
    for (int f = sub; f < parts; f += 8) top = fmaxf(top, ml[f * pitch + r].x);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float from = top == -INFINITY ? 0.f : top;
    for (int f = sub; f < parts; f += 8) {
      float2& x = ml[f * pitch + r];
      x.x = x.x == -INFINITY ? 0.f : exp2_fast(x.x - from);
      sum += x.x == 0.f ? 0.f : x.x * x.y;
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (sub == 0) {
      invs[r] = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
      if (r < rows && sum == 0.f) atomicOr(&bad, 1u << r);
    }
  }
  __syncthreads();
  auto add = [](float4& o, float y, const float4& x) {
    if (y == 0.f) return;  // that part saw no key of this row
    o.x += y * x.x; o.y += y * x.y; o.z += y * x.z; o.w += y * x.w;
  };
  auto store = [&](int r, int d, float4 o) {
    const float inv = invs[r];
    o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
    if (!(fabsf(o.x) <= 3.0e38f && fabsf(o.y) <= 3.0e38f && fabsf(o.z) <= 3.0e38f && fabsf(o.w) <= 3.0e38f)) atomicOr(&bad, 1u << r);
    const int tok = page_of(r0 + r, a.group_div);
    *reinterpret_cast<uint2*>(a.out + ((long long)(j.row0 + tok) * a.n_q + j.head * group + r0 + r - tok * group) * D + d) =
        make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
  };
  if (is_many) {
    for (int d = many_q * 4; d < D; d += kJoinDims) {
      if (d >= kJoinDims) ask(d);
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const int r = many_r + 16 * c;
        if (r >= rows) continue;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int f = 0; f < kJoinAhead; f++)
          if (f < j.parts) add(o, ml[f * pitch + r].x, x[c][f]);
#pragma unroll 4
        for (int f = kJoinAhead; f < j.parts; f++) add(o, ml[f * pitch + r].x, __ldcg(reinterpret_cast<const float4*>(part(f)) + d / 4 * set.pitch + r0 + r));
        store(r, d, o);
      }
    }
  } else {
    int span = 1;  // a power of two that holds the rows
    while (span < rows) span *= 2;
    const int groups = 16 / span, r = tid & (span - 1), q = tid / span & 15, mine = tid / (span * 16);
    const bool on = r < rows && first_dim + q * 4 < end_dim;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on) {
      for (int f0 = mine; f0 < j.parts; f0 += 4 * groups) {
        float4 y[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int f = f0 + k * groups;
          y[k] = f < j.parts ? __ldcg(reinterpret_cast<const float4*>(part(f)) + (first_dim / 4 + q) * set.pitch + r) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int f = f0 + k * groups;
          if (f < j.parts) add(o, ml[f * pitch + r].x, y[k]);
        }
      }
    }
    meet[tid] = o;
    __syncthreads();
    if (mine == 0 && on) {
      for (int k = 1; k < groups; k++) {
        const float4 y = meet[tid + k * span * 16];
        o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
      }
      store(r, first_dim + q * 4, o);
    }
  }
  __syncthreads();
  const uint32_t again = bad;
  if (again)  // rare: an infinity or a NaN among the values, a row without a key
    attend_rows<kJoinThreads>(a, *reinterpret_cast<RowsScratch<kJoinThreads>*>(join_sm), tid, {j.row0, j.head, j.seq, j.first_pos}, r0, again, first_dim, end_dim,
                              [] { __syncthreads(); });
}

// Which kernels run, and how they are cut. Sequences of up to 8 * rt rows (new tokens times query heads of a key/value head) are the kernel
// for few rows'. Where no sequence can have more, it runs alone; where sequences fill tiles of 128 rows on average, the other one takes all: a
// launch less, and no turn of the machine over the cache that leaves the tensor cores alone. Executables for 2079 rows of 32 sequences, one kernel
// and both, us: a prompt of 2048 beside 31 tokens behind 4000 (32/8 heads of 128, bf16) 180 and 202, int8 273 and 276, 4/1 heads of 256 67 and 95,
// 16/2 of 64 69 and 70; the prompt alone 82 and 88, 118 and 121, 44 and 48, 45 and 51; only the 31 tokens 105 and 107, 171 and 165, 55 and 54, 37 and 31;
// one token 28 and 23, 31 and 25, 29 and 25, 21 and 22 (a step of single tokens is better off in an executable of its own with max_new = 1).
struct Choice {
  bool few, many;
  int rt, few_blocks;
};
int few_stages(int D, bool i8) { return i8 && D > 128 ? 2 : 3; }
Choice choose(const AttnPagedArgs& a, int sms) {
  const int group = a.n_q / a.v.n_kv;
  const long long most = (long long)(a.max_new ? std::min(a.max_new, a.v.rows) : a.v.rows) * group;
  Choice c{};
  c.few = group <= kFewRows;
  c.many = !c.few || most > kFewRows;
  if (c.many && (long long)a.v.rows * group / a.v.S >= 128) c.few = false;
  c.rt = most <= 8 ? 1 : 2;
  const bool i8 = a.v.i8 != 0;
  const int per_sm = (227 * 1024) / (few_shape(a.v.D, i8, few_stages(a.v.D, i8)).smem + 4 * 1024);
  c.few_blocks = c.few ? sms * std::max(1, std::min(3, per_sm)) : 0;
  return c;
}
size_t part_bytes(const AttnPagedArgs& a, int blocks, int rows) {
  return ((size_t)blocks * 2 * attn_part_floats(a.v.D, rows) * sizeof(float) + 255) & ~(size_t)255;
}

template <int NT, int RT, int STAGES, bool I8>
cudaError_t run_few(const AttnPagedArgs& a, int blocks, cudaStream_t stream) {
  auto kernel = attn_paged_few_kernel<NT, RT, STAGES, I8>;
  static std::atomic<unsigned long long> attr_done;
  if (first_use_on_device(attr_done)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, few_shape(NT * 16, I8, STAGES).smem);
    if (e != cudaSuccess) return e;
    mark_used_on_device(attr_done);
  }
  return launch_dependent(kernel, dim3(blocks), dim3(kFewThreads), few_shape(a.v.D, I8, STAGES).smem, stream, a);
}
template <int RT>
cudaError_t run_few(const AttnPagedArgs& a, int blocks, cudaStream_t stream) {
  const int steps = a.v.D / 16;
  if (a.scales)
    return steps <= 4 ? run_few<4, RT, 3, true>(a, blocks, stream) : steps <= 8 ? run_few<8, RT, 3, true>(a, blocks, stream) : run_few<16, RT, 2, true>(a, blocks, stream);
  return steps <= 4 ? run_few<4, RT, 3, false>(a, blocks, stream) : steps <= 8 ? run_few<8, RT, 3, false>(a, blocks, stream) : run_few<16, RT, 3, false>(a, blocks, stream);
}

}  // namespace

size_t attn_paged_scratch_bytes(const AttnPagedArgs& a, int sms) {
  const Choice c = choose(a, sms);
  return (c.many ? part_bytes(a, sms, 128) : 0) + part_bytes(a, c.few_blocks, kFewRows) + (size_t)(sms + c.few_blocks) * sizeof(AttnJoin);
}
int attn_paged_launches(const AttnPagedArgs& a, int sms) {
  const Choice c = choose(a, sms);
  return 1 + (c.few ? 1 : 0) + (c.many ? 1 : 0);
}

cudaError_t launch_attn_paged(AttnPagedArgs a, int sms, void* scratch, cudaStream_t stream) {
  const Choice c = choose(a, sms);
  const int group = a.n_q / a.v.n_kv;
  a.group_div = page_divisor(group);
  a.few_rows = c.few ? 8 * c.rt : 0;
  a.wait_ns = wait_limit_ns();
  char* at = (char*)scratch;
  JoinSet sets[2] = {{(float*)at, nullptr, c.many ? sms : 0, 128, kJoinRows}, {(float*)(at + (c.many ? part_bytes(a, sms, 128) : 0)), nullptr, c.few_blocks, kFewRows, 8 * c.rt}};
  AttnJoin* const joins = (AttnJoin*)((char*)sets[1].partial + part_bytes(a, c.few_blocks, kFewRows));
  sets[0].joins = joins;
  sets[1].joins = joins + sms;
  auto shaped = [&](int tokens, int blocks, const JoinSet& set, int takes_few, int min_blocks) {
    AttnPagedArgs k = a;
    k.tokens_per_tile = tokens;
    k.max_tiles = a.v.rows / tokens + std::min(a.v.S, a.v.rows);
    k.grid = blocks;
    k.takes_few = takes_few;
    k.min_blocks = min_blocks;
    k.partial = const_cast<float*>(set.partial);
    k.joins = const_cast<AttnJoin*>(set.joins);
    return k;
  };
  if (c.few) {
    AttnPagedArgs k = shaped(8 * c.rt / group > 0 ? 8 * c.rt / group : 1, c.few_blocks, sets[1], 1, 1);
    k.piece_div = page_divisor(a.v.D * (a.scales ? 1 : 2) / 16);
    const cudaError_t e = c.rt == 1 ? run_few<1>(k, c.few_blocks, stream) : run_few<2>(k, c.few_blocks, stream);
    if (e != cudaSuccess) return e;
  }
  if (c.many) {
    const cudaError_t e = launch_attn_paged_tile(shaped(128 / group, sms, sets[0], 0, 2), stream);
    if (e != cudaSuccess) return e;
  }
  const int join_smem = std::max(std::max(sets[0].count * sets[0].join_rows, sets[1].count * sets[1].join_rows) * (int)sizeof(float2), (int)sizeof(RowsScratch<kJoinThreads>));
  static std::atomic<unsigned long long> attr_done;
  if (first_use_on_device(attr_done)) {
    const cudaError_t e = cudaFuncSetAttribute(attn_paged_join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
    if (e != cudaSuccess) return e;
    mark_used_on_device(attr_done);
  }
  return launch_dependent(attn_paged_join_kernel, dim3(sets[0].count * (128 / kJoinRows) + sets[1].count * ((a.v.D + kJoinDims - 1) / kJoinDims)), dim3(kJoinThreads),
                          join_smem, stream, a, sets[0], sets[1]);
}

}  // namespace tb200
