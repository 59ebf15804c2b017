// Rows of a tile against their keys, exactly as the mask says: keys that a row does not see are not multiplied by anything. The plain form of
// attn_paged, which the kernels fall back to for rows whose sums are not finite (a matrix product multiplies what a hidden key's value holds by
// zero, and zero times infinity is not zero). Eight rows share what is read of their keys and values; of a tile of 128 rows behind 2000 keys
// (160 heads of 16) all rows once more take 2.8 ms (row by row 92), of 128 rows behind 4000 keys (a head of 256) 3.9 ms (146). Nothing that has a limit
// may wait for it.
#pragma once
#include "kernels.h"
#include "paged.cuh"

namespace tb200 {

constexpr int kPlainRows = 8;
template <int THREADS>
struct alignas(16) RowsScratch {
  float q[kPlainRows][256];      // queries, in the end sums
  float p[THREADS][kPlainRows];  // a key's weights
  int slot[THREADS];
  uint32_t seen[THREADS];        // which of the rows see the key
  float red[THREADS / 32][kPlainRows];
  uint32_t any[THREADS / 32];
  int at[kPlainRows], pos[kPlainRows], near_key[kPlainRows];  // row of queries (of one head) or -1, position, where its window begins
};
// A tile: its first row of the chunk, key/value head, sequence, position of its first token.
struct TileRows {
  int row0, head, seq, first_pos;
};

// Rows r0 + i of the tile for every bit i of `bits`, by threads t = 0 .. THREADS - 1 (whole warps, 128 or 256) that `sync` synchronises. Writes
// dims d0 .. d1 - 1 (multiples of four). The scratch may be in use until the first `sync`, and is free again when this returns.
template <int THREADS, typename Sync>
__device__ __noinline__ void attend_rows(const AttnPagedArgs& a, RowsScratch<THREADS>& sm, int t, TileRows w, int r0, uint32_t bits, int d0, int d1, Sync sync) {
  const PagedView& v = a.v;
  const int D = v.D, group = a.n_q / v.n_kv, warp = t >> 5;
  const int32_t* const pages_of = v.table + (long long)w.seq * v.max_pages;
  auto all_or = [&](uint32_t x) {
    x = __reduce_or_sync(0xffffffffu, x);
    sync();
    if ((t & 31) == 0) sm.any[warp] = x;
    sync();
#pragma unroll 1
    for (int i = 0; i < THREADS / 32; i++) x |= sm.any[i];
    return x;
  };
  // values: a thread has four dims of every key_step-th key
  int lanes = 4;
  while (lanes * 4 < D) lanes *= 2;
  const int d = (t & (lanes - 1)) * 4, key_step = THREADS / lanes, first_key = t / lanes;
  const bool on = d < D && d >= d0 && d < d1;
  {  // a sequence without pages (an idle one of a batch, say): zeros at once
    const int newest = (int)min((long long)w.first_pos + page_of(r0 + 31 - __clz(bits), a.group_div), v.capacity - 1ll);
    uint32_t held = 0;
#pragma unroll 1
    for (int i = t; i <= page_of(newest, v.div); i += THREADS) held |= (unsigned)pages_of[i] < (unsigned)v.pages;
    if (!all_or(held)) {
#pragma unroll 1
      for (int i = warp; i < 32; i += THREADS / 32) {
        const int tok = page_of(r0 + i, a.group_div);
        uint16_t* const to = a.out + ((long long)(w.row0 + tok) * a.n_q + w.head * group + r0 + i - tok * group) * D;
        for (int k = d0 + (t & 31) * 4; (bits >> i & 1) && k < d1; k += 128) *reinterpret_cast<uint2*>(to + k) = make_uint2(0, 0);
      }
      sync();
      return;
    }
  }
  while (bits) {
    sync();
    if (t < kPlainRows) {
      uint32_t left = bits;
#pragma unroll 1
      for (int i = 0; i < t; i++) left &= left - 1;
      const int r = left ? r0 + __ffs(left) - 1 : -1, tok = r < 0 ? 0 : page_of(r, a.group_div);
      const int pos = r < 0 ? -1 : (int)min((long long)w.first_pos + tok, 0x7fffffffll);
      sm.at[t] = r < 0 ? -1 : (w.row0 + tok) * a.n_q + w.head * group + r - tok * group;
      sm.pos[t] = pos;
      sm.near_key[t] = a.window ? max(0, pos - a.window + 1) : 0;
    }
    sync();
#pragma unroll 1
    for (int i = 0; i < kPlainRows; i++) bits &= bits - 1;
    int last = -1, near_first = 0x7fffffff;
#pragma unroll 1
    for (int i = 0; i < kPlainRows; i++) {
      if (sm.at[i] < 0) continue;
      last = max(last, sm.pos[i]);
      near_first = min(near_first, sm.near_key[i]);
    }
    last = min(last, v.capacity - 1);
#pragma unroll 1
    for (int i = 0; i < kPlainRows; i++)
      for (int k = t; k < D; k += THREADS) sm.q[i][k] = sm.at[i] < 0 ? 0.f : paged_bf2f(a.q[(long long)sm.at[i] * D + k]) * a.scale;
    sync();

    float m[kPlainRows], sum[kPlainRows], o[kPlainRows][4] = {};
    uint32_t saw = 0;
#pragma unroll
    for (int i = 0; i < kPlainRows; i++) m[i] = -INFINITY, sum[i] = 0.f;
#pragma unroll 1
    for (int j0 = 0; j0 <= last; j0 += THREADS) {
      if (j0 >= a.sinks) j0 = max(j0, near_first & -THREADS);
      const int j = j0 + t;
      uint32_t seen = 0;
#pragma unroll 1
      for (int i = 0; i < kPlainRows && j <= last; i++) seen |= (j <= sm.pos[i] && (j >= sm.near_key[i] || j < a.sinks) ? 1u : 0u) << i;
      const int slot = seen ? (int)slot_of(v, w.seq, j) : -1;
      if (slot < 0) seen = 0;
      saw |= seen;
      float s[kPlainRows] = {};
      if (seen) {
        const long long at = ((long long)slot * v.n_kv + w.head) * D;
        if (a.scales) {
#pragma unroll 1
          for (int k = 0; k < D; k += 4) {
            const char4 x = *reinterpret_cast<const char4*>((const int8_t*)a.k + at + k);
#pragma unroll
            for (int i = 0; i < kPlainRows; i++) {
              const float4 q = *reinterpret_cast<const float4*>(&sm.q[i][k]);
              s[i] += q.x * x.x + q.y * x.y + q.z * x.z + q.w * x.w;
            }
          }
          const float by = a.scales[(long long)slot * 2 * v.n_kv + w.head];
#pragma unroll
          for (int i = 0; i < kPlainRows; i++) s[i] *= by;
        } else {
#pragma unroll 1
          for (int k = 0; k < D; k += 4) {
            const uint2 x = *reinterpret_cast<const uint2*>((const uint16_t*)a.k + at + k);
#pragma unroll
            for (int i = 0; i < kPlainRows; i++) {
              const float4 q = *reinterpret_cast<const float4*>(&sm.q[i][k]);
              s[i] += q.x * __uint_as_float(x.x << 16) + q.y * __uint_as_float(x.x & 0xffff0000u) + q.z * __uint_as_float(x.y << 16) +
                      q.w * __uint_as_float(x.y & 0xffff0000u);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kPlainRows; i++) {
        if (!(seen >> i & 1)) s[i] = -INFINITY;
        float top = s[i];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        if ((t & 31) == 0) sm.red[warp][i] = top;
      }
      sync();  // (and everybody is through with the last keys' weights)
#pragma unroll
      for (int i = 0; i < kPlainRows; i++) {
        float top = m[i];
        for (int k = 0; k < THREADS / 32; k++) top = fmaxf(top, sm.red[k][i]);
        const float p = s[i] == -INFINITY ? 0.f : __expf(s[i] - top), keep = m[i] == top ? 1.f : __expf(m[i] - top);
        m[i] = top;
        sum[i] = sum[i] * keep + p;
#pragma unroll
        for (int e = 0; e < 4; e++) o[i][e] *= keep;
        sm.p[t][i] = p;
      }
      sm.slot[t] = slot;
      sm.seen[t] = seen;
      sync();
      if (!on) continue;
#pragma unroll 1
      for (int k = first_key; k < THREADS; k += key_step) {
        const uint32_t who = sm.seen[k];
        if (!who) continue;
        const long long slot_k = sm.slot[k], at = (slot_k * v.n_kv + w.head) * D + d;
        float x[4];
        if (a.scales) {
          const char4 y = *reinterpret_cast<const char4*>((const int8_t*)a.vv + at);
          const float by = a.scales[slot_k * 2 * v.n_kv + v.n_kv + w.head];
          x[0] = y.x * by; x[1] = y.y * by; x[2] = y.z * by; x[3] = y.w * by;
        } else {
          const uint2 y = *reinterpret_cast<const uint2*>((const uint16_t*)a.vv + at);
          x[0] = __uint_as_float(y.x << 16); x[1] = __uint_as_float(y.x & 0xffff0000u);
          x[2] = __uint_as_float(y.y << 16); x[3] = __uint_as_float(y.y & 0xffff0000u);
        }
#pragma unroll
        for (int i = 0; i < kPlainRows; i++) {
          if (!(who >> i & 1)) continue;
          const float p = sm.p[k][i];
#pragma unroll
          for (int e = 0; e < 4; e++) o[i][e] += p * x[e];
        }
      }
    }
    // sums over the threads, and over the keys' groups in their order
    saw = all_or(saw);
#pragma unroll
    for (int i = 0; i < kPlainRows; i++) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], off);
      if ((t & 31) == 0) sm.red[warp][i] = sum[i];
    }
#pragma unroll 1
    for (int g = 0; g < key_step; g++) {
      if (on && first_key == g) {
#pragma unroll
        for (int i = 0; i < kPlainRows; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) sm.q[i][d + e] = g == 0 ? o[i][e] : sm.q[i][d + e] + o[i][e];
      }
      sync();
    }
    if (on && first_key == 0) {
#pragma unroll 1
      for (int i = 0; i < kPlainRows; i++) {
        if (sm.at[i] < 0) continue;
        float all = 0.f;
#pragma unroll 1
        for (int k = 0; k < THREADS / 32; k++) all += sm.red[k][i];
        // a row that sees no key is all zeros; one whose scores are all -inf has no weights
        auto value = [&](int e) { return saw >> i & 1 ? sm.q[i][d + e] / all : 0.f; };
        *reinterpret_cast<uint2*>(a.out + (long long)sm.at[i] * D + d) = make_uint2(pack_bf16(value(0), value(1)), pack_bf16(value(2), value(3)));
      }
    }
  }
  sync();
}

}  // namespace tb200
