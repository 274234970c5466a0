// Eviction from a paged cache by the attention weight that its keys received,
// gfx950.
//
// Of the n entries of a sequence's table, each key head keeps its first
// `sinks`, its last `recent` and, up to `keep` in all, the others of most
// weight (equal weights: the lower position; NaN is the most). The kept rows
// of K and V go, in the order of their positions, to the slots 0 .. of
// another table. An entry whose page is outside the pool holds no key and is
// never kept.
//
// Selection, one workgroup per (sequence, head): a weight as an unsigned
// integer of the same order, entries that stay whatever their weight at its
// top, absent ones at zero; a radix select finds the keep-th largest value, 11,
// 11 and 10 bits a pass from a histogram in LDS (the top 11 are the sign, the
// exponent and two bits more, so that few lanes meet in one counter), and a
// prefix sum over the workgroup gives the larger ones and the first of its
// equals their places. A lane keeps its entries in registers. Then the
// rows move, 16 bytes a lane where the row allows it, the few rows of a small
// cache by the same workgroup: that part is bound by HBM.
//
// A pass has three barriers, and the passes end where a digit's entries are all
// wanted, mostly after two.
//
// Measured (B 4, 8 heads, L 8192, keep 2048, D 128, bf16): selection 11.3 us, move
// 13.4 us (5.0 TB/s); with all three passes, five barriers each: selection 12.9 us;
// a launch a pass over 8 bits and a thread's entries one by one: 31 us. 16 heads of
// 31391 entries, keep 5042, D 64: 34.4 us both, with a thread's entries one after
// another in memory 59; 16 heads of 100000 entries, keep 4096, D 128: 120 and 525,
// the arithmetic of one CU a head.
#pragma once

#include "mtp_common.hpp"

namespace mtp {

struct EvictArgs {
  const float *weights;        // [B, Hk, L]
  const int64_t *lengths;      // [B]
  const int32_t *table;        // [B, L]
  const int32_t *out_table;    // [B, keep]
  int B, Hk, L, keep, sinks, recent, npages, page_size;
  void *k_pages, *v_pages;     // [P, B, Hk, page_size, D], by bytes: from and to
  int64_t row_bytes;
  int moves;                   // 1: the selecting workgroup moves its rows (16-byte units)
  int32_t *kept;               // [B, Hk, keep], -1 past the new length
  float *out_weights;          // [B, Hk, keep], 0 past it
  int64_t *out_lengths;        // [B]
};

constexpr uint32_t kEvictFixed = 0xffffffffu;  // above every weight, NaN among them

// Rank of entry j of weight x on a page, as an unsigned integer; 0: no entry.
__device__ __forceinline__ uint32_t evict_key(const EvictArgs &a, int n, int j, float x, int page) {
  const uint32_t bits = x == 0.f ? 0u : __float_as_uint(x);  // -0 ranks with 0
  uint32_t u = (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
  u = x != x ? kEvictFixed - 1 : u;
  u = (j < a.sinks) | (j >= n - a.recent) ? kEvictFixed : u;
  return (j < n) & (page >= 0) & (page < a.npages) ? u : 0u;
}

// Unit c (of type U) of the kept row at place j of (sequence, head) bh: from the
// slot of position `from` to that of place j.
template <typename U>
__device__ __forceinline__ void evict_copy(const EvictArgs &a, int b, int h, int j, int from,
                                           int64_t units, int64_t c) {
  const int sp = a.table[(int64_t)b * a.L + from];
  const int dp = a.out_table[(int64_t)b * a.keep + j];
  if (sp < 0 || sp >= a.npages || dp < 0 || dp >= a.npages) return;
  const int64_t plane = (int64_t)b * a.Hk + h, per = (int64_t)a.B * a.Hk;
  const int64_t so = (((int64_t)sp * per + plane) * a.page_size + from % a.page_size) * units + c;
  const int64_t to = (((int64_t)dp * per + plane) * a.page_size + j % a.page_size) * units + c;
  const U kx = ((const U *)a.k_pages)[so], vx = ((const U *)a.v_pages)[so];
  ((U *)a.k_pages)[to] = kx;
  ((U *)a.v_pages)[to] = vx;
}

constexpr int kEvictThreads = 1024;

// Inclusive sum over the workgroup, and its total. s_sum: one word a wave, whose
// earlier readers have passed a barrier since.
__device__ __forceinline__ uint32_t evict_scan(uint32_t x, uint32_t *s_sum, uint32_t &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) s_sum[wave] = x;
  __syncthreads();
  uint32_t before = 0u;
  total = 0u;
#pragma unroll
  for (int w = 0; w < kEvictThreads / 64; ++w) {
    const uint32_t y = s_sum[w];
    before += w < wave ? y : 0u;
    total += y;
  }
  return x + before;
}

// E: entries of a lane in registers (E * kEvictThreads >= L); 0: any number, read
// again for every pass. A wave has `each` runs of 256 entries one after another, a
// lane four in a row of each run, so that loads are whole lines and ballots give
// the places within a run.
template <int E>
__global__ void __launch_bounds__(kEvictThreads) evict_select_kernel(const EvictArgs a) {
  constexpr int BINS = 2048;
  constexpr int COPIES = 4;  // of a histogram, lane l in copy l % 4: fewer lanes meet
  constexpr int WAVES = kEvictThreads / 64;
  __shared__ __attribute__((aligned(8))) uint32_t s_hist[COPIES][BINS + 16];
  __shared__ uint32_t s_sum[WAVES];
  __shared__ uint2 s_cnt[WAVES];
  __shared__ uint32_t s_pick[2];
  const int th = threadIdx.x, lane = th & 63;
  const int wave = __builtin_amdgcn_readfirstlane(th >> 6);
  const int bh = blockIdx.x, b = bh / a.Hk, h = bh - b * a.Hk;
  const float *const w = a.weights + (int64_t)bh * a.L;
  const int32_t *const tab = a.table + (int64_t)b * a.L;
  const int n = (int)min(max(a.lengths[b], (int64_t)0), (int64_t)a.L);
  const int each = (n + 4 * kEvictThreads - 1) / (4 * kEvictThreads);
  const int j0 = (wave * each * 64 + lane) * 4;  // below n + 2^13
  auto load4 = [&](int j, float (&x)[4], int (&pg)[4]) {
    if (j + 4 <= n) {  // 16 bytes, of any row at a word's alignment
      typedef __attribute__((ext_vector_type(4), aligned(4))) float f32x4w;
      typedef __attribute__((ext_vector_type(4), aligned(4))) uint32_t u32x4w;
      const f32x4w x4 = *(const f32x4w *)(w + j);
      const u32x4w p4 = *(const u32x4w *)(tab + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = x4[i];
        pg[i] = (int)p4[i];
      }
    } else {  // the last one in place of entries past the end
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = w[min(j + i, n - 1)];
        pg[i] = tab[min(j + i, n - 1)];
      }
    }
  };

  constexpr int Q = E ? E / 4 : 1;
  uint32_t key[Q][4];
  float val[Q][4];
  if constexpr (E > 0) {
    int pg[Q][4];  // every load before the first use
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (q < each) load4(j0 + 256 * q, val[q], pg[q]);
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        key[q][i] = q < each ? evict_key(a, n, j0 + 256 * q + i, val[q][i], pg[q][i]) : 0u;
  }
  // f(first entry, ranks, weights) over the wave's runs, all its lanes together
  auto each_quad = [&](auto f) {
    if constexpr (E > 0) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (q < each) f(j0 + 256 * q, key[q], val[q]);
    } else {
      for (int q = 0; q < each; ++q) {
        const int j = j0 + 256 * q;
        int pg[4];
        load4(j, val[0], pg);
#pragma unroll
        for (int i = 0; i < 4; ++i) key[0][i] = evict_key(a, n, j + i, val[0][i], pg[i]);
        f(j, key[0], val[0]);
      }
    }
  };

  // thr, need: the entries to keep are those above thr and the first `need` of
  // its equals. After the pass at bit sh, thr has the bits of the keep-th
  // largest rank from sh up; where all that have them are wanted, it is one
  // less than the least of those, and no pass is left to do.
  uint32_t thr = 0u, need = (uint32_t)a.keep;
#pragma unroll
  for (int c = 0; c < COPIES; ++c) s_hist[c][th] = s_hist[c][th + 1024] = 0u;
  __syncthreads();
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int sh = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t bins = pass == 2 ? 1024u : 2048u;
    const uint32_t mask = pass == 0 ? 0u : ~0u << (pass == 1 ? 21 : 10);
    each_quad([&](int, const uint32_t(&k)[4], const float(&)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u = k[i];
        if (u != 0u && (u & mask) == thr) {
          const uint32_t bin = (u >> sh) & (bins - 1u);
          // lanes of one bin add once (equal weights, above all zeros)
          const uint32_t first = (uint32_t)__builtin_amdgcn_readfirstlane((int)bin);
          const unsigned long long all = __ballot(1);
          if (__ballot(bin == first) == all) {
            if (lane == __builtin_ctzll(all))
              atomicAdd(&s_hist[0][bin], (uint32_t)__popcll(all));
          } else {
            atomicAdd(&s_hist[lane % COPIES][bin], 1u);
          }
        }
      }
    });
    __syncthreads();
    // from the top: thread th has bins 2047 - 2 th and 2046 - 2 th, and leaves
    // them clear for the next pass
    uint32_t c0 = 0u, c1 = 0u;
#pragma unroll
    for (int c = 0; c < COPIES; ++c) {
      uint2 *const two = (uint2 *)&s_hist[c][BINS - 2 - 2 * th];
      const uint2 x = *two;
      c0 += x.y;
      c1 += x.x;
      *two = uint2{0u, 0u};
    }
    uint32_t total;
    const uint32_t incl = evict_scan(c0 + c1, s_sum, total);
    const uint32_t above = incl - c0 - c1;
    if (total < need) {  // fewer entries than wanted (first pass alone): all of them
      thr = 0u;
      need = 0u;
      break;
    }
    if (above < need && incl >= need) {
      const bool hi = above + c0 >= need;
      const uint32_t low = thr | (uint32_t)(BINS - 1 - 2 * th - (hi ? 0 : 1)) << sh;
      const uint32_t left = need - above - (hi ? 0u : c0);
      const bool whole = left == (hi ? c0 : c1);
      s_pick[0] = whole ? max(low, 1u) - 1u : low;
      s_pick[1] = whole ? 0u : left;
    }
    __syncthreads();
    thr = s_pick[0];
    need = s_pick[1];
    if (need == 0u) break;
  }

  // places: entries above thr and equals of it in the waves before
  uint32_t over = 0u, same = 0u;
  each_quad([&](int, const uint32_t(&k)[4], const float(&)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      over += (uint32_t)__popcll(__ballot(k[i] > thr));
      if (need != 0u) same += (uint32_t)__popcll(__ballot((k[i] == thr) & (k[i] != 0u)));
    }
  });
  if (lane == 0) s_cnt[wave] = uint2{over, same};
  __syncthreads();
  uint32_t at = 0u, es = 0u, all = 0u, equals = 0u;
#pragma unroll
  for (int x = 0; x < WAVES; ++x) {
    const uint2 c = s_cnt[x];
    at += x < wave ? c.x : 0u;
    es += x < wave ? c.y : 0u;
    all += c.x;
    equals += c.y;
  }
  const uint32_t taken = all + min(equals, need);
  at += min(es, need);
  int32_t *const kept = a.kept + (int64_t)bh * a.keep;
  float *const ow = a.out_weights + (int64_t)bh * a.keep;
  auto before = [&](unsigned long long m, uint32_t x) {  // x and the lanes below in m
    return (uint32_t)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32),
                                               __builtin_amdgcn_mbcnt_lo((uint32_t)m, x));
  };
  each_quad([&](int j, const uint32_t(&k)[4], const float(&x)[4]) {
    // those taken in the lanes before, then in this lane
    bool take[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) take[i] = k[i] > thr;
    if (need != 0u) {  // equals too, by their rank
      uint32_t rank = es;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned long long m = __ballot((k[i] == thr) & (k[i] != 0u));
        rank = before(m, rank);
        es += (uint32_t)__popcll(m);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool eq = (k[i] == thr) & (k[i] != 0u);
        take[i] = take[i] | (eq & (rank < need));
        rank += eq;
      }
    }
    uint32_t to = at;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned long long m = __ballot(take[i]);
      to = before(m, to);
      at += (uint32_t)__popcll(m);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (take[i]) {
        if (to < (uint32_t)a.keep) {
          kept[to] = j + i;
          ow[to] = x[i];
        }
        ++to;
      }
    }
  });
  for (int j = (int)taken + th; j < a.keep; j += kEvictThreads) {
    kept[j] = -1;
    ow[j] = 0.f;
  }
  if (h == 0 && th == 0) a.out_lengths[b] = (int64_t)taken;
  if (!a.moves) return;
  __syncthreads();  // the positions written above
  const int units = (int)(a.row_bytes / 16);
  for (int i = th; i < (int)taken * units; i += kEvictThreads)
    evict_copy<u32x4>(a, b, h, i / units, kept[i / units], units, i % units);
}

// Kept rows to their new slots, U the unit of a copy; a thread takes one unit of
// K and of V.
template <typename U>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictArgs a) {
  const int64_t units = a.row_bytes / (int64_t)sizeof(U);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / units;
  if (row >= (int64_t)a.B * a.Hk * a.keep) return;
  const int64_t bh = row / a.keep;
  const int b = (int)(bh / a.Hk), h = (int)(bh - (int64_t)b * a.Hk);
  const int from = a.kept[row];
  if (from >= 0) evict_copy<U>(a, b, h, (int)(row % a.keep), from, units, i - row * units);
}

}  // namespace mtp
