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
// top, absent ones at zero; a radix select finds the keep-th largest value,
// eight bits a pass from a histogram in LDS, and a last pass writes the
// positions of the larger ones and of the first of its equals by a prefix sum
// over the workgroup. Then the rows move, 16 bytes a lane where the row
// allows it: that part is bound by HBM.
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
  int32_t *kept;               // [B, Hk, keep], -1 past the new length
  float *out_weights;          // [B, Hk, keep], 0 past it
  int64_t *out_lengths;        // [B]
};

constexpr uint32_t kEvictFixed = 0xffffffffu;  // above every weight, NaN among them

// Entry j's rank as an unsigned integer; 0: no entry.
__device__ __forceinline__ uint32_t evict_key(const EvictArgs &a, const float *w,
                                              const int32_t *tab, int n, int j) {
  if (j >= n) return 0u;
  const int page = tab[j];
  if (page < 0 || page >= a.npages) return 0u;
  if (j < a.sinks || j >= n - a.recent) return kEvictFixed;
  const float x = w[j];
  if (x != x) return kEvictFixed - 1;
  const uint32_t u = x == 0.f ? 0u : __float_as_uint(x);  // -0 ranks with 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kEvictThreads = 1024;

__global__ void __launch_bounds__(kEvictThreads) evict_select_kernel(const EvictArgs a) {
  __shared__ uint32_t s_hist[256];
  __shared__ uint32_t s_wave[kEvictThreads / 64][2];
  __shared__ uint32_t s_pick[2];
  const int th = threadIdx.x, lane = th & 63, wave = th >> 6;
  const int bh = blockIdx.x, b = bh / a.Hk, h = bh - b * a.Hk;
  const float *const w = a.weights + (int64_t)bh * a.L;
  const int32_t *const tab = a.table + (int64_t)b * a.L;
  const int n = (int)min(max(a.lengths[b], (int64_t)0), (int64_t)a.L);

  // the keep-th largest rank: after the pass at bit s, `pre` holds its bits
  // from s up and `need` how many entries are wanted from those that share
  // them
  uint32_t pre = 0u, need = (uint32_t)a.keep;
  for (int sh = 24; sh >= 0; sh -= 8) {
    for (int i = th; i < 256; i += kEvictThreads) s_hist[i] = 0u;
    __syncthreads();
    const uint32_t mask = sh == 24 ? 0u : ~0u << (sh + 8);
    for (int j = th; j < n; j += kEvictThreads) {
      const uint32_t u = evict_key(a, w, tab, n, j);
      if ((u & mask) == (pre & mask)) atomicAdd(&s_hist[(u >> sh) & 255u], 1u);
    }
    __syncthreads();
    if (th < 64) {
      // lane i holds bins 255 - 4 i .. 252 - 4 i: a prefix sum from the top
      uint32_t c[4], sum = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = s_hist[255 - 4 * lane - i];
        sum += c[i];
      }
      uint32_t incl = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(incl, o, 64);
        if (lane >= o) incl += y;
      }
      uint32_t above = incl - sum;
      const uint32_t total = __shfl(incl, 63, 64);
      if (total < need) {  // fewer entries than wanted: all of them (rank 0 is below)
        if (lane == 0) {
          s_pick[0] = 0u;
          s_pick[1] = 0u;
        }
      } else if (above < need && incl >= need) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (above < need && above + c[i] >= need) {
            s_pick[0] = (uint32_t)(255 - 4 * lane - i);
            s_pick[1] = need - above;
          }
          above += c[i];
        }
      }
    }
    __syncthreads();
    if (s_pick[1] == 0u) {
      pre = 0u;
      need = 0u;
      break;
    }
    pre |= s_pick[0] << sh;
    need = s_pick[1];
    __syncthreads();
  }
  // rank 0 is no entry: then every entry is above it and none of its equals taken
  if (pre == 0u) need = 0u;

  // entries above `pre` and the first `need` that equal it, in order
  uint32_t taken = 0u, equal = 0u;
  int32_t *const kept = a.kept + (int64_t)bh * a.keep;
  float *const ow = a.out_weights + (int64_t)bh * a.keep;
  for (int j0 = 0; j0 < n; j0 += kEvictThreads) {
    const int j = j0 + th;
    const uint32_t u = evict_key(a, w, tab, n, j);
    const bool over = u > pre, same = u == pre && pre != 0u;
    const unsigned long long mo = __ballot(over), ms = __ballot(same);
    if (lane == 0) {
      s_wave[wave][0] = (uint32_t)__popcll(mo);
      s_wave[wave][1] = (uint32_t)__popcll(ms);
    }
    __syncthreads();
    uint32_t eb = equal, before = taken, et = equal, tt = taken;
    for (int v = 0; v < kEvictThreads / 64; ++v) {
      const uint32_t o = s_wave[v][0], s = s_wave[v][1];
      const uint32_t got = o + min(et + s, need) - min(et, need);
      if (v < wave) {
        before += got;
        eb += s;
      }
      tt += got;
      et += s;
    }
    const unsigned long long below = lane == 0 ? 0ull : ~0ull >> (64 - lane);
    const uint32_t es = eb + (uint32_t)__popcll(ms & below);
    const bool take = over || (same && es < need);
    if (take) {
      const uint32_t at = before + (uint32_t)__popcll(mo & below) + min(es, need) - min(eb, need);
      if (at < (uint32_t)a.keep) {
        kept[at] = j;
        ow[at] = w[j];
      }
    }
    taken = tt;
    equal = et;
    __syncthreads();
  }
  for (int j = (int)taken + th; j < a.keep; j += kEvictThreads) {
    kept[j] = -1;
    ow[j] = 0.f;
  }
  if (h == 0 && th == 0) a.out_lengths[b] = (int64_t)taken;
}

// Kept rows to their new slots, U the unit of a copy. Grid: (rows of the
// pool's [B, Hk, keep] in groups, 1); a thread takes one unit of K and of V.
template <typename U>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictArgs a) {
  const int64_t units = a.row_bytes / (int64_t)sizeof(U);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / units;
  if (row >= (int64_t)a.B * a.Hk * a.keep) return;
  const int64_t c = i - row * units;
  const int j = (int)(row % a.keep);
  const int64_t bh = row / a.keep;
  const int b = (int)(bh / a.Hk), h = (int)(bh - (int64_t)b * a.Hk);
  const int from = a.kept[row];
  if (from < 0) return;
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

}  // namespace mtp
