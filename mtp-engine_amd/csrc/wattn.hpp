// Attention with a sliding window and a few first tokens that stay visible,
// gfx950: what its kernels share, and the form for any sizes and strides.
//
//   out[b, h, t] = sum_j p_j v_j,  p = softmax_j(q . k_j * scale) over the keys
//   j <= pos with pos - j < window or j < sinks,  pos = first + t,
//
// key head h / G for query head h. A row that sees no key is zero. Keys are
// dense (a prompt, alone or behind earlier keys) or lie in the pages of a
// cache (page and slot of each key as in paged attention; a page outside the
// pool hides its key).
//
// A hidden key never reaches a row, whatever its K and V hold. The kernels
// that multiply whole tiles hide a key by a probability of zero, which times
// an infinite or NaN V is NaN: a row whose output is not finite is therefore
// computed again by win_row(), which reads no hidden V.
#pragma once

#include "mtp_common.hpp"
#include "wattn_args.hpp"

namespace mtp {

// The span of the rows t0 .. t1 - 1 of sequence b; first and rows are those of
// the whole call.
__device__ __forceinline__ WinSpan win_span(const WinArgs &a, int b, int t0, int t1) {
  WinSpan s;
  const int64_t st = a.start_dev ? a.start_dev[a.start_per_row ? b : 0] : a.start_host;
  // past L + window every start sees the same keys: none but the sinks, or
  // (no window) all
  const int64_t most = (int64_t)a.L + (a.window == kWinNone ? 0 : a.window);
  s.first = (int)min(max(st, (int64_t)-a.T), most);
  int end = a.L;
  s.rows = a.T;
  if (a.lengths) {
    end = (int)min(max(a.lengths[b], (int64_t)0), (int64_t)a.L);
    s.rows = min(a.T, max(0, end - s.first));
  }
  t1 = min(t1, s.rows);
  s.hi = t0 < t1 ? max(0, min(end, s.first + t1)) : 0;
  s.lo = a.window == kWinNone ? 0 : max(0, s.first + t0 - a.window + 1);
  s.ns = min(min(a.sinks, s.lo), s.hi);
  s.lo = min(max(s.lo, s.ns), s.hi);
  return s;
}

__device__ __forceinline__ WinSpan win_span(const WinArgs &a, int b) {
  return win_span(a, b, 0, a.T);
}

// Whether the row at position pos sees key j (j below the span's end).
__device__ __forceinline__ bool win_sees(const WinArgs &a, int pos, int j) {
  return (j <= pos) & ((j > pos - a.window) | (j < a.sinks));  // no branches
}

// Element offset of key j's row in k (and, dense, by its own strides in v), or
// false where its page is outside the pool.
template <bool PAGED>
__device__ __forceinline__ bool win_key_at(const WinArgs &a, int b, int hk, int j, int64_t &ko,
                                           int64_t &vo) {
  if constexpr (PAGED) {
    const int page = a.table[(int64_t)b * a.ld_tab + j];
    ko = vo = (int64_t)page * a.p_sp + (int64_t)b * a.k_sb + (int64_t)hk * a.k_sh +
              (int64_t)(j % a.page_size) * a.k_st;
    return page >= 0 && page < a.npages;
  } else {
    ko = (int64_t)b * a.k_sb + (int64_t)hk * a.k_sh + (int64_t)j * a.k_st;
    vo = (int64_t)b * a.v_sb + (int64_t)hk * a.v_sh + (int64_t)j * a.v_st;
    return true;
  }
}

// Four elements from d on of row (b, h, t) of the output; CT's 4-element rows
// are aligned (o strides and address in whole 16 bytes).
template <int CT>
__device__ __forceinline__ void win_store4(const WinArgs &a, int b, int h, int t, int d, f32x4 v) {
  const int64_t at = (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + (int64_t)t * a.o_st + d;
  if constexpr (CT == MTP_F32) {
    *(f32x4 *)((float *)a.out + at) = v;
  } else {
    uint2 w;
    w.x = pack2<CT>(v[0], v[1]);
    w.y = pack2<CT>(v[2], v[3]);
    *(uint2 *)((uint16_t *)a.out + at) = w;
  }
}

// LDS of one wave in win_row(), floats.
__host__ __device__ constexpr int win_row_lds(int d) { return d + 64 * 3 + 2; }
// LDS writes of this wave before, its reads after.
__device__ __forceinline__ void win_wave_sync() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

// One row (b, h, t) by one wave, 64 keys at a time: lane i takes key i's
// score, then the lanes take the elements d of the sum over V. NV = ceil(D /
// 64) at least. Scores and (max, sum) are kept where a.scores is set.
template <int NV, bool PAGED>
__device__ __forceinline__ void win_row(const WinArgs &a, int ct, int b, int h, int t,
                                        const WinSpan &s, float *lds, bool keep) {
  float *const s_q = lds, *const s_p = lds + a.D;
  int64_t *const s_off = (int64_t *)(lds + ((a.D + 65) & ~1));  // 8-byte aligned
  const int lane = threadIdx.x & 63;
  const int hk = h / a.G;
  const int pos = s.first + t;
  const int64_t qo = (int64_t)b * a.q_sb + (int64_t)h * a.q_sh + (int64_t)t * a.q_st;
  win_wave_sync();  // earlier uses of this LDS
  for (int d = lane; d < a.D; d += 64) s_q[d] = load_as_f32(a.q, ct, qo + d);
  win_wave_sync();
  const int64_t row = ((int64_t)b * a.Hk + hk) * a.G * a.T + (int64_t)t * a.G + (h - hk * a.G);
  float m = -INFINITY, l = 0.f, o[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) o[i] = 0.f;
  const int n = t < s.rows ? s.count() : 0;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const int i = i0 + lane, j = s.key(i);
    int64_t ko = 0, vo = 0;
    bool ok = i < n && win_sees(a, pos, j);
    if (ok) ok = win_key_at<PAGED>(a, b, hk, j, ko, vo);
    float sc = 0.f;
    if (ok) {
      for (int d = 0; d < a.D; ++d) sc = fmaf(s_q[d], load_as_f32(a.k, ct, ko + d), sc);
    }
    sc = ok ? sc * a.scale : -INFINITY;
    if (keep && i < n) a.scores[row * a.ld_sc + i] = sc;
    float mx = sc;
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor(mx, w, 64));
    const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = mn;
    const float p = ok ? __builtin_amdgcn_exp2f(sc - ref) : 0.f;
    l = l * alpha + sum_over_lanes<64>(p);
    s_p[lane] = p;
    s_off[lane] = vo;
    win_wave_sync();
#pragma unroll
    for (int e = 0; e < NV; ++e) o[e] *= alpha;
    for (unsigned long long seen = __ballot(ok); seen; seen &= seen - 1) {
      const int c = __builtin_ctzll(seen);
      const float pc = s_p[c];
      const int64_t off = s_off[c];
#pragma unroll
      for (int e = 0; e < NV; ++e) {
        const int d = lane + 64 * e;
        if (d < a.D) o[e] = fmaf(pc, load_as_f32(a.v, ct, off + d), o[e]);
      }
    }
    win_wave_sync();
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a NaN sum stays NaN
  const int64_t oo = (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + (int64_t)t * a.o_st;
#pragma unroll
  for (int e = 0; e < NV; ++e) {
    const int d = lane + 64 * e;
    if (d < a.D) store_from_f32(a.out, ct, oo + d, o[e] * inv);
  }
  if (keep && lane == 0) {
    a.pml[row * 2] = m;
    a.pml[row * 2 + 1] = l;
  }
}

// Any sizes and strides: one wave per row.
template <int NV, bool PAGED>
__global__ void __launch_bounds__(64) win_rows_generic_kernel(const WinArgs a, int ct) {
  extern __shared__ __attribute__((aligned(16))) float s_row[];
  const int64_t r = blockIdx.x;
  const int t = (int)(r % a.T);
  const int h = (int)((r / a.T) % a.H);
  const int b = (int)(r / ((int64_t)a.T * a.H));
  win_row<NV, PAGED>(a, ct, b, h, t, win_span(a, b), s_row, a.scores != nullptr);
}

}  // namespace mtp
