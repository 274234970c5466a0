// Windowed attention for few rows and many keys, gfx950: new tokens over a
// paged cache in fp32, bf16 and f16, and the prompts that the prompt kernel
// does not take (fp32 ones above all). Definitions in wattn.hpp.
//
// The G * T rows of a (sequence, key head) - query heads of a group read the
// same keys - go by blocks of 16 * RT (row r = t * G + head); a block's
// visible keys, counted without gaps (WinSpan), are split into nchunks equal
// parts, one per workgroup, so that few rows still fill the chip; chunks join
// in win_merge_kernel, in order. Within a workgroup four waves take steps of
// SK keys in turn and join at the end; a step has no barrier:
//   * K rows go from memory to the registers that the matrix product wants
//     them in: lane l holds bytes 64 c + 16 (l / 16) .. + 15 of key l % 16,
//     for every 64-byte piece c of the row, one load each.
//   * S^T[key][row] = K Q^T, 16 x 16 tiles with Q^T in registers: lane l has
//     keys 4 (l / 16) + i of row l % 16, so a row's maximum takes two lane
//     swaps and its sum none until the end.
//   * O^T[d][row] += V^T P^T takes the S^T registers as they are (rounded to
//     the 16-bit type; fp32 stays). V rows, loaded like K's, pass through the
//     wave's own part of LDS: 16-bit ones come back by transposing reads, four
//     keys of one d a lane.
//   * the next step's K and V are asked for as soon as this step's have left
//     their registers, before its softmax; the page numbers one step earlier.
// The running maximum moves only when a step exceeds it by more than 2^8.
//
// Bound: HBM, K and V read once per row block (blocks of one key head run on
// one XCD and meet in its L2). 16 KB a wave in flight, two or more waves per
// SIMD.
#pragma once

#include "wattn.hpp"

namespace mtp {

typedef short win_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((ext_vector_type(4), aligned(4))) float f32x4u;

// Transposing LDS read: in each 16-lane group lane j receives element j % 4 of
// the 8-byte reads of lanes 4 i + j / 4, i = 0 .. 3.
__device__ __forceinline__ uint64_t win_tr16(const unsigned char *p) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                          (__attribute__((address_space(3))) win_s16x4 *)p));
#else
  (void)p;
  return 0;
#endif
}

// Place of a row's 16-byte chunks: chunk c of row r at c ^ win_swz(r), so that
// 16 rows' stores of one chunk and the reads of V fall on distinct banks.
template <int CT, int RB>
__device__ __forceinline__ int win_swz(int r) {
  if constexpr (CT == MTP_F32) return r & 15;
  else if constexpr (RB >= 256) return ((r & 3) << 2) | ((r >> 2) & 3);
  else return ((r >> 2) & 1) | (r & 2) | (((r >> 3) & 1) << 2);
}

template <int CT, int D, int RT, bool PAGED>
__global__ void __launch_bounds__(64 * kWinSplitWaves, 2) win_split_kernel(const WinArgs a) {
  constexpr int EB = dtype_bytes(CT);
  constexpr int RB = D * EB;           // bytes of a row
  constexpr int NC = RB / 64;          // 64-byte pieces of a row
  constexpr int SK = win_split_keys(RB);
  constexpr int KT = SK / 16;          // key tiles of a step
  constexpr int NW = kWinSplitWaves;
  constexpr int RP = 16 * RT;
  static_assert(RB % 128 == 0 && (CT == MTP_F32 || KT == 2), "whole products");
  constexpr int kRegion = SK * RB;     // a wave's V rows
  constexpr int kMerge = NW * 16 * (D + 4) * 4;
  constexpr int kLds = NW * kRegion > kMerge ? NW * kRegion : kMerge;
  __shared__ __attribute__((aligned(16))) unsigned char lds[kLds];
  __shared__ float s_ml[NW][16][2];
  __shared__ unsigned s_bad[RT];

  const int th = threadIdx.x, lane = th & 63;
  const int wave = __builtin_amdgcn_readfirstlane(th >> 6);
  const int g = lane >> 4, l16 = lane & 15;
  const int bh = blockIdx.x, b = bh / a.Hk, hk = bh - b * a.Hk;
  const int rb = a.rblocks - 1 - (int)blockIdx.y;  // the longest blocks first
  const int c = blockIdx.z;
  const int nrows = a.G * a.T, row0 = rb * RP;
  const WinSpan s = win_span(a, b, row0 / a.G, (min(nrows, row0 + RP) - 1) / a.G + 1);
  const int n = s.count();
  const int per = ((n + a.nchunks - 1) / a.nchunks + SK - 1) / SK * SK;
  const int c0 = min(n, c * per), c1 = min(n, c0 + per);
  if (c0 >= c1 && c > 0) return;  // the merge knows (chunk 0 writes rows without keys)
  const int nst = (c1 - c0 + SK - 1) / SK;

  // ---- rows of this lane: r = row0 + 16 rt + l16
  int pos[RT];
  u32x4 qf[RT][NC];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + 16 * rt + l16, t = r / a.G, h = hk * a.G + (r - t * a.G);
    const bool live = r < nrows && t < s.rows;
    pos[rt] = live ? s.first + t : -1;  // -1 sees nothing
    const char *const qp = (const char *)a.q + ((int64_t)b * a.q_sb + (int64_t)h * a.q_sh +
                                                (int64_t)t * a.q_st) * EB + 16 * g;
#pragma unroll
    for (int k = 0; k < NC; ++k)
      qf[rt][k] = live ? *(const u32x4 *)(qp + 64 * k) : u32x4{0u, 0u, 0u, 0u};
  }
  const int pmin = s.first + row0 / a.G;  // of the block's first row; its last:
  const int pmax = s.first + min(s.rows, (min(nrows, row0 + RP) - 1) / a.G + 1) - 1;
  // call-wide index of a key's score
  const WinSpan whole = a.scores ? win_span(a, b) : s;

  // ---- key sources
  const int64_t kbase = (int64_t)b * a.k_sb + (int64_t)hk * a.k_sh;
  const int64_t vbase = (int64_t)b * a.v_sb + (int64_t)hk * a.v_sh;
  const int32_t *const tab = PAGED ? a.table + (int64_t)b * a.ld_tab : nullptr;
  const int pmask = (a.page_size & (a.page_size - 1)) == 0 ? a.page_size - 1 : -1;

  u32x4 kr[KT][NC], vr[KT][NC];
  int pg[KT];            // pages of the step asked for next
  uint32_t okn = 0u;     // keys present of the step asked for last: bit 16 kt + key
  auto index_of = [&](int st, int kt) { return c0 + st * SK + 16 * kt + l16; };
  auto load_pages = [&](int st) {
    if constexpr (PAGED) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const int i = index_of(st, kt);
        pg[kt] = i < c1 ? tab[s.key(i)] : -1;
      }
    }
  };
  int64_t ko[KT], vo[KT];
  bool ok[KT];
  auto locate = [&](int st) {
    uint32_t m = 0u;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int i = index_of(st, kt), j = s.key(i);
      ok[kt] = i < c1;
      if constexpr (PAGED) {
        ok[kt] = ok[kt] && pg[kt] >= 0 && pg[kt] < a.npages;
        const int in = pmask >= 0 ? (j & pmask) : j % a.page_size;
        ko[kt] = vo[kt] = ((int64_t)pg[kt] * a.p_sp + kbase + (int64_t)in * a.k_st) * EB + 16 * g;
      } else {
        ko[kt] = (kbase + (int64_t)j * a.k_st) * EB + 16 * g;
        vo[kt] = (vbase + (int64_t)j * a.v_st) * EB + 16 * g;
      }
      m |= (uint32_t)(__ballot(ok[kt]) & 0xffffull) << (16 * kt);
    }
    okn = m;
  };
  auto fetch = [&](u32x4 (&r)[KT][NC], const void *base, const int64_t (&off)[KT]) {
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        r[kt][k] = u32x4{0u, 0u, 0u, 0u};
        if (ok[kt]) r[kt][k] = *(const u32x4 *)((const char *)base + off[kt] + 64 * k);
      }
  };

  // ---- state: of row l16 of each tile
  float m[RT], l[RT];
  f32x4 o[RT][D / 16];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  unsigned char *const vl = lds + wave * kRegion;

  if (wave < nst) {
    load_pages(wave);
    locate(wave);
    fetch(kr, a.k, ko);
    fetch(vr, a.v, vo);
    load_pages(wave + NW);
  }
  for (int st = wave; st < nst; st += NW) {
    const uint32_t okm = okn;
    f32x4 sc[RT][KT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          if constexpr (CT == MTP_F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              x = mfma16_f32(__uint_as_float(kr[kt][k][e]), __uint_as_float(qf[rt][k][e]), x);
          } else {
            x = mfma16<CT>(kr[kt][k], qf[rt][k], x);
          }
        }
        sc[rt][kt] = x;
      }
    // V to the wave's rows in LDS
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const int r = 16 * kt + l16;
        *(u32x4 *)(vl + r * RB + 16 * ((4 * k + g) ^ win_swz<CT, RB>(r))) = vr[kt][k];
      }
    const int i0 = c0 + st * SK;
    if (st + NW < nst) {
      locate(st + NW);
      fetch(kr, a.k, ko);
      fetch(vr, a.v, vo);
      load_pages(st + 2 * NW);
    }
    // ---- scores in units of log 2; hidden ones -inf
    const int jlo = s.key(i0), jhi = s.key(min(i0 + SK, c1) - 1);
    const bool all = okm == (KT == 2 ? 0xffffffffu : 0xffffu) && jhi <= pmin &&
                     jlo > pmax - a.window && row0 + RP <= nrows && s.rows == a.T;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        sc[rt][kt] *= a.scale;
        if (!all) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = s.key(i0 + 16 * kt + 4 * g + i);
            const bool see = (((okm >> (16 * kt + 4 * g + i)) & 1u) != 0) & win_sees(a, pos[rt], j);
            sc[rt][kt][i] = see ? sc[rt][kt][i] : -INFINITY;
          }
        }
      }
    }
    if (a.scores) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int r = row0 + 16 * rt + l16;
        float *const sp = a.scores + ((int64_t)bh * nrows + r) * a.ld_sc;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const int i = i0 + 16 * kt + 4 * g;
          if (r >= nrows || i >= c1) continue;
          const int w = whole.index(s.key(i));
          if (i + 3 < c1 && whole.index(s.key(i + 3)) == w + 3) {
            *(f32x4u *)(sp + w) = sc[rt][kt];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (i + e < c1) sp[whole.index(s.key(i + e))] = sc[rt][kt][e];
          }
        }
      }
    }
    // ---- softmax of the step
    u32x4 pb[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float mx = fmaxf(fmaxf(sc[rt][0][0], sc[rt][0][1]), fmaxf(sc[rt][0][2], sc[rt][0][3]));
      if constexpr (KT == 2)
        mx = fmaxf(mx, fmaxf(fmaxf(sc[rt][1][0], sc[rt][1][1]), fmaxf(sc[rt][1][2], sc[rt][1][3])));
      mx = max_over_lane_groups(mx);
      if (__ballot(mx > m[rt] + 8.f) != 0) {
        const float mn = fmaxf(m[rt], mx), ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m[rt] - ref);
        m[rt] = mn;
        l[rt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) o[rt][dt] *= alpha;
      }
      const float ref = m[rt] == -INFINITY ? 0.f : m[rt];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[rt][kt][i] = __builtin_amdgcn_exp2f(sc[rt][kt][i] - ref);
          l[rt] += sc[rt][kt][i];
        }
      if constexpr (CT != MTP_F32) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          pb[rt][2 * kt] = pack2<CT>(sc[rt][kt][0], sc[rt][kt][1]);
          pb[rt][2 * kt + 1] = pack2<CT>(sc[rt][kt][2], sc[rt][kt][3]);
        }
      }
    }
    // ---- O^T += V^T P^T
    win_wave_sync();
    if constexpr (CT == MTP_F32) {
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 16 * kt + 4 * g + i, d = 16 * dt + l16;
            const float v =
                *(const float *)(vl + r * RB + 16 * ((d >> 2) ^ win_swz<CT, RB>(r)) + 4 * (d & 3));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mfma16_f32(v, sc[rt][kt][i], o[rt][dt]);
          }
    } else {
      // 16-lane group g reads rows 4 g + j / 4 (and 16 further) at elements
      // 16 dt + 4 (j % 4) .. + 3
      const int ra = 4 * g + (l16 >> 2), rc = ra + 16;
      const unsigned char *const pa = vl + ra * RB + 8 * (l16 & 1);
      const unsigned char *const pc = vl + rc * RB + 8 * (l16 & 1);
      const int sa = win_swz<CT, RB>(ra), sb = win_swz<CT, RB>(rc);
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        const int ch = 2 * dt + ((l16 & 3) >> 1);
        const uint64_t lo = win_tr16(pa + 16 * (ch ^ sa)), hi = win_tr16(pc + 16 * (ch ^ sb));
        const u32x4 va = {(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mfma16<CT>(va, pb[rt], o[rt][dt]);
      }
    }
    win_wave_sync();
  }

  // ---- the four waves join, one row tile at a time: thread (row, 16 lanes)
  // takes D / 16 elements of a row over the waves in order
  const int mr = th >> 4, md = (th & 15) * 4;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float ls = sum_over_lane_groups(l[rt]);
    __syncthreads();
    float *const so = (float *)lds + wave * 16 * (D + 4) + l16 * (D + 4);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) *(f32x4 *)(so + 16 * dt + 4 * g) = o[rt][dt];
    if (g == 0) {
      s_ml[wave][l16][0] = m[rt];
      s_ml[wave][l16][1] = ls;
    }
    if (th == 0) s_bad[rt] = 0u;
    __syncthreads();
    float M = -INFINITY, L = 0.f, e[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, s_ml[w][mr][0]);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      e[w] = __builtin_amdgcn_exp2f(s_ml[w][mr][0] - ref);
      L = fmaf(s_ml[w][mr][1], e[w], L);
    }
    const int r = row0 + 16 * rt + mr, t = r / a.G, h = hk * a.G + (r - t * a.G);
    if (a.nchunks > 1) {
      if (r < nrows) {
        const int64_t at = (((int64_t)bh * a.rblocks + rb) * a.nchunks + c) * RP + 16 * rt + mr;
        if ((th & 15) == 0) {
          a.pml[at * 2] = M;
          a.pml[at * 2 + 1] = L;
        }
#pragma unroll
        for (int d = md; d < D; d += 64) {
          f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < NW; ++w)
            O += *(const f32x4 *)((float *)lds + (w * 16 + mr) * (D + 4) + d) * e[w];
          *(f32x4 *)(a.part + at * D + d) = O;
        }
      }
      continue;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    bool bad = false;
    if (r < nrows) {
      if (a.scores && (th & 15) == 0) {
        const int64_t at = (int64_t)bh * nrows + r;
        a.ml[at * 2] = M;
        a.ml[at * 2 + 1] = L;
      }
#pragma unroll
      for (int d = md; d < D; d += 64) {
        f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w)
          O += *(const f32x4 *)((float *)lds + (w * 16 + mr) * (D + 4) + d) * e[w];
        O *= inv;
#pragma unroll
        for (int i = 0; i < 4; ++i) bad = bad || !(fabsf(O[i]) < INFINITY);
        win_store4<CT>(a, b, h, t, d, O);
      }
    }
    if (bad) atomicOr(&s_bad[rt], 1u << mr);
  }
  if (a.nchunks > 1) return;
  __syncthreads();
  // ---- rows that are not finite: again without their hidden keys
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    int k = 0;
    for (unsigned bad = s_bad[rt]; bad; bad &= bad - 1, ++k) {
      if (k % NW != wave) continue;
      const int r = row0 + 16 * rt + __builtin_ctz(bad), t = r / a.G;
      win_row<(D + 63) / 64, PAGED>(a, CT, b, hk * a.G + (r - t * a.G), t, s,
                                    (float *)lds + wave * ((win_row_lds(D) + 3) & ~3), false);
    }
  }
}

// Joins the chunks of the split kernel in order, a wave per row.
template <int CT, int D, int RT, bool PAGED>
__global__ void __launch_bounds__(256) win_merge_kernel(const WinArgs a) {
  constexpr int SK = win_split_keys(D * dtype_bytes(CT));
  constexpr int RP = 16 * RT, E = D / 64;
  constexpr int F = 8;  // chunks in flight
  __shared__ float s_row[4][(win_row_lds(D) + 3) & ~3];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nrows = a.G * a.T;
  const int64_t id = (int64_t)blockIdx.x * 4 + wave;
  if (id >= (int64_t)a.B * a.Hk * nrows) return;
  const int bh = (int)(id / nrows), r = (int)(id - (int64_t)bh * nrows);
  const int b = bh / a.Hk, hk = bh - b * a.Hk;
  const int rb = r / RP, row0 = rb * RP, t = r / a.G, h = hk * a.G + (r - t * a.G);
  const WinSpan s = win_span(a, b, row0 / a.G, (min(nrows, row0 + RP) - 1) / a.G + 1);
  const int n = s.count();
  const int per = ((n + a.nchunks - 1) / a.nchunks + SK - 1) / SK * SK;
  const int nc = n > 0 ? (n + per - 1) / per : 1;
  const int64_t base = ((int64_t)bh * a.rblocks + rb) * a.nchunks * RP + (r - row0);
  float M = -INFINITY;
  for (int c = lane; c < nc; c += 64) M = fmaxf(M, a.pml[(base + (int64_t)c * RP) * 2]);
#pragma unroll
  for (int w = 32; w > 0; w >>= 1) M = fmaxf(M, __shfl_xor(M, w, 64));
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int q0 = 0; q0 < nc; q0 += 64) {
    float fm = -INFINITY, fl = 0.f;
    if (q0 + lane < nc) {
      const int64_t at = (base + (int64_t)(q0 + lane) * RP) * 2;
      fm = a.pml[at];
      fl = a.pml[at + 1];
    }
    const float f = __builtin_amdgcn_exp2f(fm - ref);
    L += sum_over_lanes<64>(fl * f);
    const int most = min(64, nc - q0);
    for (int c = 0; c < most; c += F) {
      float x[F][E];
#pragma unroll
      for (int u = 0; u < F; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e)
          x[u][e] = c + u < most ? a.part[(base + (int64_t)(q0 + c + u) * RP) * D + lane + 64 * e]
                                 : 0.f;
#pragma unroll
      for (int u = 0; u < F; ++u) {
        const float fc = __shfl(f, (c + u) & 63, 64);
        if (c + u < most) {
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] = fmaf(x[u][e], fc, o[e]);
        }
      }
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int64_t oo = (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + (int64_t)t * a.o_st;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float y = o[e] * inv;
    bad = bad || !(fabsf(y) < INFINITY);
    store_from_f32(a.out, CT, oo + lane + 64 * e, y);
  }
  if (a.scores && lane == 0) {
    a.ml[id * 2] = M;
    a.ml[id * 2 + 1] = L;
  }
  // not finite: again without the hidden keys
  if (__ballot(bad) != 0) win_row<E, PAGED>(a, CT, b, h, t, s, s_row[wave], false);
}

}  // namespace mtp
