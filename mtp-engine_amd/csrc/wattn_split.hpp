// Windowed attention for few rows and many keys, gfx950: new tokens over a
// paged cache in fp32, bf16 and f16, and the prompts that the prompt kernel
// does not take (fp32 ones above all). Definitions in wattn.hpp.
//
// The G * T rows of a (sequence, key head) - query heads of a group read the
// same keys - go by blocks of 16 * RT (row r = t * G + head); a block's
// visible keys, counted without gaps (WinSpan), are split into nchunks equal
// parts, one per workgroup, so that few rows still fill the chip. The chunks
// join in their order: by the block's last workgroup to arrive, or in
// win_join_kernel where there is more to join (or the weights are wanted).
// Within a workgroup NW waves take steps of SK keys in turn and join at the end;
// a step has no barrier:
//   * K and V rows go from memory to registers, whole rows a load, and from
//     there to the wave's own part of LDS; the next step's rows are asked for
//     as soon as these have left the registers, their pages one step earlier.
//   * S^T[key][row] = K Q^T, 16 x 16 tiles: lane l has keys 4 (l / 16) + i of
//     row l % 16, so a row's maximum takes two lane swaps and its sum none
//     until the end.
//   * O^T[d][row] += V^T P^T takes the S^T registers as they are (rounded to
//     the 16-bit type; fp32 stays); 16-bit V comes from LDS by transposing
//     reads, four keys of one d a lane.
// The running maximum moves only when a step exceeds it by more than 2^8.
//
// Bound of new tokens: HBM, K and V read once per row block (blocks of one key
// head run on one XCD and meet in its L2). 16 KB a wave in flight, two waves per
// SIMD. 131072 keys of 8 heads (537 MB): 87.5 us, 6.1 TB/s; 8 sequences of 1366 ..
// 4096 keys (101 MB): 23.5 us. The first of these with loads in the order of the
// K operand (16 rows of 64 bytes each), without LDS for K: 106 us; with three
// waves per SIMD of smaller chunks: 122. Bound of fp32 prompts: the fp32 matrix
// instructions and the arithmetic beside them, 65 % of the former's peak (T 4096, 8
// heads of 64, no window: 173 us; with a shuffle for every row's address instead
// of scalar arithmetic 192), and the ends of short blocks (B 2, T 1000, window 256,
// 16 heads: 35 us, where they take 16). Blocks of 64 rows: 258 and 40 us.
#pragma once

#include "wattn_weights.hpp"
#include "wstream.hpp"

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

// Keys of each chunk of n keys, in whole steps.
template <int SK>
__device__ __forceinline__ int win_chunk(int n, int nchunks) {
  return max(1, ((n + nchunks - 1) / nchunks + SK - 1) / SK) * SK;
}

template <int CT, int D, int RT, bool PAGED, int NW>
__global__ void __launch_bounds__(64 * NW, 2) win_split_kernel(const WinArgs a) {
  constexpr int EB = dtype_bytes(CT);
  constexpr int RB = D * EB;           // bytes of a row
  constexpr int NC = RB / 64;          // 64-byte pieces of a row
  constexpr int SK = win_split_keys(CT);
  constexpr int KT = SK / 16;          // key tiles of a step
  constexpr int RP = 16 * RT;
  static_assert(RB % 128 == 0 && (CT == MTP_F32 || KT == 2), "whole products");
  constexpr int LPK = RB / 16, KPI = 64 / LPK, NL = SK / KPI;  // loads of K (of V) a step
  constexpr int kRegion = 2 * SK * RB; // a wave's K and V rows
  constexpr int kMerge = NW * 16 * (D + 4) * 4;
  constexpr int kLds = NW * kRegion;
  constexpr int kEnd = NW * 16 * 2 * 4 + 16;
  // two tiles of 256 bytes a row: Q^T from LDS, or the registers run out
  constexpr bool QL = RT == 2 && RB >= 256;
  __shared__ u32x4 s_q[QL ? RT * NC * 64 : 1];
  __shared__ __attribute__((aligned(16))) unsigned char lds[kLds];
  // at its end what is needed once the steps are done: so two workgroups of
  // fp32 rows of 512 bytes fit a CU (B 2, T 405, window 292, 32 heads: 51.6 us against 64.6)
  static_assert(kMerge + kEnd <= kLds, "the join's sums and these");
  float(*const s_ml)[16][2] = (float(*)[16][2])(lds + kLds - kEnd);
  unsigned *const s_bad = (unsigned *)(lds + kLds - 16);
  int *const s_last = (int *)(lds + kLds - 4);

  const int th = threadIdx.x, lane = th & 63;
  const int wave = __builtin_amdgcn_readfirstlane(th >> 6);
  const int g = lane >> 4, l16 = lane & 15;
  const int bh = blockIdx.x, b = bh / a.Hk, hk = bh - b * a.Hk;
  const int rb = a.rblocks - 1 - (int)blockIdx.y;  // the longest blocks first
  const int c = blockIdx.z;
  const int nrows = a.G * a.T, row0 = rb * RP;
  const WinSpan s = win_span(a, b, row0 / a.G, (min(nrows, row0 + RP) - 1) / a.G + 1);
  const int n = s.count();
  const int per = win_chunk<SK>(n, a.nchunks);
  const int c0 = (int)min((int64_t)n, (int64_t)c * per);
  const int c1 = (int)min((int64_t)n, (int64_t)c0 + per);
  const int64_t unit = (((int64_t)bh * a.rblocks + rb) * a.nchunks + c) * RP;  // its rows' partials
  if (c0 >= c1 && a.nchunks > 1 && !a.ticket) {  // a chunk without keys
    if (th < RP) {
      a.pml[(unit + th) * 2] = -INFINITY;
      a.pml[(unit + th) * 2 + 1] = 0.f;
    }
    return;
  }
  const int nst = (c1 - c0 + SK - 1) / SK;

  // ---- rows of this lane: r = row0 + 16 rt + l16
  int pos[RT];
  const char *qp[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + 16 * rt + l16, t = r / a.G, h = hk * a.G + (r - t * a.G);
    const bool live = r < nrows && t < s.rows;
    pos[rt] = live ? s.first + t : -1;  // -1 sees nothing
    qp[rt] = live ? (const char *)a.q + ((int64_t)b * a.q_sb + (int64_t)h * a.q_sh +
                                         (int64_t)t * a.q_st) * EB + 16 * g
                  : nullptr;
  }
  // Q^T: piece k of tile rt, all of them, or (QL) each wave some, shared in LDS
  constexpr int NQ = QL ? (RT * NC + NW - 1) / NW : RT * NC;
  u32x4 qf[NQ];
  auto load_q = [&]() {
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int p = QL ? wave + NW * i : i;
      const char *const at = RT == 2 && p >= NC ? qp[RT - 1] : qp[0];
      qf[i] = u32x4{0u, 0u, 0u, 0u};
      if (at && p < RT * NC) qf[i] = *(const u32x4 *)(at + 64 * (p % NC));
    }
  };
  const int pmin = s.first + row0 / a.G;  // of the block's first row; its last:
  const int pmax = s.first + min(s.rows, (min(nrows, row0 + RP) - 1) / a.G + 1) - 1;
  // call-wide index of a key's score
  const WinSpan whole = a.scores ? win_span(a, b) : s;

  // ---- key sources
  const int64_t kbase = (int64_t)b * a.k_sb + (int64_t)hk * a.k_sh;
  const int64_t vbase = (int64_t)b * a.v_sb + (int64_t)hk * a.v_sh;
  const int32_t *const tab = PAGED ? a.table + (int64_t)b * a.ld_tab : nullptr;
  const int pmask = (a.page_size & (a.page_size - 1)) == 0 ? a.page_size - 1 : -1;

  // Lane i looks up key i % SK of a step; a load instruction takes KPI whole
  // rows, LPK lanes each.
  u32x4 kr[NL], vr[NL];
  int pg = -1;           // page of the step asked for next
  uint32_t okn = 0u;     // keys present of the step asked for last
  auto index_of = [&](int st) { return c0 + st * SK + (lane & (SK - 1)); };
  auto load_pages = [&](int st) {
    if constexpr (PAGED) {
      const int i = index_of(st);
      pg = i < c1 ? tab[s.key(i)] : -1;
    }
  };
  auto shfl64 = [&](int64_t x, int from) {
    return (int64_t)((uint64_t)(uint32_t)__shfl((int)(x >> 32), from, 64) << 32 |
                     (uint32_t)__shfl((int)x, from, 64));
  };
  // dense: the lane's first row and chunk of a step at key 0
  const char *const kd = (const char *)a.k + (kbase + lane / LPK * a.k_st) * EB + 16 * (lane % LPK);
  const char *const vd = (const char *)a.v + (vbase + lane / LPK * a.v_st) * EB + 16 * (lane % LPK);
  auto fetch = [&](int st) {
    if constexpr (!PAGED) {
      const int i0 = c0 + st * SK;
      if (i0 >= s.ns && i0 + SK <= c1) {  // whole, keys in a row: addresses by the scalar unit
        okn = SK == 32 ? 0xffffffffu : 0xffffu;
        const int64_t j0 = s.lo + (i0 - s.ns);
#pragma unroll
        for (int n = 0; n < NL; ++n) {
          kr[n] = ld16(kd + (j0 + n * KPI) * a.k_st * EB);
          vr[n] = ld16(vd + (j0 + n * KPI) * a.v_st * EB);
        }
        return;
      }
    }
    const int i = index_of(st), j = s.key(i);
    bool ok = i < c1;
    int64_t ko, vo;
    if constexpr (PAGED) {
      ok = ok && pg >= 0 && pg < a.npages;
      const int in = pmask >= 0 ? (j & pmask) : j % a.page_size;
      ko = vo = ((int64_t)pg * a.p_sp + kbase + (int64_t)in * a.k_st) * EB;
    } else {
      ko = (kbase + (int64_t)j * a.k_st) * EB;
      vo = (vbase + (int64_t)j * a.v_st) * EB;
    }
    okn = (uint32_t)(__ballot(ok) & (SK == 32 ? 0xffffffffull : 0xffffull));
    // a cache is read once; a prompt's keys again by the next row block
    auto row16 = [](const void *p, int64_t off) {
      return PAGED ? ld_nt16((const char *)p + off) : ld16((const char *)p + off);
    };
    const bool every = okn == (SK == 32 ? 0xffffffffu : 0xffffu);  // the usual step
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int r = n * KPI + lane / LPK;
      const int64_t c16 = 16 * (lane % LPK);
      const int64_t kof = shfl64(ko, r) + c16, vof = PAGED ? kof : shfl64(vo, r) + c16;
      if (every) {
        kr[n] = row16(a.k, kof);
        vr[n] = row16(a.v, vof);
      } else {
        kr[n] = vr[n] = u32x4{0u, 0u, 0u, 0u};
        if ((okn >> r) & 1u) {
          kr[n] = row16(a.k, kof);
          vr[n] = row16(a.v, vof);
        }
      }
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
  unsigned char *const kl = lds + wave * kRegion, *const vl = kl + SK * RB;

  load_pages(wave);
  load_q();
  if (wave < nst) {
    fetch(wave);
    load_pages(wave + NW);
  }
  if constexpr (QL) {
#pragma unroll
    for (int i = 0; i < NQ; ++i)
      if (wave + NW * i < RT * NC) s_q[(wave + NW * i) * 64 + lane] = qf[i];
    lds_barrier();  // loads in flight go on
  }
  for (int st = wave; st < nst; st += NW) {
    const uint32_t okm = okn;
    const int i0 = c0 + st * SK;
    // rows to the wave's part of LDS
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int r = n * KPI + lane / LPK;
      const int at = r * RB + 16 * ((lane % LPK) ^ win_swz<CT, RB>(r));
      *(u32x4 *)(kl + at) = kr[n];
      *(u32x4 *)(vl + at) = vr[n];
    }
    if (st + NW < nst) {
      fetch(st + NW);
      load_pages(st + 2 * NW);
    }
    win_wave_sync();
    f32x4 sc[RT][KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int r = 16 * kt + l16;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) sc[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const u32x4 x = *(const u32x4 *)(kl + r * RB + 16 * ((4 * k + g) ^ win_swz<CT, RB>(r)));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          u32x4 y;
          if constexpr (QL) y = s_q[(rt * NC + k) * 64 + lane];
          else y = qf[rt * NC + k];
          if constexpr (CT == MTP_F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              sc[rt][kt] = mfma16_f32(__uint_as_float(x[e]), __uint_as_float(y[e]), sc[rt][kt]);
          } else {
            sc[rt][kt] = mfma16<CT>(x, y, sc[rt][kt]);
          }
        }
      }
    }
    // ---- scores in units of log 2; hidden ones -inf
    const int jlo = s.key(i0), jhi = s.key(min(i0 + SK, c1) - 1);
    // a step that every row sees whole; a row that is no query's keeps what it
    // has and is dropped at the end
    const bool all =
        okm == (KT == 2 ? 0xffffffffu : 0xffffu) && jhi <= pmin && jlo > pmax - a.window;
    const bool line = jlo >= a.sinks;  // keys jlo, jlo + 1, ...
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        sc[rt][kt] *= a.scale;
        if (!all) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = 16 * kt + 4 * g + i, j = line ? jlo + c : s.key(i0 + c);
            const bool see = (((okm >> c) & 1u) != 0) & win_sees(a, pos[rt], j);
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
          if (line && i0 + SK <= c1) {
            *(f32x4u *)(sp + whole.index(jlo) + (i - i0)) = sc[rt][kt];
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

  // the block's partials, with tickets: 16 bytes a lane at the device's
  // coherence point (the hand-off of mtp_common.hpp)
  const __amdgpu_buffer_rsrc_t prs =
      make_rsrc(a.part + (unit - (int64_t)c * RP) * D,
                a.ticket ? (uint32_t)a.nchunks * (uint32_t)(RP * D * 4) : 0u);
  // ---- the waves join, one row tile at a time: TR threads to a row, each
  // takes some of its elements over the waves in order
  constexpr int TR = 4 * NW;
  const int mr = th / TR, mt = th % TR, md = mt * 4;
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
    const int64_t at = unit + 16 * rt + mr;
    const bool query = r < nrows && t < s.rows;
    if (!query) M = -INFINITY, L = 0.f;
    if (mt == 0 && a.ticket) {
      pub_f32(a.pml + at * 2, M);
      pub_f32(a.pml + at * 2 + 1, L);
    } else if (mt == 0 && (a.nchunks > 1 || a.scores)) {
      a.pml[at * 2] = M;
      a.pml[at * 2 + 1] = L;
    }
    if (a.nchunks > 1) {
      if (r < nrows) {
#pragma unroll
        for (int d = md; d < D; d += 4 * TR) {
          f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < NW; ++w)
            O += *(const f32x4 *)((float *)lds + (w * 16 + mr) * (D + 4) + d) * e[w];
          if (a.ticket) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, O), prs,
                                                   (uint32_t)((c * RP + 16 * rt + mr) * D + d) * 4u,
                                                   0, kSc1);
          } else {
            *(f32x4 *)(a.part + at * D + d) = O;
          }
        }
      }
      continue;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    bool bad = false;
    if (r < nrows) {
#pragma unroll
      for (int d = md; d < D; d += 4 * TR) {
        f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w)
          O += *(const f32x4 *)((float *)lds + (w * 16 + mr) * (D + 4) + d) * e[w];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          O[i] = query ? O[i] * inv : 0.f;
          bad = bad || !(fabsf(O[i]) < INFINITY);
        }
        win_store4<CT>(a, b, h, t, d, O);
      }
    }
    if (bad) atomicOr(&s_bad[rt], 1u << mr);
  }
  if (a.nchunks > 1) {
    if (!a.ticket) return;
    // ---- the last workgroup of the block to arrive joins its chunks, in order
    wait_stores();
    __syncthreads();
    unsigned *const tk = a.ticket + (int64_t)bh * a.rblocks + rb;
    if (th == 0) *s_last = ticket_add(tk) == (unsigned)a.nchunks - 1;
    __syncthreads();
    if (!*s_last) return;
    if (th == 0) ticket_reset(tk);
    const int64_t base = unit - (int64_t)c * RP;  // the block's first chunk
    const int nr = min(RP, nrows - row0), nc = a.nchunks;
    float *const s_f = (float *)lds;  // [row][chunk] maximum, sum
    static_assert(RP * kWinTicketChunks * 8 + kEnd <= kLds, "the chunks' maxima and sums");
    constexpr int F = 8, Q = D / 4;  // chunks in flight; four elements a thread
    auto fetch4 = [&](f32x4 (&x)[F], int q0, int i) {
#pragma unroll
      for (int u = 0; u < F; ++u)
        x[u] = __builtin_bit_cast(
            f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                       prs, (uint32_t)((min(q0 + u, nc - 1) * RP + i / Q) * D + i % Q * 4) * 4u, 0,
                       kSc1));
    };
    f32x4 x[F];
    fetch4(x, 0, min(th, nr * Q - 1));
    for (int i = th; i < nr * nc; i += 64 * NW) {
      const int64_t at = (base + (int64_t)(i % nc) * RP + i / nc) * 2;
      s_f[2 * i] = get_f32(a.pml + at);
      s_f[2 * i + 1] = get_f32(a.pml + at + 1);
    }
    __syncthreads();
    for (int i = th; i < nr * Q; i += 64 * NW) {
      if (i != th) fetch4(x, 0, i);
      const int rr = i / Q, d = i % Q * 4;
      const float *const f = s_f + 2 * rr * nc;
      float M = -INFINITY, L = 0.f;
      f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int q = 0; q < nc; ++q) M = fmaxf(M, f[2 * q]);
      const float ref = M == -INFINITY ? 0.f : M;
      for (int q0 = 0; q0 < nc; q0 += F) {
        f32x4 y[F];
#pragma unroll
        for (int u = 0; u < F; ++u) y[u] = x[u];
        if (q0 + F < nc) fetch4(x, q0 + F, i);
#pragma unroll
        for (int u = 0; u < F; ++u) {
          if (q0 + u < nc) {
            const float e = __builtin_amdgcn_exp2f(f[2 * (q0 + u)] - ref);
            L = fmaf(f[2 * (q0 + u) + 1], e, L);
            if (e != 0.f) O += y[u] * e;
          }
        }
      }
      const int r = row0 + rr, t = r / a.G, h = hk * a.G + (r - t * a.G);
      const float inv = L == 0.f ? 0.f : 1.f / L;
      bool bad = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        O[j] *= inv;
        bad = bad || !(fabsf(O[j]) < INFINITY);
      }
      win_store4<CT>(a, b, h, t, d, O);
      if (bad) atomicOr(&s_bad[rr / 16], 1u << (rr % 16));
    }
  }
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

// Joins the chunks of the split kernel: W waves per row take chunks w, w + W,
// ... and join in order; workgroups from a.joins on add to the weights.
template <int CT, int D, bool PAGED, int W>
__global__ void __launch_bounds__(256) win_join_kernel(const WinArgs a) {
  constexpr int E = D / 64;
  constexpr int F = 8;  // chunks in flight
  __shared__ __attribute__((aligned(16))) float s_row[4][(win_row_lds(D) + 3) & ~3];
  __shared__ float s_a[256], s_b[256];
  if ((int)blockIdx.x >= a.joins) {
    const int id = (int)blockIdx.x - a.joins, kbs = (int)((a.ld_sc + 255) / 256);
    win_weights(a, id / kbs, id % kbs, s_a, s_b);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nrows = a.G * a.T;
  const int64_t id = ((int64_t)blockIdx.x * 4 + wave) / W;
  const int w = wave % W;
  const bool live = id < (int64_t)a.B * a.Hk * nrows;  // of a whole row: W divides 4
  const int bh = live ? (int)(id / nrows) : 0, r = live ? (int)(id - (int64_t)bh * nrows) : 0;
  const int b = bh / a.Hk, hk = bh - b * a.Hk;
  const int rb = r / a.rp, t = r / a.G, h = hk * a.G + (r - t * a.G);
  const int nc = live ? a.nchunks : 0;
  const int64_t base = ((int64_t)bh * a.rblocks + rb) * a.nchunks * a.rp + (r - rb * a.rp);
  float M = -INFINITY;
  for (int c = lane; c < nc; c += 64) M = fmaxf(M, a.pml[(base + (int64_t)c * a.rp) * 2]);
  float L = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  float ref = 0.f;
  // chunk w + W (q0 + lane) in lane `lane`; a chunk without keys (-inf) has
  // written no row
  for (int q0 = 0; w + W * q0 < nc; q0 += 64) {
    float fm = -INFINITY, fl = 0.f;
    const int mine = w + W * (q0 + lane);
    if (mine < nc) {
      const int64_t at = (base + (int64_t)mine * a.rp) * 2;
      fm = a.pml[at];
      fl = a.pml[at + 1];
    }
    const int most = min(64, (nc - w - W * q0 + W - 1) / W);
    float f = 0.f;
    for (int c = 0; c < most; c += F) {
      float x[F][E];
#pragma unroll
      for (int u = 0; u < F; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          x[u][e] = 0.f;
          if (c + u < most)
            x[u][e] =
                a.part[(base + (int64_t)(w + W * (q0 + c + u)) * a.rp) * D + lane + 64 * e];
        }
      if (c == 0) {  // the maximum of the row, while the first chunks are on their way
        if (q0 == 0) {
#pragma unroll
          for (int y = 32; y > 0; y >>= 1) M = fmaxf(M, __shfl_xor(M, y, 64));
          ref = M == -INFINITY ? 0.f : M;
        }
        f = __builtin_amdgcn_exp2f(fm - ref);
        L += sum_over_lanes<64>(fl * f);
      }
#pragma unroll
      for (int u = 0; u < F; ++u) {
        const float fc = __shfl(f, (c + u) & 63, 64);
        const bool has = c + u < most && fc != 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = has ? fmaf(x[u][e], fc, o[e]) : o[e];
      }
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) s_row[wave][lane + 64 * e] = o[e];
    if (lane == 0) s_a[wave] = L;
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (int x = 1; x < W; ++x) {
      L += s_a[wave + x];
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += s_row[wave + x][lane + 64 * e];
    }
  }
  if (!live) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int64_t oo = (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + (int64_t)t * a.o_st;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float y = o[e] * inv;
    bad = bad || !(fabsf(y) < INFINITY);
    store_from_f32(a.out, CT, oo + lane + 64 * e, y);
  }
  // not finite: again without the hidden keys
  if (__ballot(bad) != 0)
    win_row<E, PAGED>(a, CT, b, h, t, win_span(a, b), s_row[wave], false);
}

}  // namespace mtp
