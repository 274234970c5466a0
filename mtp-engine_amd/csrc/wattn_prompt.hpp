// Windowed attention of prompts, gfx950: many rows against dense 16-bit keys
// at head dims 64 and 128. Definitions in wattn.hpp.
//
// The G * T rows of a (sequence, key head) - row r = t * G + head, so the heads
// of a group share every key - go by blocks of 32 * NW, one workgroup each,
// wave w the rows 32 w .. + 31; the block's visible keys, counted without gaps
// (WinSpan), by tiles of 64:
//   * K and V rows go from memory to LDS by buffer loads with the LDS bit, tile
//     i + 1 while tile i is multiplied; a key past the span reads zeros. Chunk
//     c of a row (16 bytes) lies at c ^ win_swz(row), which the load picks by
//     its source address.
//   * S^T[key][row] = K Q^T on v_mfma_f32_32x32x16, Q^T in registers: lane l
//     has 16 keys 8 (v / 4) + 4 (l / 32) + v % 4 of row l % 32, so a row's
//     maximum takes one lane swap and its sum none until the end.
//   * O^T[d][row] += V^T P^T with the S^T registers, rounded to the 16-bit
//     type, as they are; V^T from the rows in LDS by transposing reads.
// Few blocks behind many keys go with their keys in chunks, one a workgroup, which
// win_join_kernel joins: T 512, 32 / 8 heads, D 128: 32768 keys 307 us (890
// TFLOP/s), 8192 keys 92.6; whole 733 and 170.
// The running maximum moves only when a tile exceeds it by more than 2^8. A
// wave passes over a tile that none of its rows sees. Only tiles at the edge
// of a wave's window compare positions.
//
// Blocks of four waves, two of them on a CU, so that one multiplies while the
// other is in its softmax: 128 rows against one block of 256 on a CU: 37.5 us
// against 43.5 (B 4, T 1025, L 2049, H 16, D 64), 85 against 90 (T 4096,
// window 1024, H 32 / 8, D 128), 420 against 418 (T 8192, window 4096).
#pragma once

#include "wattn_split.hpp"

namespace mtp {

typedef __attribute__((ext_vector_type(16))) float win_f32x16;

template <int CT>
__device__ __forceinline__ win_f32x16 win_mfma32(u32x4 a, u32x4 b, win_f32x16 c) {
  if constexpr (CT == MTP_BF16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// 16 bytes a lane from the buffer to LDS, lane i at lds + 16 i.
__device__ __forceinline__ void win_dma16(__amdgpu_buffer_rsrc_t r, unsigned char *lds,
                                          uint32_t voff) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16,
                                           voff, 0, 0, 0);
#else
  (void)r; (void)lds; (void)voff;
#endif
}

template <int CT, int D, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 2)))
win_prompt_kernel(const WinArgs a) {
  constexpr int RB = 2 * D;              // bytes of a row
  constexpr int SK = kWinTileKeys;       // keys of a tile
  constexpr int KBY = SK * RB;           // K bytes of a tile
  constexpr int RPI = 1024 / RB;         // rows of a copy instruction
  constexpr int NI = SK / RPI / NW;      // copy instructions of K (of V) per wave and tile
  constexpr int RP = 32 * NW;            // rows of a block
  static_assert(NI >= 1 && NI * NW * RPI == SK, "whole copies");
  // One dynamic array, bytes of win_prompt_lds(): with a second LDS variable the
  // compiler lets every LDS read wait for the copies in flight.
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];

  const int th = threadIdx.x, lane = th & 63;
  const int wave = __builtin_amdgcn_readfirstlane(th >> 6);
  const int hi = lane >> 5, l32 = lane & 31;
  const int bh = blockIdx.x, b = bh / a.Hk, hk = bh - b * a.Hk;
  const int rb = a.rblocks - 1 - (int)blockIdx.y;  // the longest blocks first
  const int nrows = a.G * a.T, row0 = rb * RP;
  const WinSpan s = win_span(a, b, row0 / a.G, (min(nrows, row0 + RP) - 1) / a.G + 1);
  const int n = s.count();
  // the tiles of this chunk of the block's keys
  const int per = ((n + SK - 1) / SK + a.nchunks - 1) / a.nchunks;
  const int first = min((int)blockIdx.z * per, (n + SK - 1) / SK);
  const int last = min(first + per, (n + SK - 1) / SK);

  // ---- the wave's rows, and the positions of its first and last live one
  const int r = row0 + 32 * wave + l32, t = r / a.G, h = hk * a.G + (r - t * a.G);
  const bool live = r < nrows && t < s.rows;
  const int pos = live ? s.first + t : -1;  // -1 sees nothing
  const int w0 = row0 + 32 * wave;
  const bool idle = w0 >= nrows || w0 / a.G >= s.rows;
  const int pmin = s.first + w0 / a.G;
  const int pmax = s.first + min(s.rows, (min(nrows, w0 + 32) - 1) / a.G + 1) - 1;
  u32x4 qf[D / 16];
  {
    const uint16_t *const qp = (const uint16_t *)a.q + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh +
                               (int64_t)t * a.q_st + 8 * hi;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
      qf[k] = live ? *(const u32x4 *)(qp + 16 * k) : u32x4{0u, 0u, 0u, 0u};
  }

  // ---- copies
  const uint32_t kst = (uint32_t)a.k_st * 2u, vst = (uint32_t)a.v_st * 2u;
  const __amdgpu_buffer_rsrc_t krs =
      make_rsrc((const uint16_t *)a.k + (int64_t)b * a.k_sb + (int64_t)hk * a.k_sh,
                (uint32_t)(a.L - 1) * kst + RB);
  const __amdgpu_buffer_rsrc_t vrs =
      make_rsrc((const uint16_t *)a.v + (int64_t)b * a.v_sb + (int64_t)hk * a.v_sh,
                (uint32_t)(a.L - 1) * vst + RB);
  auto issue = [&](int tile, int buf) {
    unsigned char *const kb = lds + buf * 2 * KBY;
#pragma unroll
    for (int u = 0; u < NI; ++u) {
      const int in = wave + NW * u;
      const int row = in * RPI + lane / (RB / 16);
      const uint32_t ch = 16u * (uint32_t)((lane % (RB / 16)) ^ win_swz<CT, RB>(row));
      const int i = tile * SK + row;
      const uint32_t j = (uint32_t)s.key(i);
      win_dma16(krs, kb + in * 1024, i < n ? j * kst + ch : kOOB);
      win_dma16(vrs, kb + KBY + in * 1024, i < n ? j * vst + ch : kOOB);
    }
  };

  float m = -INFINITY, l = 0.f;
  win_f32x16 o[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[dt][v] = 0.f;

  auto compute = [&](int tile, int buf) {
    const int i0 = tile * SK;
    const int jlo = s.key(i0), jhi = s.key(min(i0 + SK, n) - 1);
    if (idle || jlo > pmax || (jhi <= pmin - a.window && jlo >= a.sinks)) return;  // wave-uniform
    const unsigned char *const kb = lds + buf * 2 * KBY, *const vb = kb + KBY;
    win_f32x16 sc[SK / 32];
#pragma unroll
    for (int u = 0; u < SK / 32; ++u) {
#pragma unroll
      for (int v = 0; v < 16; ++v) sc[u][v] = 0.f;
      const int kr = 32 * u + l32;
      const unsigned char *const krow = kb + kr * RB;
      const int sw = win_swz<CT, RB>(kr);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        sc[u] = win_mfma32<CT>(*(const u32x4 *)(krow + 16 * ((2 * k + hi) ^ sw)), qf[k], sc[u]);
    }
    // hidden scores -inf; a row that is no query's keeps what it has and is
    // dropped at the end
    if (!(jhi <= pmin && jlo > pmax - a.window && i0 + SK <= n)) {
      if (jlo >= a.sinks && jhi - jlo < SK) {
        // the window alone: distances below the row's position
        const int d = pos - jlo - 4 * hi, e = min(pos, s.key(n - 1)) - jlo - 4 * hi;
#pragma unroll
        for (int u = 0; u < SK / 32; ++u)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int c = 32 * u + 8 * (v >> 2) + (v & 3);
            sc[u][v] = (c <= e) & (c > d - a.window) ? sc[u][v] : -INFINITY;
          }
      } else {
#pragma unroll
        for (int u = 0; u < SK / 32; ++u)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int i = i0 + 32 * u + 8 * (v >> 2) + 4 * hi + (v & 3);
            sc[u][v] = (i < n) & win_sees(a, pos, s.key(i)) ? sc[u][v] : -INFINITY;
          }
      }
    }
    float mx = sc[0][0];
#pragma unroll
    for (int u = 0; u < SK / 32; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) mx = fmaxf(mx, sc[u][v]);
    {
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx),
                                                       false, false);
      mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * a.scale;
    }
    if (__ballot(mx > m + 8.f) != 0) {
      const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - ref);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) o[dt] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    u32x4 pb[SK / 16];
#pragma unroll
    for (int u = 0; u < SK / 32; ++u) {
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        sc[u][v] = __builtin_amdgcn_exp2f(fmaf(sc[u][v], a.scale, -ref));
        l += sc[u][v];
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          pb[2 * u + s2][i] = pack2<CT>(sc[u][8 * s2 + 2 * i], sc[u][8 * s2 + 2 * i + 1]);
    }
    // 16-lane group G reads rows 4 (G / 2) + j / 4 (and 8 further) of a
    // 16-key step, elements 32 dt + 16 (G % 2) + 4 (j % 4) .. + 3
    const int G = lane >> 4, j = lane & 15;
#pragma unroll
    for (int s2 = 0; s2 < SK / 16; ++s2) {
      const int ra = 16 * s2 + 4 * (G >> 1) + (j >> 2), rc = ra + 8;
      const unsigned char *const pa = vb + ra * RB + 8 * (j & 1);
      const unsigned char *const pc = vb + rc * RB + 8 * (j & 1);
      const int sa = win_swz<CT, RB>(ra), sb = win_swz<CT, RB>(rc);
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) {
        const int ch = 4 * dt + 2 * (G & 1) + ((j & 3) >> 1);
        const uint64_t lo = win_tr16(pa + 16 * (ch ^ sa)), up = win_tr16(pc + 16 * (ch ^ sb));
        const u32x4 va = {(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)up, (uint32_t)(up >> 32)};
        o[dt] = win_mfma32<CT>(va, pb[s2], o[dt]);
      }
    }
  };

  // Q in registers before the copies go out (its wait then counts no copy)
#pragma unroll
  for (int k = 0; k < D / 16; ++k) asm volatile("" ::"v"(qf[k]));
  if (first < last) issue(first, first & 1);
  for (int i = first; i < last; ++i) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (i + 1 < last) issue(i + 1, (i + 1) & 1);
    compute(i, i & 1);
  }

  // ---- rows out: lane holds d = 32 dt + 8 (v / 4) + 4 hi + v % 4 of its row
  {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false,
                                                     false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  if (a.nchunks > 1) {  // partials for win_join_kernel, which reads none of a chunk without keys
    const int64_t at =
        (((int64_t)bh * a.rblocks + rb) * a.nchunks + blockIdx.z) * RP + 32 * wave + l32;
    if (r >= nrows) return;
    if (hi == 0) {
      a.pml[at * 2] = live ? m : -INFINITY;
      a.pml[at * 2 + 1] = live ? l : 0.f;
    }
    if (!live || first >= last) return;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
        *(f32x4 *)(a.part + at * D + 32 * dt + 8 * r4 + 4 * hi) =
            f32x4{o[dt][4 * r4], o[dt][4 * r4 + 1], o[dt][4 * r4 + 2], o[dt][4 * r4 + 3]};
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  bool bad = false;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) {
    o[dt] *= inv;
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      f32x4 x = {o[dt][4 * r4], o[dt][4 * r4 + 1], o[dt][4 * r4 + 2], o[dt][4 * r4 + 3]};
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        x[v] = live ? x[v] : 0.f;
        bad = bad || !(fabsf(x[v]) < INFINITY);
      }
      if (r < nrows) win_store4<CT>(a, b, h, t, 32 * dt + 8 * r4 + 4 * hi, x);
    }
  }
  const unsigned long long wrong = __ballot(bad && r < nrows);
  __syncthreads();  // every wave is past its tiles: their LDS is free
  // rows that are not finite: again without their hidden keys
  for (unsigned x = (unsigned)wrong | (unsigned)(wrong >> 32); x; x &= x - 1) {
    const int rr = w0 + __builtin_ctz(x), tt = rr / a.G;
    win_row<D / 64, false>(a, CT, b, hk * a.G + (rr - tt * a.G), tt, s,
                           (float *)lds + wave * ((win_row_lds(D) + 3) & ~3), false);
  }
}

}  // namespace mtp
