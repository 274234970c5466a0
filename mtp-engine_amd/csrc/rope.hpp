// Norms of queries and keys for each head with the position rotation in the
// same pass, gfx950; on request keys and values go straight into their pages.
//
//   y = x * rsqrt(mean_d(x^2) + eps) * w[d]       (norm off: y = x)
//   (y_a, y_b) -> (y_a cos t - y_b sin t, y_b cos t + y_a sin t),
//   t = position * inv_freq[i], for the rot / 2 pairs i of the first rot
//   elements: (a, b) = (i, i + rot / 2), or (2 i, 2 i + 1) when interleaved;
//   elements from rot on are normed only.
//
// The angle is reduced in 64 bits: position * inv_freq / 2 pi, less its
// nearest whole number, so a position of some hundred thousand costs no
// accuracy (fp32 would leave an error of position * 2^-24 radians). sin and
// cos of the rest, the norm and the rotation are fp32; an output is rounded
// once.
//
// Bound: HBM, each row read and written once. A row of D elements lies over
// LPR lanes, 16 bytes each, so a wave takes 64 / LPR rows at a time; a wave
// stays with one token, whose D / 2 angles its lanes compute once and keep
// for all of the token's heads. In the half form the partner element of a
// pair is the same place of another lane's 16 bytes: the raw row is
// exchanged (half the lane traffic of fp32 values) and normed on both sides.
#pragma once

#include "mtp_common.hpp"

namespace mtp {

struct RopeArgs {
  const void *q, *k, *v;  // [B, H or Hk, T, D] by element strides, d contiguous; v null: no pages
  int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st;
  void *qo, *ko;          // outputs by element strides; ko null: keys go to the pages
  int64_t qo_sb, qo_sh, qo_st, ko_sb, ko_sh, ko_st;
  void *k_pages, *v_pages;  // [P, B, Hk, page_size, D]
  int64_t p_sp, p_sb, p_sh;
  const int32_t *table;   // [B, ld_tab]
  int64_t ld_tab;
  int page_size, npages;
  const void *inv_freq;   // [rot / 2], fp32 or (freq64) fp64
  int freq64;
  const float *wq, *wk;   // [D] or null (ones)
  const int64_t *pos;     // [*, T] positions, or null: start + t
  int64_t pos_sb;
  const int64_t *start_dev;
  int start_per_row;
  int64_t start_host;
  int B, T, H, Hk, D, rot, norm, interleaved;
  int hs;                 // waves per token
  float eps;
};

// sin and cos of position * inv_freq[i].
__device__ __forceinline__ void rope_angle(const RopeArgs &a, int64_t pos, int i, float &s,
                                           float &c) {
  const double f = a.freq64 ? ((const double *)a.inv_freq)[i]
                            : (double)((const float *)a.inv_freq)[i];
  const double turns = (double)pos * (f * 0.15915494309189533577);
  sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
}

// Where token (b, t) is stored in the pages of its row, or -1.
__device__ __forceinline__ int64_t rope_slot(const RopeArgs &a, int b, int64_t at) {
  if (at < 0 || at >= a.ld_tab) return -1;
  const int page = a.table[(int64_t)b * a.ld_tab + at];
  if (page < 0 || page >= a.npages) return -1;
  return (int64_t)page * a.p_sp + (int64_t)b * a.p_sb + (int64_t)(at % a.page_size) * a.D;
}

template <int DT>
__device__ __forceinline__ void rope_unpack(u32x4 w, float *f) {
  if constexpr (DT == MTP_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 p = unpack2<DT>(w[i]);
      f[2 * i] = p[0];
      f[2 * i + 1] = p[1];
    }
  }
}
template <int DT>
__device__ __forceinline__ u32x4 rope_pack(const float *f) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == MTP_F32) w[i] = __float_as_uint(f[i]);
    else w[i] = pack2<DT>(f[2 * i], f[2 * i + 1]);
  }
  return w;
}

// 16-byte form: rows of whole 16-byte chunks, at most LPR of them, every
// pair's halves in whole chunks. Wave (token, part) takes the rows part *
// RPI + i of the token, then every hs * RPI further on.
template <int DT, int LPR, bool INTER>
__global__ void __launch_bounds__(256) rope_kernel(const RopeArgs a) {
  constexpr int VEC = 16 / dtype_bytes(DT);
  constexpr int RPI = 64 / LPR;
  constexpr int U = 4;  // rows of a lane in flight
  const int lane = threadIdx.x & 63;
  const int64_t wid = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t tok = wid / a.hs;
  const int part = (int)(wid % a.hs);
  if (tok >= (int64_t)a.B * a.T) return;
  const int b = (int)(tok / a.T), t = (int)(tok % a.T);
  const int c = lane % LPR, d0 = c * VEC;
  const bool on = d0 < a.D;
  const int64_t start = a.start_dev ? a.start_dev[a.start_per_row ? b : 0] : a.start_host;
  const int64_t at = start + t;
  const int64_t pos = a.pos ? a.pos[(int64_t)b * a.pos_sb + t] : at;
  const int64_t slot = a.v ? rope_slot(a, b, at) : -1;
  const int nqk = a.H + a.Hk, nr = nqk + (a.v ? a.Hk : 0);

  // angles of the lane's elements (a pair shares one)
  constexpr int NF = INTER ? VEC / 2 : VEC;
  float cs[NF], sn[NF];
  const int half = a.rot >> 1;
  const bool rotated = d0 < a.rot;
  const int f0 = INTER ? d0 / 2 : (d0 < half ? d0 : d0 - half);
#pragma unroll
  for (int i = 0; i < NF; ++i) {
    cs[i] = 1.f;
    sn[i] = 0.f;
    if (on && rotated) rope_angle(a, pos, f0 + i, sn[i], cs[i]);
    if (!INTER && d0 < half) sn[i] = -sn[i];  // the first of a pair loses y_b sin t
  }
  const int hc = half / VEC;
  const int mate = INTER || !rotated ? lane : (d0 < half ? lane + hc : lane - hc);
  const int m0 = d0 + (mate - lane) * VEC;  // the partner's first element
  const float inv_d = 1.f / (float)a.D;

  auto src_of = [&](int r) -> const char * {
    int64_t off;
    const char *p;
    if (r < a.H) {
      p = (const char *)a.q;
      off = (int64_t)b * a.q_sb + (int64_t)r * a.q_sh + (int64_t)t * a.q_st;
    } else if (r < nqk) {
      p = (const char *)a.k;
      off = (int64_t)b * a.k_sb + (int64_t)(r - a.H) * a.k_sh + (int64_t)t * a.k_st;
    } else {
      p = (const char *)a.v;
      off = (int64_t)b * a.v_sb + (int64_t)(r - nqk) * a.v_sh + (int64_t)t * a.v_st;
    }
    return p + (off + d0) * dtype_bytes(DT);
  };
  auto dst_of = [&](int r) -> char * {
    int64_t off;
    char *p;
    if (r < a.H) {
      p = (char *)a.qo;
      off = (int64_t)b * a.qo_sb + (int64_t)r * a.qo_sh + (int64_t)t * a.qo_st;
    } else if (a.ko && r < nqk) {
      p = (char *)a.ko;
      off = (int64_t)b * a.ko_sb + (int64_t)(r - a.H) * a.ko_sh + (int64_t)t * a.ko_st;
    } else {
      if (slot < 0) return nullptr;
      p = (char *)(r < nqk ? a.k_pages : a.v_pages);
      off = slot + (int64_t)(r < nqk ? r - a.H : r - nqk) * a.p_sh;
    }
    return p + (off + d0) * dtype_bytes(DT);
  };

  for (int r0 = part * RPI + lane / LPR; r0 - lane / LPR < nr; r0 += U * a.hs * RPI) {
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * a.hs * RPI;
      w[u] = u32x4{0u, 0u, 0u, 0u};
      if (on && r < nr) w[u] = *(const u32x4 *)src_of(r);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * a.hs * RPI;
      if (r - lane / LPR >= nr) break;  // wave-uniform
      float x[VEC], y[VEC];
      rope_unpack<DT>(w[u], x);
      float rs = 1.f;
      if (a.norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) ss = fmaf(x[i], x[i], ss);
        rs = rsqrtf(sum_over_lanes<LPR>(ss) * inv_d + a.eps);
      }
      const float *const g = r < a.H ? a.wq : a.wk;
      const bool gain = a.norm && g != nullptr;
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] *= rs * (gain && on ? g[d0 + i] : 1.f);
      if constexpr (INTER) {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          y[i] = x[i] * cs[i / 2] - x[i + 1] * sn[i / 2];
          y[i + 1] = x[i + 1] * cs[i / 2] + x[i] * sn[i / 2];
        }
      } else {
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __shfl(w[u][i], mate, 64);
        rope_unpack<DT>(o, y);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float z = y[i] * (rs * (gain && on ? g[m0 + i] : 1.f));
          y[i] = rotated ? x[i] * cs[i] + z * sn[i] : x[i];
        }
      }
      if (on && r < nr)
        if (char *const p = dst_of(r)) *(u32x4 *)p = r < nqk ? rope_pack<DT>(y) : w[u];
    }
  }
}

// Any sizes and strides: one wave per row, the normed row in LDS.
constexpr int kRopeMaxD = 4096;
__global__ void __launch_bounds__(64) rope_generic_kernel(const RopeArgs a, int dt) {
  __shared__ float s_y[kRopeMaxD];
  const int lane = threadIdx.x;
  const int nqk = a.H + a.Hk, nr = nqk + (a.v ? a.Hk : 0);
  const int r = (int)(blockIdx.x % (unsigned)nr);
  const int64_t tok = blockIdx.x / (unsigned)nr;
  const int b = (int)(tok / a.T), t = (int)(tok % a.T);
  const int64_t start = a.start_dev ? a.start_dev[a.start_per_row ? b : 0] : a.start_host;
  const int64_t pos = a.pos ? a.pos[(int64_t)b * a.pos_sb + t] : start + t;
  const void *src;
  void *dst;
  int64_t so, dof;
  if (r < a.H) {
    src = a.q;
    so = (int64_t)b * a.q_sb + (int64_t)r * a.q_sh + (int64_t)t * a.q_st;
    dst = a.qo;
    dof = (int64_t)b * a.qo_sb + (int64_t)r * a.qo_sh + (int64_t)t * a.qo_st;
  } else {
    const int h = r < nqk ? r - a.H : r - nqk;
    src = r < nqk ? a.k : a.v;
    so = r < nqk ? (int64_t)b * a.k_sb + (int64_t)h * a.k_sh + (int64_t)t * a.k_st
                 : (int64_t)b * a.v_sb + (int64_t)h * a.v_sh + (int64_t)t * a.v_st;
    if (r < nqk && a.ko) {
      dst = a.ko;
      dof = (int64_t)b * a.ko_sb + (int64_t)h * a.ko_sh + (int64_t)t * a.ko_st;
    } else {
      const int64_t slot = rope_slot(a, b, start + t);
      if (slot < 0) return;  // the whole wave
      dst = r < nqk ? a.k_pages : a.v_pages;
      dof = slot + (int64_t)h * a.p_sh;
    }
  }
  if (r >= nqk) {
    for (int d = lane; d < a.D; d += 64)
      store_from_f32(dst, dt, dof + d, load_as_f32(src, dt, so + d));
    return;
  }
  float ss = 0.f;
  for (int d = lane; d < a.D; d += 64) {
    const float x = load_as_f32(src, dt, so + d);
    ss = fmaf(x, x, ss);
  }
  const float rs = a.norm ? rsqrtf(sum_over_lanes<64>(ss) / (float)a.D + a.eps) : 1.f;
  const float *const g = a.norm ? (r < a.H ? a.wq : a.wk) : nullptr;
  for (int d = lane; d < a.D; d += 64)
    s_y[d] = load_as_f32(src, dt, so + d) * rs * (g ? g[d] : 1.f);
  __syncthreads();
  const int half = a.rot >> 1;
  for (int d = lane; d < a.D; d += 64) {
    float y = s_y[d];
    if (d < a.rot) {
      const int i = a.interleaved ? d >> 1 : (d < half ? d : d - half);
      const bool first = a.interleaved ? !(d & 1) : d < half;
      const int m = a.interleaved ? d ^ 1 : (first ? d + half : d - half);
      float s, c;
      rope_angle(a, pos, i, s, c);
      y = first ? y * c - s_y[m] * s : y * c + s_y[m] * s;
    }
    store_from_f32(dst, dt, dof + d, y);
  }
}

}  // namespace mtp
