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
// 4096 tokens of 32 + 8 heads of 128 in bf16 (84 MB): 16.7 us, 5.0 TB/s, what a
// large copy reaches; 8 tokens: 6.1 us, a launch and the latencies of position,
// page, rows and store in turn.
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

// sin and cos of position * f.
__device__ __forceinline__ void rope_angle(int64_t pos, double f, float &s, float &c) {
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
// pair's halves in whole chunks. A token's rows come in steps of RPI: those of
// its queries, then of its keys, then of its values; wave (token, part) takes
// the steps part, part + hs, ...
template <int DT, int LPR, bool INTER>
__global__ void __launch_bounds__(256) rope_kernel(const RopeArgs a) {
  constexpr int VEC = 16 / dtype_bytes(DT);
  constexpr int RPI = 64 / LPR;
  constexpr int U = 4;  // steps in flight
  const int lane = threadIdx.x & 63;
  const int64_t wid =
      (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tok = wid / a.hs;
  const int part = (int)(wid % a.hs);
  if (tok >= (int64_t)a.B * a.T) return;
  const int b = (int)(tok / a.T), t = (int)(tok % a.T);
  const int sub = lane / LPR, c = lane % LPR, d0 = c * VEC;
  const bool on = d0 < a.D;
  const int nq = (a.H + RPI - 1) / RPI, nk = (a.Hk + RPI - 1) / RPI;
  const int steps = nq + nk + (a.v ? nk : 0);

  const char *const qs = (const char *)a.q +
      ((int64_t)b * a.q_sb + (int64_t)t * a.q_st + d0) * dtype_bytes(DT);
  const char *const ks = (const char *)a.k +
      ((int64_t)b * a.k_sb + (int64_t)t * a.k_st + d0) * dtype_bytes(DT);
  const char *const vs = (const char *)a.v +
      ((int64_t)b * a.v_sb + (int64_t)t * a.v_st + d0) * dtype_bytes(DT);
  u32x4 w[U];
  auto fetch = [&](int st) -> u32x4 {  // st is the same for the wave
    u32x4 x = {0u, 0u, 0u, 0u};
    if (st < nq) {
      const int r = st * RPI + sub;
      if (on && r < a.H) x = *(const u32x4 *)(qs + (int64_t)r * a.q_sh * dtype_bytes(DT));
    } else if (st < steps) {
      const bool key = st < nq + nk;
      const int r = (st - nq - (key ? 0 : nk)) * RPI + sub;
      if (on && r < a.Hk)
        x = *(const u32x4 *)((key ? ks : vs) +
                             (int64_t)r * (key ? a.k_sh : a.v_sh) * dtype_bytes(DT));
    }
    return x;
  };
  // the first rows are asked for before what their results need is computed
#pragma unroll
  for (int u = 0; u < U; ++u) w[u] = fetch(part + u * a.hs);

  const int half = a.rot >> 1;
  const bool rotated = on && d0 < a.rot;
  const int hc = half / VEC;
  const int mate = INTER || !rotated ? lane : (d0 < half ? lane + hc : lane - hc);
  const int e0 = on ? d0 : 0, m0 = e0 + (mate - lane) * VEC;  // the partner's first element
  // every load of the token before the first use of one: frequencies as raw
  // bits, so that their conversion does not wait here
  constexpr int NF = INTER ? VEC / 2 : VEC;
  const int f0 = !rotated ? 0 : INTER ? d0 / 2 : (d0 < half ? d0 : d0 - half);
  uint32_t flo[NF], fhi[NF];
#pragma unroll
  for (int i = 0; i < NF; ++i) flo[i] = fhi[i] = 0u;
  if (a.rot > 0) {
    if (a.freq64) {
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        const uint2 x = ((const uint2 *)a.inv_freq)[f0 + i];
        flo[i] = x.x;
        fhi[i] = x.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NF; ++i) flo[i] = ((const uint32_t *)a.inv_freq)[f0 + i];
    }
  }
  // y = rs * (x * A + partner * B): A the gain times cos, B the partner's gain
  // times -+ sin, for queries and for keys; a chunk that is not rotated has
  // zeros for its partner, as it may hold an infinity itself
  float A[2][VEC], B[2][VEC];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const float *const g = !a.norm ? nullptr : q == 0 ? a.wq : a.wk;
#pragma unroll
    for (int i = 0; i < VEC; ++i) A[q][i] = B[q][i] = 1.f;
    if (g) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        A[q][i] = g[e0 + i];
        B[q][i] = g[INTER ? e0 + (i ^ 1) : m0 + i];
      }
    }
  }
  const int64_t start = a.start_dev ? a.start_dev[a.start_per_row ? b : 0] : a.start_host;
  const int64_t at = start + t;
  const int64_t pos = a.pos ? a.pos[(int64_t)b * a.pos_sb + t] : at;
  const int64_t slot = a.v ? rope_slot(a, b, at) : -1;
#pragma unroll
  for (int i = 0; i < NF; ++i) {
    float sn = 0.f, cs = 1.f;
    if (rotated) {
      const double f = a.freq64 ? __longlong_as_double((long long)fhi[i] << 32 | flo[i])
                                : (double)__uint_as_float(flo[i]);
      rope_angle(pos, f, sn, cs);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if constexpr (INTER) {
        A[q][2 * i] *= cs;
        A[q][2 * i + 1] *= cs;
        B[q][2 * i] *= -sn;
        B[q][2 * i + 1] *= sn;
      } else {
        A[q][i] *= cs;
        B[q][i] *= d0 < half ? -sn : sn;
      }
    }
  }
  const float inv_d = 1.f / (float)a.D;

  auto turn = [&](u32x4 raw, const float(&ca)[VEC], const float(&cb)[VEC]) -> u32x4 {
    float x[VEC], y[VEC];
    rope_unpack<DT>(raw, x);
    float rs = 1.f;
    if (a.norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) ss = fmaf(x[i], x[i], ss);
      rs = rsqrtf(sum_over_lanes<LPR>(ss) * inv_d + a.eps);
    }
    if constexpr (INTER) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) y[i] = rotated ? x[i ^ 1] : 0.f;
    } else {
      u32x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t z = __shfl(raw[i], mate, 64);
        o[i] = rotated ? z : 0u;
      }
      rope_unpack<DT>(o, y);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) y[i] = rs * fmaf(x[i], ca[i], y[i] * cb[i]);
    return rope_pack<DT>(y);
  };

  for (int s0 = part; s0 < steps; s0 += U * a.hs) {
    u32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = w[u];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = fetch(s0 + (U + u) * a.hs);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int st = s0 + u * a.hs;
      if (st < nq) {
        const u32x4 y = turn(x[u], A[0], B[0]);
        const int r = st * RPI + sub;
        if (on && r < a.H)
          *(u32x4 *)((char *)a.qo + ((int64_t)b * a.qo_sb + (int64_t)r * a.qo_sh +
                                     (int64_t)t * a.qo_st + d0) * dtype_bytes(DT)) = y;
      } else if (st < nq + nk) {
        const u32x4 y = turn(x[u], A[1], B[1]);
        const int r = (st - nq) * RPI + sub;
        if (on && r < a.Hk) {
          if (a.ko)
            *(u32x4 *)((char *)a.ko + ((int64_t)b * a.ko_sb + (int64_t)r * a.ko_sh +
                                       (int64_t)t * a.ko_st + d0) * dtype_bytes(DT)) = y;
          else if (slot >= 0)
            *(u32x4 *)((char *)a.k_pages + (slot + (int64_t)r * a.p_sh + d0) * dtype_bytes(DT)) = y;
        }
      } else if (st < steps) {
        const int r = (st - nq - nk) * RPI + sub;
        if (on && r < a.Hk && slot >= 0)
          *(u32x4 *)((char *)a.v_pages + (slot + (int64_t)r * a.p_sh + d0) * dtype_bytes(DT)) =
              x[u];
      }
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
      rope_angle(pos, a.freq64 ? ((const double *)a.inv_freq)[i]
                               : (double)((const float *)a.inv_freq)[i], s, c);
      y = first ? y * c - s_y[m] * s : y * c + s_y[m] * s;
    }
    store_from_f32(dst, dt, dof + d, y);
  }
}

}  // namespace mtp
