// C ABI of the serving operators around the paged KV cache: per-head norms
// with the position rotation, windowed attention of prompts and of new tokens
// over the cache, eviction by attention weight. Declarations are in
// include/mtp_hip.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstddef>

#include "abi_util.hpp"
#include "evict.hpp"
#include "rope.hpp"
#include "wattn.hpp"
#include "wattn_weights.hpp"

using namespace mtp;

// The layouts that mtp_hip/_lib.py packs.
static_assert(sizeof(mtp_rope_args) == 336 && offsetof(mtp_rope_args, eps) == 312, "mtp_rope_args");
static_assert(sizeof(mtp_window_args) == 280 && offsetof(mtp_window_args, scale) == 264,
              "mtp_window_args");

namespace {

bool mult(std::initializer_list<int64_t> v, int64_t m) {
  for (int64_t x : v)
    if (x % m != 0) return false;
  return true;
}

// ---- norms and rotation
typedef void (*RopeKernel)(RopeArgs);

template <int DT, int LPR>
RopeKernel rope_form(bool inter) {
  return inter ? rope_kernel<DT, LPR, true> : rope_kernel<DT, LPR, false>;
}
template <int DT>
RopeKernel rope_lanes(int64_t chunks, bool inter, int &lpr) {
  if (chunks <= 4) return lpr = 4, rope_form<DT, 4>(inter);
  if (chunks <= 8) return lpr = 8, rope_form<DT, 8>(inter);
  if (chunks <= 16) return lpr = 16, rope_form<DT, 16>(inter);
  if (chunks <= 32) return lpr = 32, rope_form<DT, 32>(inter);
  if (chunks <= 64) return lpr = 64, rope_form<DT, 64>(inter);
  return nullptr;
}

// The 16-byte form, or null: rows, strides and addresses of whole 16 bytes,
// a rotation whose halves are whole chunks.
RopeKernel rope_pick(const RopeArgs &a, int dt, int &lpr) {
  const int64_t e = 16 / dtype_bytes(dt);
  if (a.D % e != 0 || (a.interleaved ? a.rot % e : (a.rot / 2) % e) != 0) return nullptr;
  if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.qo) || (a.ko && !aligned16(a.ko)) ||
      (a.v && (!aligned16(a.v) || !aligned16(a.k_pages) || !aligned16(a.v_pages))))
    return nullptr;
  if (!mult({a.q_sb, a.q_sh, a.q_st, a.k_sb, a.k_sh, a.k_st, a.v_sb, a.v_sh, a.v_st, a.qo_sb,
             a.qo_sh, a.qo_st, a.ko_sb, a.ko_sh, a.ko_st},
            e))
    return nullptr;
  switch (dt) {
    case MTP_F32: return rope_lanes<MTP_F32>(a.D / e, a.interleaved, lpr);
    case MTP_BF16: return rope_lanes<MTP_BF16>(a.D / e, a.interleaved, lpr);
    case MTP_F16: return rope_lanes<MTP_F16>(a.D / e, a.interleaved, lpr);
  }
  return nullptr;
}

int rope_launch(RopeArgs &a, int dt, hipStream_t st) {
  int lpr = 0;
  const int64_t toks = (int64_t)a.B * a.T;
  if (RopeKernel k = rope_pick(a, dt, lpr)) {
    // a wave per token, more of them while the chip has room: up to one for
    // every 64 / lpr rows
    const int64_t rpi = 64 / lpr, room = (int64_t)device_cus() * 8;
    const int64_t most = (a.H + rpi - 1) / rpi + (a.v ? 2 : 1) * ((a.Hk + rpi - 1) / rpi);
    a.hs = (int)std::max<int64_t>(1, std::min((room + toks - 1) / toks, most));
    const int64_t blocks = (toks * a.hs + 3) / 4;
    if (blocks > INT32_MAX) return MTP_ERR_SHAPE;
    hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(256), 0, st, a);
  } else {
    const int64_t nr = a.H + a.Hk + (a.v ? a.Hk : 0);
    if (toks * nr > INT32_MAX) return MTP_ERR_SHAPE;
    hipLaunchKernelGGL(rope_generic_kernel, dim3((unsigned)(toks * nr)), dim3(64), 0, st, a, dt);
  }
  return launch_status();
}

// What both entry points check and fill in; > 0: nothing to do.
int rope_args(RopeArgs &a, const mtp_rope_args *p) {
  if (!p) return MTP_ERR_NULL;
  if (!is_float_dt(p->dtype)) return MTP_ERR_DTYPE;
  const int64_t B = p->B, T = p->T, H = p->H, Hk = p->Hk, D = p->D, rot = p->rot;
  if (B < 0 || T < 0 || H < 0 || Hk < 0 || D <= 0 || D > kRopeMaxD || rot < 0 || rot > D ||
      rot % 2 != 0 || B > INT32_MAX || T > INT32_MAX || H > 65535 || Hk > 65535)
    return MTP_ERR_SHAPE;
  if (B == 0 || T == 0 || H + Hk == 0) return 1;
  if ((H > 0 && (!p->q || !p->q_out)) || (Hk > 0 && !p->k) || (rot > 0 && !p->inv_freq))
    return MTP_ERR_NULL;
  a.q = p->q;
  a.k = p->k;
  a.qo = p->q_out;
  a.q_sb = p->q_st[0], a.q_sh = p->q_st[1], a.q_st = p->q_st[2];
  a.k_sb = p->k_st[0], a.k_sh = p->k_st[1], a.k_st = p->k_st[2];
  a.qo_sb = p->qo_st[0], a.qo_sh = p->qo_st[1], a.qo_st = p->qo_st[2];
  a.inv_freq = p->inv_freq;
  a.freq64 = p->freq_f64 ? 1 : 0;
  a.wq = p->q_weight;
  a.wk = p->k_weight;
  a.pos = p->positions;
  a.pos_sb = p->pos_sb;
  a.start_dev = p->start_dev;
  a.start_per_row = p->start_per_row ? 1 : 0;
  a.start_host = p->start_host;
  a.B = (int)B;
  a.T = (int)T;
  a.H = (int)H;
  a.Hk = (int)Hk;
  a.D = (int)D;
  a.rot = (int)rot;
  a.norm = p->norm ? 1 : 0;
  a.interleaved = p->interleaved ? 1 : 0;
  a.eps = p->eps;
  return MTP_OK;
}

// ---- windowed attention
struct WinPlan {
  int prompt = 0;          // chunks of the prompt kernel, where the strides let it take the call
  int rt = 0;              // else the split kernel: row tiles of a block; 0: one wave per row
  int nw = 4;              // its waves
  int rblocks = 1, nchunks = 1;
  bool joined = false;     // its chunks joined by their last workgroup
  int64_t ld_sc = 0;       // scores (with weights)
  size_t sc_off = 0, part_off = 0, pml_off = 0, total = 0;
};

// Keys that t queries can see of a sequence at most.
int64_t win_most(int64_t t, int64_t L, int64_t window, int64_t sinks) {
  if (window == kWinNone) return L;
  return std::min(L, std::min(sinks, L) + window + t - 1);
}

int win_window(int64_t window) {
  return window < 0 || window >= kWinNone / 2 ? kWinNone : (int)window;
}

// Chunks of keys with which dense 16-bit rows take the prompt kernel; 0: the split
// kernel. By estimates of the times, in us, fitted to 176 sizes (head dim 64 and
// 128; 1 .. 32 (batch, key head) pairs, 33 .. 17500 rows, 33 .. 4000 keys, no
// window):
//   prompt  5 + 1.25 a tile of the longest block, or 1.6 a tile over the 512
//           blocks that run at once (head dim 64: 4, 0.9 and 1.1); with chunks 6
//           more and the partials' bytes at 3 TB/s
//   split   8 + 45 a million keys of all the 32-row blocks (head dim 64: 7, 28)
// e.g. at head dim 128: 32 pairs, T 1000, L 1000: 27.9 and 38.7 us measured; 8
// pairs, T 1000, L 4000: 85.0 and 50.8; one pair of 33 rows and keys: 5.6, 8.1. 8
// pairs of four heads, T 512: L 8192 92.6 with chunks, 170 with one or split; L
// 32768 307 and 733.
int win_prompt_chunks(int dt, int64_t units, int64_t G, int64_t T, int64_t D, int64_t L,
                      int64_t window, int64_t sinks) {
  if (!win_prompt_pick(dt, (int)std::min<int64_t>(D, 1 << 20))) return 0;
  const double rows = (double)(G * T);
  const double mean =
      (double)std::min(win_most(1, L, window, sinks), std::max<int64_t>(1, L - T / 2));
  const double most = (double)win_most(std::min(T, kWinPromptRows / G + 2), L, window, sinks);
  const double blocks = std::ceil(rows / kWinPromptRows) * units;
  const bool small = D == 64;
  double best = (small ? 7. : 8.) +
                (small ? 28e-6 : 45e-6) * std::ceil(rows / 32.) * units * (mean + 32.);
  int chunks = 0;
  for (int c = 1; c <= 8 && (c == 1 || blocks * c <= 512.); c *= 2) {
    const double t = (small ? 4. : 5.) +
                     std::max((small ? 0.9 : 1.25) * std::ceil(most / kWinTileKeys / c),
                              (small ? 1.1 : 1.6) * blocks * (mean / kWinTileKeys + c) / 512.) +
                     (c > 1 ? 6. + 8e-6 / 3. * rows * units * c * D : 0.);
    if (t < best) best = t, chunks = c;
  }
  return chunks;
}

// Rows of 16 whole bytes at 64 or 128 elements take the split kernel, dense
// 16-bit ones the prompt kernel where it is faster.
WinPlan win_plan(int dt, int64_t B, int64_t H, int64_t Hk, int64_t T, int64_t D, int64_t L,
                 int window, int64_t sinks, bool paged, bool weights) {
  WinPlan p;
  if (B <= 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || T <= 0 || L <= 0) return p;
  const int64_t rows = H / Hk * T, units = B * Hk;
  size_t at = kCounterBytes;
  if (win_split_pick(dt, (int)std::min<int64_t>(D, 1 << 20), 1, false, 4)) {
    p.prompt = paged ? 0 : win_prompt_chunks(dt, units, H / Hk, T, D, L, window, sinks);
    p.rt = rows > 16 ? 2 : 1;
    const int64_t rp = 16 * p.rt;
    p.rblocks = (int)((rows + rp - 1) / rp);
    const int64_t most = win_most(std::min(T, (rp - 1) / (H / Hk) + 2), L, window, sinks);
    const int64_t wgs = units * p.rblocks, sk = win_split_keys(dt);
    // eight waves, a workgroup a CU, where that many workgroups suffice (chunks
    // of a step for every wave); else four, so that two of them share a CU
    p.nw = wgs <= device_cus() ? 8 : 4;
    const int64_t room = 8 / p.nw * (int64_t)device_cus() / wgs;
    // (the prompt kernel needs no chunks; a call that it cannot take has one)
    if (!p.prompt) p.nchunks = (int)std::max<int64_t>(1, std::min(room, most / (8 * sk)));
    // up to 128 KB of a block's partials the last workgroup joins, more of them
    // take longer on one CU than a launch of their own (8 KB: 23.9 us and 25.3;
    // 32 KB: 15.0 and 15.6; 128 KB: 12.2 and 13.8; 256 KB: 16.7 and 14.8)
    p.joined = p.nchunks > 1 && !weights && p.nchunks <= kWinTicketChunks &&
               std::min(rp, rows) * p.nchunks * D * 4 <= 128 << 10 && wgs <= kCounterSlots;
    const int64_t pblocks = (rows + kWinPromptRows - 1) / kWinPromptRows;
    const int64_t parts =
        p.prompt > 1 ? units * pblocks * p.prompt * kWinPromptRows : wgs * p.nchunks * rp;
    const bool chunks = p.prompt > 1 || p.nchunks > 1;
    if (chunks) {
      p.part_off = at;
      at += align_up((size_t)parts * (size_t)D * 4, 256);
    }
    if (chunks || weights) {
      p.pml_off = at;
      at += align_up((size_t)std::max(parts, B * H * T) * 8, 256);
    }
  } else if (weights) {
    p.pml_off = at;
    at += align_up((size_t)(B * H * T) * 8, 256);
  }
  if (weights) {
    p.ld_sc = win_most(T, L, window, sinks);
    p.sc_off = at;
    at += align_up((size_t)(B * H * T) * (size_t)p.ld_sc * 4, 256);
  }
  p.total = at > kCounterBytes ? at : 0;
  return p;
}

// The weights alone, after the kernel that takes a wave per row.
__global__ void __launch_bounds__(256) win_weights_kernel(const WinArgs a) {
  __shared__ float s_a[256], s_b[256];
  win_weights(a, blockIdx.y, blockIdx.x, s_a, s_b);
}

template <bool PAGED>
void (*win_generic(int64_t d))(WinArgs, int) {
  if (d <= 64) return win_rows_generic_kernel<1, PAGED>;
  if (d <= 128) return win_rows_generic_kernel<2, PAGED>;
  if (d <= 256) return win_rows_generic_kernel<4, PAGED>;
  return win_rows_generic_kernel<16, PAGED>;
}
constexpr int64_t kWinMaxD = 1024;

int win_launch(WinArgs &a, int dt, void *workspace, size_t workspace_bytes, hipStream_t st) {
  const WinPlan p = win_plan(dt, a.B, a.H, a.Hk, a.T, a.D, a.L, a.window, a.sinks,
                             a.table != nullptr, a.weights != nullptr);
  if (p.total > 0 && (!workspace || workspace_bytes < p.total)) return MTP_ERR_WORKSPACE;
  const int64_t rows = (int64_t)a.B * a.H * a.T;
  if (rows > INT32_MAX) return MTP_ERR_SHAPE;
  unsigned char *const w8 = (unsigned char *)workspace;
  if (a.weights) {
    a.scores = (float *)(w8 + p.sc_off);
    a.ld_sc = p.ld_sc;
  }
  a.part = (float *)(w8 + p.part_off);
  a.pml = (float *)(w8 + p.pml_off);
  const int64_t e = 16 / dtype_bytes(dt);
  const bool whole = aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.out) &&
                     mult({a.q_sb, a.q_sh, a.q_st, a.k_sb, a.k_sh, a.k_st, a.v_sb, a.v_sh, a.v_st,
                           a.o_sb, a.o_sh, a.o_st, a.p_sp},
                          e);
  int s;
  // the prompt kernel: dense keys whose rows a buffer's 32-bit offsets reach
  const int64_t reach = ((int64_t)1 << 31) / 2 - a.D;
  const bool near = a.k_st >= 0 && a.v_st >= 0 && (a.L - 1) * a.k_st < reach &&
                    (a.L - 1) * a.v_st < reach;
  const int64_t pblocks = ((int64_t)a.G * a.T + kWinPromptRows - 1) / kWinPromptRows;
  // (its maximum is that of the products, so it takes no scale below zero)
  // the chunks' join, and the weights
  const bool paged = a.table != nullptr;
  auto join = [&]() {
    // four waves to a row of many chunks while the chip has room for them
    const int mw = a.nchunks > 8 && rows <= 8 * (int64_t)device_cus() ? 4 : 1;
    a.joins = a.nchunks > 1 ? (int)((rows * mw + 3) / 4) : 0;
    const int64_t sums = a.weights ? (p.ld_sc + 255) / 256 * a.B * a.Hk : 0;
    if (a.joins + sums > INT32_MAX) return (int)MTP_ERR_SHAPE;
    hipLaunchKernelGGL(win_join_pick(dt, a.D, paged, mw), dim3((unsigned)(a.joins + sums)),
                       dim3(256), 0, st, a);
    return launch_status();
  };
  if (p.prompt && near && whole && a.scale > 0.f && pblocks <= 65535) {
    a.rblocks = (int)pblocks;
    a.rp = kWinPromptRows;
    a.nchunks = p.prompt;
    hipLaunchKernelGGL(
        win_prompt_pick(dt, a.D),
        dim3((unsigned)(a.B * a.Hk), (unsigned)pblocks, (unsigned)p.prompt),
        dim3(kWinPromptRows * 2), win_prompt_lds(a.D), st, a);
    s = launch_status();
    return s == MTP_OK && p.prompt > 1 ? join() : s;
  }
  if (p.rt && whole && p.rblocks <= 65535) {
    a.rblocks = p.rblocks;
    a.rp = 16 * p.rt;
    a.nchunks = p.nchunks;
    a.ticket = p.joined ? (unsigned *)w8 : nullptr;
    hipLaunchKernelGGL(win_split_pick(dt, a.D, p.rt, paged, p.nw),
                       dim3((unsigned)(a.B * a.Hk), (unsigned)p.rblocks, (unsigned)p.nchunks),
                       dim3(64 * p.nw), 0, st, a);
    s = launch_status();
    return s == MTP_OK && !p.joined && (p.nchunks > 1 || a.weights) ? join() : s;
  }
  a.rblocks = 1;
  a.rp = a.G * a.T;
  hipLaunchKernelGGL(a.table ? win_generic<true>(a.D) : win_generic<false>(a.D),
                     dim3((unsigned)rows), dim3(64), win_row_lds(a.D) * 4, st, a, dt);
  s = launch_status();
  if (s != MTP_OK || !a.weights) return s;
  hipLaunchKernelGGL(win_weights_kernel, dim3((unsigned)((p.ld_sc + 255) / 256),
                                              (unsigned)(a.B * a.Hk)),
                     dim3(256), 0, st, a);
  return launch_status();
}

// What both entry points check and fill in; > 0: nothing to do.
int win_args(WinArgs &a, const mtp_window_args *p) {
  if (!p) return MTP_ERR_NULL;
  if (!is_float_dt(p->dtype)) return MTP_ERR_DTYPE;
  const int64_t B = p->B, H = p->H, Hk = p->Hk, T = p->T, D = p->D, L = p->L;
  if (B < 0 || T < 0 || H < 0 || Hk <= 0 || H % Hk != 0 || D <= 0 || D > kWinMaxD || L < 0 ||
      B > INT32_MAX || H > 65535 || T > kWinMaxKeys || L > kWinMaxKeys)
    return MTP_ERR_SHAPE;
  if (p->window == 0 || p->window < -1 || p->sinks < 0) return MTP_ERR_ARG;
  if (B == 0 || T == 0 || H == 0) return 1;
  if (!p->q || !p->out || (L > 0 && (!p->k || !p->v))) return MTP_ERR_NULL;
  a.q = p->q;
  a.q_sb = p->q_st[0], a.q_sh = p->q_st[1], a.q_st = p->q_st[2];
  a.k = p->k;
  a.v = p->v;
  a.out = p->out;
  a.o_sb = p->out_st[0], a.o_sh = p->out_st[1], a.o_st = p->out_st[2];
  a.B = (int)B;
  a.H = (int)H;
  a.Hk = (int)Hk;
  a.G = (int)(H / Hk);
  a.T = (int)T;
  a.D = (int)D;
  a.L = (int)L;
  a.window = win_window(p->window);
  a.sinks = (int)std::min(p->sinks, L);
  a.scale = p->scale * 1.44269504088896340736f;
  a.nchunks = 1;
  return MTP_OK;
}

}  // namespace

extern "C" {

int mtp_qk_norm_rope(const mtp_rope_args *p, void *stream) {
  RopeArgs a{};
  const int s = rope_args(a, p);
  if (s != MTP_OK) return s > 0 ? MTP_OK : s;
  if (p->Hk > 0 && !p->k_out) return MTP_ERR_NULL;
  a.ko = p->k_out;
  a.ko_sb = p->ko_st[0], a.ko_sh = p->ko_st[1], a.ko_st = p->ko_st[2];
  return rope_launch(a, p->dtype, (hipStream_t)stream);
}

int mtp_qk_norm_rope_write(const mtp_rope_args *p, void *stream) {
  RopeArgs a{};
  const int s = rope_args(a, p);
  if (s < 0) return s;
  if (p->num_pages < 0 || p->page_size <= 0 || p->ld_tab < 0 || p->num_pages > INT32_MAX ||
      p->page_size > INT32_MAX)
    return MTP_ERR_SHAPE;
  if (s > 0) return MTP_OK;
  if (p->Hk > 0 &&
      (!p->v || !p->k_pages || !p->v_pages || (p->ld_tab > 0 && !p->page_table)))
    return MTP_ERR_NULL;
  a.v = p->v;
  a.v_sb = p->v_st[0], a.v_sh = p->v_st[1], a.v_st = p->v_st[2];
  a.k_pages = p->k_pages;
  a.v_pages = p->v_pages;
  a.p_sh = p->page_size * p->D;
  a.p_sb = p->Hk * a.p_sh;
  a.p_sp = p->B * a.p_sb;
  a.table = p->page_table;
  a.ld_tab = p->ld_tab;
  a.page_size = (int)p->page_size;
  a.npages = (int)p->num_pages;
  return rope_launch(a, p->dtype, (hipStream_t)stream);
}

size_t mtp_window_attention_workspace_bytes(int dtype, int64_t B, int64_t H, int64_t Hk, int64_t T,
                                            int64_t D, int64_t L, int64_t window, int64_t sinks,
                                            int paged, int weights) {
  if (!is_float_dt(dtype) || T > kWinMaxKeys || L > kWinMaxKeys || B > INT32_MAX || H > 65535)
    return 0;
  return win_plan(dtype, B, H, Hk, T, D, L, win_window(window), std::max<int64_t>(sinks, 0),
                  paged != 0, weights != 0)
      .total;
}

int mtp_window_attention(const mtp_window_args *p, void *stream) {
  WinArgs a{};
  const int s = win_args(a, p);
  if (s < 0) return s;
  if (p->L < p->T) return MTP_ERR_SHAPE;
  if (s > 0) return MTP_OK;
  a.k_sb = p->k_st[0], a.k_sh = p->k_st[1], a.k_st = p->k_st[2];
  a.v_sb = p->v_st[0], a.v_sh = p->v_st[1], a.v_st = p->v_st[2];
  a.start_host = p->L - p->T;
  a.lengths = p->lengths;
  return win_launch(a, p->dtype, p->workspace, p->workspace_bytes, (hipStream_t)stream);
}

int mtp_paged_window_attention(const mtp_window_args *p, void *stream) {
  WinArgs a{};
  const int s = win_args(a, p);
  if (s < 0) return s;
  if (p->num_pages < 0 || p->num_pages > INT32_MAX || p->page_size <= 0 ||
      p->page_size > INT32_MAX || (p->weights && p->B * p->Hk > 65535))
    return MTP_ERR_SHAPE;
  if (s > 0) return MTP_OK;
  if (p->L > 0 && !p->page_table) return MTP_ERR_NULL;
  a.k_st = p->D;
  a.k_sh = p->page_size * p->D;
  a.k_sb = p->Hk * a.k_sh;
  a.p_sp = p->B * a.k_sb;
  a.v_sb = a.k_sb, a.v_sh = a.k_sh, a.v_st = a.k_st;
  a.table = p->page_table;
  a.ld_tab = p->L;
  a.page_size = (int)p->page_size;
  a.npages = (int)p->num_pages;
  a.start_dev = p->start_dev;
  a.start_per_row = p->start_per_row ? 1 : 0;
  a.start_host = p->start_host;
  a.weights = p->L > 0 ? p->weights : nullptr;
  return win_launch(a, p->dtype, p->workspace, p->workspace_bytes, (hipStream_t)stream);
}

int mtp_kv_evict(const float *weights, const int64_t *lengths, int64_t B, int64_t Hk, int64_t L,
                 int64_t keep, int64_t sinks, int64_t recent, void *k_pages, void *v_pages,
                 int64_t num_pages, int64_t page_size, int64_t row_bytes,
                 const int32_t *page_table, const int32_t *out_table,
                 int32_t *kept, float *out_weights, int64_t *out_lengths, void *stream) {
  if (B < 0 || Hk < 0 || L < 0 || keep <= 0 || row_bytes <= 0 || num_pages < 0 ||
      page_size <= 0 || num_pages > INT32_MAX || page_size > INT32_MAX || L > kWinMaxKeys ||
      keep > kWinMaxKeys || B * Hk > INT32_MAX || row_bytes > (1 << 20))
    return MTP_ERR_SHAPE;
  if (sinks < 0 || recent < 0 || sinks + recent > keep) return MTP_ERR_ARG;
  if (B == 0 || Hk == 0) return MTP_OK;
  if (!lengths || !kept || !out_weights || !out_lengths || !out_table ||
      (L > 0 && (!weights || !page_table)) ||
      (num_pages > 0 && (!k_pages || !v_pages)))
    return MTP_ERR_NULL;
  EvictArgs a{};
  a.weights = weights;
  a.lengths = lengths;
  a.table = page_table;
  a.out_table = out_table;
  a.B = (int)B;
  a.Hk = (int)Hk;
  a.L = (int)L;
  a.keep = (int)keep;
  a.sinks = (int)sinks;
  a.recent = (int)recent;
  a.npages = (int)num_pages;
  a.page_size = (int)page_size;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.row_bytes = row_bytes;
  a.kept = kept;
  a.out_weights = out_weights;
  a.out_lengths = out_lengths;
  hipStream_t st = (hipStream_t)stream;
  // the copy's unit: the largest that divides a row and the addresses
  const uintptr_t bits = (uintptr_t)row_bytes | (uintptr_t)k_pages | (uintptr_t)v_pages;
  const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
  const int64_t blocks = (B * Hk * keep * (row_bytes / unit) + 255) / 256;
  if (blocks > INT32_MAX) return MTP_ERR_SHAPE;
  // up to 64 KB of a head's K the selecting workgroup moves its rows itself
  // (against a second launch: 64 KB of 8 heads 14.4 us and 15.9, 128 KB of 8
  // 16.7 and 16.5, of 64 heads 21.9 and 17.1)
  a.moves = num_pages > 0 && unit == 16 && keep * row_bytes <= 64 << 10;
  // entries of a lane kept in registers, where they fit
  const int64_t each = (L + kEvictThreads - 1) / kEvictThreads;
  void (*const sel)(EvictArgs) = each <= 4    ? evict_select_kernel<4>
                                 : each <= 8  ? evict_select_kernel<8>
                                 : each <= 16 ? evict_select_kernel<16>
                                 : each <= 32 ? evict_select_kernel<32>
                                              : evict_select_kernel<0>;
  hipLaunchKernelGGL(sel, dim3((unsigned)(B * Hk)), dim3(kEvictThreads), 0, st, a);
  int s = launch_status();
  if (s != MTP_OK || num_pages == 0 || a.moves) return s;
  void (*const mv)(EvictArgs) = unit == 16  ? evict_move_kernel<u32x4>
                                : unit == 4 ? evict_move_kernel<uint32_t>
                                : unit == 2 ? evict_move_kernel<uint16_t>
                                            : evict_move_kernel<uint8_t>;
  hipLaunchKernelGGL(mv, dim3((unsigned)blocks), dim3(256), 0, st, a);
  return launch_status();
}

}  // extern "C"
