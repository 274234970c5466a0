// Arguments of the windowed attention kernels (wattn*.hpp), shared with the
// host code that plans them.
#pragma once

#include <stdint.h>

#include "../../include/mtp_hip.h"

namespace mtp {

// Key and row positions, with the window added, stay within 31 bits.
constexpr int64_t kWinMaxKeys = (int64_t)1 << 29;
constexpr int kWinNone = 1 << 30;  // window: every earlier key is visible

struct WinArgs {
  const void *q;                  // [B, H, T, D] by element strides, d contiguous
  int64_t q_sb, q_sh, q_st;
  const void *k, *v;              // dense [B, Hk, L, D] by element strides, or
                                  // (table) pages [P, B, Hk, page_size, D]
  int64_t k_sb, k_sh, k_st, v_sb, v_sh, v_st;
  const int32_t *table;           // [B, ld_tab] physical page of each key, or null: dense
  int64_t ld_tab, p_sp;           // pages: p_sp the page stride; k_sb, k_sh, k_st their others
  int page_size, npages;
  void *out;                      // by element strides
  int64_t o_sb, o_sh, o_st;
  int B, H, Hk, G, T, D;          // G = H / Hk query heads to a key head
  int L;                          // keys of a sequence at most
  int window, sinks;              // window: kWinNone for none
  const int64_t *start_dev;       // position of query 0, per sequence (start_per_row) or shared
  int start_per_row;
  int64_t start_host;
  const int64_t *lengths;         // [B] keys and queries of each sequence (dense), or null
  float scale;                    // of the scores, in units of log 2
  float *scores;                  // [B * Hk][G * T][ld_sc] masked scores, or null
  int64_t ld_sc;
  float *weights;                 // [B, Hk, L], added to
  // rows of a (batch, key head) in rblocks blocks of rp, keys of a block in
  // nchunks chunks
  int rblocks, rp, nchunks;
  float *part;                    // [b * Hk + hk][row block][chunk][rp][D], nchunks > 1
  float *pml;                     // the same with (maximum, sum) for D; with scores too
  unsigned *ticket;               // null, or arrivals per (b * Hk + hk, row block): the last
                                  // workgroup joins the chunks
  int joins;                      // workgroups that join chunks, before those for the weights
};

// The keys that the queries of one sequence see: [0, ns) and [lo, hi), the
// union over its rows; row t stands at position first + t and sees those keys
// j <= first + t with j > first + t - window or j < sinks; rows from `rows` on
// see nothing.
struct WinSpan {
  int first, rows, ns, lo, hi;
  __host__ __device__ int count() const { return ns + hi - lo; }
  // Key of compact index i < count(), and back.
  __host__ __device__ int key(int i) const { return i < ns ? i : lo + (i - ns); }
  __host__ __device__ int index(int j) const { return j < ns ? j : j - lo + ns; }
};

// Keys of a wave's step in the split kernel (wattn_split.hpp): whole K = 32
// products of 16-bit types; fp32 with half as many keeps three waves on a SIMD
// at head dim 64 (B 2, T 1000, H 16, window 256: 39 us against 43.6).
constexpr int win_split_keys(int ct) { return ct == MTP_F32 ? 16 : 32; }

typedef void (*WinKernel)(WinArgs);
// The split kernel for rows of type ct and head dim d in tiles of 16 * rt rows
// (rt 1 or 2) with nw waves (4 or 8); null for other shapes. Grid (B * Hk, row
// blocks, chunks).
WinKernel win_split_pick(int ct, int d, int rt, bool paged, int nw);
constexpr int kWinTicketChunks = 64;  // chunks of a block at most, with tickets
// The join of its chunks with 1 or 4 waves a row, 4 / waves rows a workgroup,
// and after those a.joins workgroups one for every 256 keys of a (batch, key
// head) that adds to the weights.
WinKernel win_join_pick(int ct, int d, bool paged, int waves);

// The prompt kernel (wattn_prompt.hpp) for 16-bit rows of head dim d: blocks of
// kWinPromptRows rows, two threads each, tiles of kWinTileKeys keys; null for
// other shapes. Grid (B * Hk, row blocks, chunks).
constexpr int kWinPromptRows = 128, kWinTileKeys = 64;
WinKernel win_prompt_pick(int ct, int d);
constexpr int win_prompt_lds(int d) { return 2 * 2 * kWinTileKeys * 2 * d; }

}  // namespace mtp
