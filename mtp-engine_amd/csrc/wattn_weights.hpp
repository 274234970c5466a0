// Sums of the windowed attention's probabilities by key (wattn.hpp), from the
// scores that it kept.
#pragma once

#include "wattn.hpp"

namespace mtp {

// Adds to a.weights, for the 256 keys `kb` of (sequence, key head) bh, the
// weight that they received: sum over the head's rows of exp2(score - max) /
// sum, rows in order, so the result does not depend on timing. A thread takes a
// key, eight rows' scores in flight.
__device__ __forceinline__ void win_weights(const WinArgs &a, int bh, int kb, float (&s_m)[256],
                                            float (&s_i)[256]) {
  const int b = bh / a.Hk;
  const WinSpan s = win_span(a, b);
  const int n = s.count();
  if (kb * 256 >= n) return;  // the whole workgroup
  const int i = kb * 256 + threadIdx.x;
  const int rows = a.G * s.rows, j = s.key(min(i, n - 1));
  const int pad = a.G * a.T;  // rows of the scores
  float w = 0.f;
  for (int r0 = 0; r0 < rows; r0 += 256) {
    __syncthreads();
    if (r0 + (int)threadIdx.x < rows) {
      // the row's maximum and sum over its chunks
      const int r = r0 + threadIdx.x, rb = r / a.rp;
      const float *ml = a.pml + (((int64_t)bh * a.rblocks + rb) * a.nchunks * a.rp + (r - rb * a.rp)) * 2;
      float m = -INFINITY, l = 0.f;
      for (int c = 0; c < a.nchunks; ++c, ml += 2 * a.rp) {
        const float m2 = ml[0], mn = fmaxf(m, m2), ref = mn == -INFINITY ? 0.f : mn;
        l = l * __builtin_amdgcn_exp2f(m - ref) + ml[1] * __builtin_amdgcn_exp2f(m2 - ref);
        m = mn;
      }
      s_m[threadIdx.x] = m == -INFINITY ? 0.f : m;
      s_i[threadIdx.x] = l == 0.f ? 0.f : 1.f / l;
    }
    __syncthreads();
    if (i >= n) continue;
    const int most = min(256, rows - r0);
    const float *const sc = a.scores + ((int64_t)bh * pad + r0) * a.ld_sc + i;
    int t = r0 / a.G, g = r0 - t * a.G;
    constexpr int F = 8;
    for (int r = 0; r < most; r += F) {
      float x[F];
#pragma unroll
      for (int u = 0; u < F; ++u) {
        // a row keeps the scores of the keys that it sees (and perhaps others)
        const bool see = (r + u < most) & win_sees(a, s.first + t, j);
        x[u] = -INFINITY;
        if (see) x[u] = sc[(int64_t)(r + u) * a.ld_sc];
        if (++g == a.G) g = 0, ++t;
      }
#pragma unroll
      for (int u = 0; u < F; ++u) {
        const int q = min(r + u, most - 1);
        w = fmaf(__builtin_amdgcn_exp2f(x[u] - s_m[q]), s_i[q], w);
      }
    }
  }
  if (i < n) a.weights[(int64_t)bh * a.L + j] += w;
}

}  // namespace mtp
