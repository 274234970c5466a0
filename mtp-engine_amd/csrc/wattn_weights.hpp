// Sums of the windowed attention's probabilities by key (wattn.hpp), from the
// scores that it kept.
#pragma once

#include "wattn.hpp"

namespace mtp {

// Adds to a.weights, for the 256 keys `kb` of (sequence, key head) bh, the
// weight that they received: sum over the head's rows of exp2(score - max) /
// sum, rows in order, so the result does not depend on timing. A thread takes a
// key; 16 rows' scores are in flight, the first of them while the rows' maxima
// and sums are joined from their chunks. 20 rows of 64 (sequence, head)s by 4100
// keys (21 MB of scores), beside the join of the rows: 13 us; the whole call 48.1
// us, with eight rows in flight 50.4.
__device__ __forceinline__ void win_weights(const WinArgs &a, int bh, int kb, float (&s_m)[256],
                                            float (&s_i)[256]) {
  constexpr int F = 16, C = 4;
  const int b = bh / a.Hk;
  const WinSpan s = win_span(a, b);
  const int n = s.count();
  if (kb * 256 >= n) return;  // the whole workgroup
  const int i = kb * 256 + threadIdx.x, ii = min(i, n - 1);
  const int rows = a.G * s.rows, j = s.key(ii);
  const float *const sc = a.scores + (int64_t)bh * a.G * a.T * a.ld_sc + ii;
  // a row keeps the scores of the keys that it sees; at others there is anything
  auto fetch = [&](float (&x)[F], int r) {
#pragma unroll
    for (int u = 0; u < F; ++u) x[u] = sc[(int64_t)min(r + u, rows - 1) * a.ld_sc];
  };
  float *const at = a.weights + (int64_t)bh * a.L + j;
  float w = 0.f, x[F];
  if (rows > 0) fetch(x, 0);
  const float before = *at;
  for (int r0 = 0; r0 < rows; r0 += 256) {
    __syncthreads();
    if (r0 + (int)threadIdx.x < rows) {
      // the row's maximum and sum over its chunks
      const int r = r0 + threadIdx.x, rb = r / a.rp;
      const float *const ml =
          a.pml + (((int64_t)bh * a.rblocks + rb) * a.nchunks * a.rp + (r - rb * a.rp)) * 2;
      float m = -INFINITY, l = 0.f;
      for (int c0 = 0; c0 < a.nchunks; c0 += C) {
        float cm[C], cl[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const float *const p = ml + (int64_t)min(c0 + c, a.nchunks - 1) * 2 * a.rp;
          cm[c] = p[0];
          cl[c] = p[1];
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const float mn = fmaxf(m, cm[c]), ref = mn == -INFINITY ? 0.f : mn;
          const float more = c0 + c < a.nchunks ? cl[c] : 0.f;
          l = l * __builtin_amdgcn_exp2f(m - ref) + more * __builtin_amdgcn_exp2f(cm[c] - ref);
          m = mn;
        }
      }
      s_m[threadIdx.x] = m == -INFINITY ? 0.f : m;
      s_i[threadIdx.x] = l == 0.f ? 0.f : 1.f / l;
    }
    __syncthreads();
    const int most = min(256, rows - r0);
    int t = r0 / a.G, g = r0 - t * a.G;
    for (int r = 0; r < most; r += F) {
      float y[F];
#pragma unroll
      for (int u = 0; u < F; ++u) y[u] = x[u];
      if (r0 + r + F < rows) fetch(x, r0 + r + F);
#pragma unroll
      for (int u = 0; u < F; ++u) {
        const bool see = (r + u < most) & win_sees(a, s.first + t, j);
        const int q = min(r + u, most - 1);
        const float p = __builtin_amdgcn_exp2f(y[u] - s_m[q]) * s_i[q];
        w += see ? p : 0.f;
        if (++g == a.G) g = 0, ++t;
      }
    }
  }
  if (i < n) *at = before + w;
}

}  // namespace mtp
