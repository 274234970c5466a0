// Sums of the windowed attention's probabilities by key (wattn.hpp), from the
// scores that it kept.
#pragma once

#include "wattn.hpp"

namespace mtp {

// The weight of every key that a query saw, added to a.weights: sum over the
// rows of the key's head of exp2(score - max) / sum, rows in order, so the
// result does not depend on timing. Grid (keys / 256, B * Hk).
__global__ void __launch_bounds__(256) win_weights_kernel(const WinArgs a) {
  __shared__ float s_m[256], s_i[256];
  const int bh = blockIdx.y, b = bh / a.Hk;
  const WinSpan s = win_span(a, b);
  const int n = s.count();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if ((int)blockIdx.x * 256 >= n) return;  // the whole workgroup
  const int rows = a.G * a.T;
  float w = 0.f;
  for (int r0 = 0; r0 < rows; r0 += 256) {
    const int r = r0 + threadIdx.x;
    __syncthreads();
    if (r < rows) {
      const float *const ml = a.ml + ((int64_t)bh * rows + r) * 2;
      const float m = ml[0], l = ml[1];
      s_m[threadIdx.x] = m == -INFINITY ? 0.f : m;
      s_i[threadIdx.x] = l == 0.f ? 0.f : 1.f / l;
    }
    __syncthreads();
    if (i < n) {
      const int most = min(256, rows - r0);
      const float *const sc = a.scores + ((int64_t)bh * rows + r0) * a.ld_sc + i;
      // a row keeps the scores of the keys that it sees (and perhaps others)
      for (int r = 0; r < most; ++r) {
        const int t = (r0 + r) / a.G;
        if (t < s.rows && win_sees(a, s.first + t, s.key(i)))
          w = fmaf(__builtin_amdgcn_exp2f(sc[(int64_t)r * a.ld_sc] - s_m[r]), s_i[r], w);
      }
    }
  }
  if (i < n) a.weights[(int64_t)bh * a.L + s.key(i)] += w;
}

}  // namespace mtp
