// Products of a few rows with 4-bit weights under group scales (dsv41_gemv_w4):
// y[m][n] = sum over groups of s[n][g] * sum over k in g of x[m][k] (w[n][k] - z[n][g]).
#pragma once

#include "gqa.cuh"

namespace dsv41 {

constexpr int kW4MaxRows = 48;

struct GemvW4Args {
  const uint8_t* w;
  const void* scales;
  const uint8_t* zeros;  // or null: 8
  const void* x;
  void* y;
  int M, N, K, group;
  int64_t x_ld, y_ld;
};

// Grid ceil(N / 8), 256 threads: a warp a weight row; the lanes take its 8-weight words in turn.
template <bool F16>
__global__ void __launch_bounds__(256) gemv_w4_kernel(const GemvW4Args a) {
  using T = typename Act<F16>::T;
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= a.N) return;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(a.w + (int64_t)n * (a.K / 2));
  const int groups = a.K / a.group;
  const T* sc = reinterpret_cast<const T*>(a.scales) + (int64_t)n * groups;
  for (int m0 = 0; m0 < a.M; m0 += 8) {
    float acc[8] = {};
    for (int i = lane; i < a.K / 8; i += 32) {
      const int g = 8 * i / a.group;
      const uint32_t v = w[i];
      const float s = Act<F16>::f(sc[g]);
      const int z = a.zeros ? a.zeros[(int64_t)n * groups + g] : 8;
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        if (m0 + m >= a.M) break;
        const T* x = reinterpret_cast<const T*>(a.x) + (m0 + m) * a.x_ld + 8 * i;
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) t += Act<F16>::f(x[j]) * (float)((int)((v >> (4 * j)) & 15) - z);
        acc[m] += t * s;
      }
    }
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const float t = warp_sum(acc[m]);
      if (lane == 0 && m0 + m < a.M) reinterpret_cast<T*>(a.y)[(m0 + m) * a.y_ld + n] = Act<F16>::r(t);
    }
  }
}

}  // namespace dsv41
