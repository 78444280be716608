// Matrix product in 8-bit integers with a scale per token and per channel
// (pq8_gemm_i8, pq8_linear_i8):
//
//   acc[m, j] = sum_k q[m, k] w[j, k]        (exact, 32-bit integers)
//   y[m, j]   = epilogue(acc s[m] t[j] + bias[j])
//
// Integer sums have one value whatever their order, so splitting K over CTAs
// or threads changes no bit of the result.
#pragma once

#include <cuda.h>

#include "pq8_rows.cuh"

namespace pq8 {

struct I8Params {
  const int8_t* w;       // [n, k]
  const float* w_scale;  // [n]
  const int8_t* x;       // [m, k]
  const float* x_scale;  // [m]
  void* y;               // [m, out_cols]
  const float* bias;     // [n] or NULL
  const void* resid;     // [m, out_cols], y's type
  int* status;
  int m, n, k, epi, out_cols;
  float alpha;
};

// The value of one output before the activation; bias may be absent (0).
__device__ __forceinline__ float i8_scaled(int acc, float s, float t, float b) {
  return fmaf(static_cast<float>(acc) * s, t, b);
}

// ---------------------------------------------------------------------------
// A few tokens (m <= 8 per pass): the weights are read once, 16 bytes per lane, by
// dp4a; HBM-bound. A warp takes R channels over the whole of K, a lane every
// 32nd 16-byte chunk; the lanes' sums meet in one reduction per output.
constexpr int kI8GemvThreads = 256;

template <typename T, int M, int R>
__global__ void __launch_bounds__(kI8GemvThreads) i8_gemv_kernel(const I8Params p) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31;
  const int unit = static_cast<int>(blockIdx.x) * (kI8GemvThreads / 32) + (threadIdx.x >> 5);
  const bool glu = p.epi == PQ8_EPI_GLU;
  const int half = p.n >> 1;
  // channel of local row r: consecutive ones, or for GLU the pairs (j, j + n / 2)
  constexpr int P = R > 1 ? R / 2 : 1;
  const int j0 = unit * (glu ? P : R);
  if (j0 >= p.out_cols) return;
  auto channel = [&](int r) { return glu ? (r < P ? j0 + r : half + j0 + r - P) : j0 + r; };
  auto valid = [&](int r) { return glu ? j0 + r % P < half : j0 + r < p.n; };
  const int chunks = p.k >> 4;
  for (int m0 = static_cast<int>(blockIdx.y) * M; m0 < p.m; m0 += static_cast<int>(gridDim.y) * M) {
  int acc[R][M];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < M; ++i) acc[r][i] = 0;
  const int4* wrow[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    wrow[r] = reinterpret_cast<const int4*>(p.w + static_cast<size_t>(valid(r) ? channel(r) : 0) * p.k);
  const int4* xrow[M];
#pragma unroll
  for (int i = 0; i < M; ++i)
    xrow[i] = reinterpret_cast<const int4*>(p.x + static_cast<size_t>(min(m0 + i, p.m - 1)) * p.k);
#pragma unroll 2
  for (int c = lane; c < chunks; c += 32) {
    int4 wv[R];
#pragma unroll
    for (int r = 0; r < R; ++r) wv[r] = __ldg(wrow[r] + c);
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int4 xv = __ldg(xrow[i] + c);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        acc[r][i] = __dp4a(wv[r].x, xv.x, acc[r][i]);
        acc[r][i] = __dp4a(wv[r].y, xv.y, acc[r][i]);
        acc[r][i] = __dp4a(wv[r].z, xv.z, acc[r][i]);
        acc[r][i] = __dp4a(wv[r].w, xv.w, acc[r][i]);
      }
    }
  }
  // every lane gets every sum; lane i keeps the outputs of token i
  int mine[R];
#pragma unroll
  for (int r = 0; r < R; ++r) mine[r] = 0;
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int sum = __reduce_add_sync(0xffffffffu, acc[r][i]);
      if (lane == i) mine[r] = sum;
    }
  const int row = m0 + lane;
  if (lane >= M || row >= p.m) continue;
  const float s = p.x_scale[row];
  float z[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = valid(r) ? channel(r) : 0;
    z[r] = i8_scaled(mine[r], s, p.w_scale[j], p.bias ? p.bias[j] : 0.0f);
  }
  T* y = static_cast<T*>(p.y) + static_cast<size_t>(row) * p.out_cols;
  const T* res = static_cast<const T*>(p.resid) + static_cast<size_t>(row) * p.out_cols;
  if (glu) {
#pragma unroll
    for (int r = 0; r < P; ++r)
      if (valid(r)) y[j0 + r] = from_f32<T>(z[r] / (1.0f + expf(-z[R > 1 ? r + P : 0])));
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (valid(r)) {
        float v = act_f32(z[r], p.epi);
        if (p.epi == PQ8_EPI_RESIDUAL) v = fmaf(p.alpha, z[r], to_f32(res[j0 + r]));
        y[j0 + r] = from_f32<T>(v);
      }
  }
  }
}

}  // namespace pq8
