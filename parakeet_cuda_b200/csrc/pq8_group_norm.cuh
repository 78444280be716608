// Group norm with an activation, channels last (pq8_group_norm,
// pq8_group_norm_quantize): rows of `channels` values, windows of consecutive
// rows; mean and variance over the rows of one window and the channels of one
// group,
//   y = act((x - mean) / sqrt(var + eps) * w + b).
// Sums are fp64, taken of x minus the group's first value of the window, so
// that neither a large common offset nor a long window costs digits.
#pragma once

#include "pq8_rows.cuh"

namespace pq8 {

struct GroupNormParams {
  const void* x;
  const float* w;  // [channels]
  const float* b;  // [channels]
  const int* offsets;  // [windows + 1], or NULL: windows of rows / windows rows
  int rows, windows, channels, groups, epi, round_out;
  double eps;
  int chunks;      // row chunks per window of the sums
  int slab;        // whole groups per CTA
};

// Rows [lo, hi) of window w. Offsets come from device memory: they are held
// to 0 <= lo <= hi <= rows, whatever they say.
__device__ __forceinline__ void window_rows(const GroupNormParams& p, int w, int* lo, int* hi) {
  if (p.offsets == nullptr) {
    const int t = p.rows / p.windows;
    *lo = w * t;
    *hi = *lo + t;
  } else {
    *lo = min(max(p.offsets[w], 0), p.rows);
    *hi = min(max(p.offsets[w + 1], *lo), p.rows);
  }
}

// The rows of chunk `c` of `chunks` equal parts of [lo, hi).
__device__ __forceinline__ void chunk_rows(int lo, int hi, int c, int chunks, int* r0, int* r1) {
  const int per = (hi - lo + chunks - 1) / chunks;
  *r0 = min(static_cast<long long>(lo) + static_cast<long long>(c) * per, static_cast<long long>(hi));
  *r1 = min(*r0 + per, hi);
}

constexpr int kNormThreads = 256;

// How a CTA's threads cover rows of a slab of `cols` columns in units of U:
// `tx` threads along the columns, `ty` rows at a time.
struct SlabShape {
  int units, tx, ty, x, y;
  __device__ __forceinline__ SlabShape(int cols, int unit) {
    units = cols / unit;
    tx = min(units, kNormThreads);
    ty = kNormThreads / tx;
    x = static_cast<int>(threadIdx.x) % tx;
    y = static_cast<int>(threadIdx.x) / tx;
  }
};

struct GroupSum {
  double s, q;  // sums of x - first and its square
};

// Partial sums of one row chunk of one window for the groups of one slab:
// partial[window][chunk][group]. Thread (x, y) adds rows y, y + ty, ... of
// its columns; then a warp per group adds the threads' sums in a fixed order.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kNormThreads)
    group_stats_kernel(const GroupNormParams p, GroupSum* __restrict__ partial) {
  constexpr int E = VEC ? kChunk<T> : 1;
  __shared__ GroupSum red[kNormThreads];
  griddep_wait();
  griddep_launch();
  const int cg = p.channels / p.groups, g0 = static_cast<int>(blockIdx.z) * p.slab, ng = min(p.slab, p.groups - g0);
  for (int w = blockIdx.y; w < p.windows; w += gridDim.y) {
    int lo, hi, r0, r1;
    window_rows(p, w, &lo, &hi);
    chunk_rows(lo, hi, blockIdx.x, p.chunks, &r0, &r1);
    const SlabShape sh(ng * cg, E);
    const T* x = static_cast<const T*>(p.x) + static_cast<size_t>(g0) * cg;
    GroupSum a{0.0, 0.0};
    if (sh.y < sh.ty) {
      for (int u = sh.x; u < sh.units; u += sh.tx) {  // more than one pass only when the slab is one group
        const int g = u * E / cg;
        const float first = lo < hi ? to_f32(x[static_cast<size_t>(lo) * p.channels + static_cast<size_t>(g) * cg]) : 0.0f;
        for (int r = r0 + sh.y; r < r1; r += sh.ty) {
          const T* xr = x + static_cast<size_t>(r) * p.channels + u * E;
          float v[E];
          if constexpr (VEC) load_chunk<T, E>(xr, true, v);
          else v[0] = to_f32(xr[0]);
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const double d = static_cast<double>(v[i]) - static_cast<double>(first);
            a.s += d;
            a.q += d * d;
          }
        }
      }
    }
    __syncthreads();  // red has been read (previous window)
    red[threadIdx.x] = a;
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = ng > 1 ? cg / E : sh.tx;  // threads along x of one group
    for (int g = warp; g < ng; g += kNormThreads / 32) {
      double s = 0.0, q = 0.0;
      for (int i = lane; i < per * sh.ty; i += 32) {
        const GroupSum t = red[(i / per) * sh.tx + g * per + i % per];
        s += t.s;
        q += t.q;
      }
      s = warp_sum_f64(s);
      q = warp_sum_f64(q);
      if (lane == 0)
        partial[(static_cast<size_t>(w) * p.chunks + blockIdx.x) * p.groups + g0 + g] = GroupSum{s, q};
    }
  }
}

// Mean and 1 / sqrt(var + eps) of groups [g0, g0 + ng) of a window, from its
// chunks' sums added in chunk order, into `stat` (shared memory). All threads.
template <typename T>
__device__ __forceinline__ void group_finish(const GroupNormParams& p, const GroupSum* partial, int w, int lo, int hi,
                                             int g0, int ng, GroupStat* stat) {
  const int cg = p.channels / p.groups;
  const T* x = static_cast<const T*>(p.x);
  __syncthreads();  // stat has been read (previous window)
  for (int g = threadIdx.x; g < ng; g += blockDim.x) {
    double s = 0.0, q = 0.0;
    for (int c = 0; c < p.chunks; ++c) {
      const GroupSum t = partial[(static_cast<size_t>(w) * p.chunks + c) * p.groups + g0 + g];
      s += t.s;
      q += t.q;
    }
    if (hi > lo) {
      const double n = static_cast<double>(hi - lo) * cg;
      const double first =
          static_cast<double>(to_f32(x[static_cast<size_t>(lo) * p.channels + static_cast<size_t>(g0 + g) * cg]));
      const double m = s / n;
      stat[g] = GroupStat{first + m, 1.0 / sqrt(fmax(q / n - m * m, 0.0) + p.eps)};
    }
  }
  __syncthreads();
}

// Normalise and activate the rows of one chunk of one window, one slab.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kNormThreads)
    group_apply_kernel(const GroupNormParams p, const GroupSum* __restrict__ partial, T* __restrict__ y) {
  constexpr int E = VEC ? kChunk<T> : 1;
  extern __shared__ GroupStat stat[];
  griddep_wait();
  griddep_launch();
  const int cg = p.channels / p.groups, g0 = static_cast<int>(blockIdx.z) * p.slab, ng = min(p.slab, p.groups - g0);
  for (int w = blockIdx.y; w < p.windows; w += gridDim.y) {
    int lo, hi, r0, r1;
    window_rows(p, w, &lo, &hi);
    chunk_rows(lo, hi, blockIdx.x, gridDim.x, &r0, &r1);
    group_finish<T>(p, partial, w, lo, hi, g0, ng, stat);
    const SlabShape sh(ng * cg, E);
    if (sh.y >= sh.ty) continue;
    for (int u = sh.x; u < sh.units; u += sh.tx) {
      const GroupStat st = stat[u * E / cg];
      const float m_hi = static_cast<float>(st.mean), m_lo = static_cast<float>(st.mean - static_cast<double>(m_hi));
      const float rs = static_cast<float>(st.rstd);
      const int col = g0 * cg + u * E;
      float g[E], h[E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        g[i] = p.w[col + i];
        h[i] = p.b[col + i];
      }
      for (int r = r0 + sh.y; r < r1; r += sh.ty) {
        const size_t at = static_cast<size_t>(r) * p.channels + col;
        float v[E];
        if constexpr (VEC) load_chunk<T, E>(static_cast<const T*>(p.x) + at, true, v);
        else v[0] = to_f32(static_cast<const T*>(p.x)[at]);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          v[i] = act_f32(fmaf(((v[i] - m_hi) - m_lo) * rs, g[i], h[i]), p.epi);
          if (p.round_out) v[i] = tf32_round(v[i]);
        }
        if constexpr (VEC) store_chunk<T, E>(y + at, true, v);
        else y[at] = from_f32<T>(v[0]);
      }
    }
  }
}

// Normalise, activate and quantise the rows of one chunk of one window: rows
// whole, as their scale needs every channel.
template <typename T, int CHUNKS, int WARPS, bool VEC>
__global__ void __launch_bounds__(kRowThreads, 3)
    group_quantize_kernel(const GroupNormParams p, const GroupSum* __restrict__ partial, int8_t* __restrict__ q,
                          float* __restrict__ scale) {
  extern __shared__ GroupStat stat[];  // [groups], then their fp32 form
  float4* const fast = reinterpret_cast<float4*>(stat + p.groups);
  __shared__ double team_smem[2 * WARPS];
  __shared__ float warp_top[kRowThreads / 32];
  constexpr int kTeams = kRowThreads / (32 * WARPS);
  const RowTeam<WARPS> team{team_smem};
  griddep_wait();
  griddep_launch();
  GroupNormSource<T, VEC> src;
  src.w = p.w;
  src.b = p.b;
  src.stat = stat;
  src.fast = fast;
  src.group_width = p.channels / p.groups;
  src.whole = src.group_width % kChunk<T> == 0;
  src.epi = p.epi;
  src.top_b = cta_max_abs(p.b, p.channels, warp_top);
  for (int w = blockIdx.y; w < p.windows; w += gridDim.y) {
    int lo, hi, r0, r1;
    window_rows(p, w, &lo, &hi);
    chunk_rows(lo, hi, blockIdx.x, gridDim.x, &r0, &r1);
    group_finish<T>(p, partial, w, lo, hi, 0, p.groups, stat);
    for (int g = threadIdx.x; g < p.groups; g += blockDim.x) {
      const float m = static_cast<float>(stat[g].mean);
      fast[g] = make_float4(m, static_cast<float>(stat[g].mean - static_cast<double>(m)),
                            static_cast<float>(stat[g].rstd), 0.0f);
    }
    __syncthreads();
    for (int r = r0 + static_cast<int>(threadIdx.x) / (32 * WARPS); r < r1; r += kTeams) {
      src.x = static_cast<const T*>(p.x) + static_cast<size_t>(r) * p.channels;
      const float s = quantize_row<CHUNKS, WARPS>(src, p.channels, q + static_cast<size_t>(r) * p.channels, team);
      if (team.index() == 0) scale[r] = s;
    }
  }
}

}  // namespace pq8
