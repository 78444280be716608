// Rows of activations to 8-bit integers with one scale per row, optionally
// after a LayerNorm or a group norm with its activation (pq8_quantize_rows,
// pq8_layer_norm_quantize, pq8_group_norm_quantize; the rows' int8 product is
// pq8_i8.cuh).
//
//   s = max|h| / 127 (rounded to fp32),  q = h / s to the nearest integer, ties to even.
//
// The integers are those of the exact quotient, whatever h is computed from.
// A one-step difference in one value moves an output of the product that
// follows by about 1/1000 of its size, far more than the fp32 rounding of
// everything else, so "nearly always the nearest integer" would not do.
// Each value is computed in fp32 with a bound on its error; the few whose
// quotient lies within that bound of a border between two integers (about one
// in 10^4) are computed again in fp64, and so are the candidates for the
// row's maximum. Row sums (mean, variance) are fp64.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "pq8_block.cuh"
#include "pq8_device.cuh"

namespace pq8 {

// ---------------------------------------------------------------------------
// Element types (PQ8_F32, PQ8_F16, PQ8_BF16)
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// Rounded to nearest even once.
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// Elements of a 16-byte chunk.
template <typename T>
constexpr int kChunk = 16 / static_cast<int>(sizeof(T));

// `E` consecutive elements as floats; one 16-byte load when `vec` says the address allows it.
template <typename T, int E>
__device__ __forceinline__ void load_chunk(const T* p, bool vec, float (&v)[E]) {
  static_assert(E * sizeof(T) == 16, "a chunk is 16 bytes");
  if (vec) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = to_f32(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = to_f32(p[i]);
  }
}
template <typename T, int E>
__device__ __forceinline__ void store_chunk(T* p, bool vec, const float (&v)[E]) {
  if (vec) {
    uint4 u;
    T* t = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < E; ++i) t[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = u;
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) p[i] = from_f32<T>(v[i]);
  }
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_max_f64(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Reductions over the WARPS warps that share a row. Sums are added in a fixed
// order (lanes by butterfly, then warps in turn).
template <int WARPS>
struct RowTeam {
  double* smem;  // WARPS doubles, when WARPS > 1
  __device__ __forceinline__ int index() const { return WARPS == 1 ? (threadIdx.x & 31) : static_cast<int>(threadIdx.x); }
  __device__ __forceinline__ double gather(double v, bool sum) const {
    if constexpr (WARPS == 1) {
      return v;
    } else {
      __syncthreads();  // the previous reduction has been read
      if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
      __syncthreads();
      double r = smem[0];
#pragma unroll
      for (int i = 1; i < WARPS; ++i) r = sum ? r + smem[i] : fmax(r, smem[i]);
      return r;
    }
  }
  __device__ __forceinline__ double sum(double v) const { return gather(warp_sum_f64(v), true); }
  __device__ __forceinline__ double max(double v) const { return gather(warp_max_f64(v), false); }
  __device__ __forceinline__ float max(float v) const {
    return WARPS == 1 ? warp_max(v) : static_cast<float>(gather(static_cast<double>(warp_max(v)), false));
  }
  __device__ __forceinline__ bool any(bool p) const {
    return WARPS == 1 ? __any_sync(0xffffffffu, p) : __syncthreads_or(p) != 0;
  }
};

__device__ __forceinline__ double act_f64(double z, int epi) {
  if (epi == PQ8_EPI_RELU) return z > 0.0 ? z : 0.0;
  if (epi == PQ8_EPI_SILU) return z / (1.0 + exp(-z));
  return z;
}
__device__ __forceinline__ float act_f32(float z, int epi) {
  if (epi == PQ8_EPI_RELU) return fmaxf(z, 0.0f);
  if (epi == PQ8_EPI_SILU) return silu_exact(z);
  return z;
}

// ---------------------------------------------------------------------------
// Where a row's values come from. A source gives, for a chunk of columns, the
// fp32 values, whose error against the exact ones is at most
// rel |value| + abs; and the exact value of one column in fp64.

// The row itself: nothing to compute, no error.
template <typename T>
struct PlainSource {
  static constexpr bool kExact = true, kLayerNorm = false;
  static constexpr int E = kChunk<T>;
  const T* x;
  bool vec;
  float rel = 0.0f, abs = 0.0f;
  __device__ __forceinline__ void raw(int c, float (&v)[E]) const { load_chunk<T, E>(x + c * E, vec, v); }
  template <typename Team>
  __device__ __forceinline__ void prepare(const Team&, int, const float*, int) {}
  __device__ __forceinline__ void value(int, float (&)[E]) const {}
  __device__ __forceinline__ double exact(int col) const { return static_cast<double>(to_f32(x[col])); }
};

// LayerNorm of the row. fp32 error: the deviation (x - mean_hi) - mean_lo is
// rounded twice relative to its own size (the mean's own rounding is in
// mean_lo), then one rounding each for rstd, the product and the multiply-add:
// under 6 x 2^-24 (|h| + |b|), taken as 2^-21.
template <typename T>
struct LayerNormSource {
  static constexpr bool kExact = false, kLayerNorm = true;
  static constexpr int E = kChunk<T>;
  const T* x;
  bool vec;
  const float* w;
  const float* b;
  double eps;
  float rel = 0x1p-21f, abs = 0.0f;
  double mean = 0.0, rstd = 0.0;
  float mean_hi = 0.0f, mean_lo = 0.0f, rs = 0.0f;
  __device__ __forceinline__ void raw(int c, float (&v)[E]) const { load_chunk<T, E>(x + c * E, vec, v); }
  // Mean and variance of the row: from the chunks held in `cached` (chunk
  // index + j * team size), or read again when cached is NULL.
  template <typename Team, int CHUNKS>
  __device__ __forceinline__ void stats(const Team& team, int threads, const float (&cached)[CHUNKS * E], int chunks) {
    const int tid = team.index();
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j)
      if (tid + j * threads < chunks) {
#pragma unroll
        for (int i = 0; i < E; ++i) s += static_cast<double>(cached[j * E + i]);
      }
    mean = team.sum(s) / (static_cast<double>(chunks) * E);
    double q = 0.0;
    float bm = 0.0f;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j)
      if (tid + j * threads < chunks) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const double d = static_cast<double>(cached[j * E + i]) - mean;
          q += d * d;
          bm = fmaxf(bm, fabsf(b[(tid + j * threads) * E + i]));
        }
      }
    finish(team, q, bm, chunks);
  }
  template <typename Team>
  __device__ __forceinline__ void stats_streamed(const Team& team, int threads, int chunks) {
    const int tid = team.index();
    double s = 0.0;
    float v[E];
    for (int c = tid; c < chunks; c += threads) {
      raw(c, v);
#pragma unroll
      for (int i = 0; i < E; ++i) s += static_cast<double>(v[i]);
    }
    mean = team.sum(s) / (static_cast<double>(chunks) * E);
    double q = 0.0;
    float bm = 0.0f;
    for (int c = tid; c < chunks; c += threads) {
      raw(c, v);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const double d = static_cast<double>(v[i]) - mean;
        q += d * d;
        bm = fmaxf(bm, fabsf(b[c * E + i]));
      }
    }
    finish(team, q, bm, chunks);
  }
  template <typename Team>
  __device__ __forceinline__ void finish(const Team& team, double q, float bm, int chunks) {
    rstd = 1.0 / sqrt(team.sum(q) / (static_cast<double>(chunks) * E) + eps);
    abs = 0x1p-21f * team.max(bm);
    mean_hi = static_cast<float>(mean);
    mean_lo = static_cast<float>(mean - static_cast<double>(mean_hi));
    rs = static_cast<float>(rstd);
  }
  __device__ __forceinline__ void value(int c, float (&v)[E]) const {
#pragma unroll
    for (int i = 0; i < E; ++i)
      v[i] = fmaf(((v[i] - mean_hi) - mean_lo) * rs, __ldg(w + c * E + i), __ldg(b + c * E + i));
  }
  __device__ __forceinline__ double exact(int col) const {
    return (static_cast<double>(to_f32(x[col])) - mean) * rstd * static_cast<double>(w[col]) +
           static_cast<double>(b[col]);
  }
};

// Group norm with its activation; mean and 1 / sqrt(var + eps) of the row's
// window come from tables indexed by group. The error bound adds the
// activation's: |act'| <= 1.1, and SiLU's own rounding.
struct GroupStat {
  double mean, rstd;
};
template <typename T>
struct GroupNormSource {
  static constexpr bool kExact = false, kLayerNorm = false;
  static constexpr int E = kChunk<T>;
  const T* x;
  bool vec;
  const float* w;
  const float* b;
  const GroupStat* stat;  // [groups], shared memory
  int group_width;
  int epi;
  float rel = 0x1p-20f, abs;  // abs = 2^-20 (max|b| + 1)
  __device__ __forceinline__ void raw(int c, float (&v)[E]) const { load_chunk<T, E>(x + c * E, vec, v); }
  __device__ __forceinline__ void value(int c, float (&v)[E]) const {
    int g = c * E / group_width, left = (g + 1) * group_width - c * E;
    GroupStat s = stat[g];
    float hi = static_cast<float>(s.mean), lo = static_cast<float>(s.mean - static_cast<double>(hi));
    float rs = static_cast<float>(s.rstd);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (left == 0) {
        s = stat[++g];
        left = group_width;
        hi = static_cast<float>(s.mean);
        lo = static_cast<float>(s.mean - static_cast<double>(hi));
        rs = static_cast<float>(s.rstd);
      }
      --left;
      v[i] = act_f32(fmaf(((v[i] - hi) - lo) * rs, __ldg(w + c * E + i), __ldg(b + c * E + i)), epi);
    }
  }
  __device__ __forceinline__ double exact(int col) const {
    const GroupStat s = stat[col / group_width];
    const double z = (static_cast<double>(to_f32(x[col])) - s.mean) * s.rstd * static_cast<double>(w[col]) +
                     static_cast<double>(b[col]);
    return act_f64(z, epi);
  }
};

// ---------------------------------------------------------------------------
// One row, by a team of WARPS warps. CHUNKS > 0: each thread holds up to CHUNKS
// chunks of the row in registers (width <= CHUNKS * E * 32 * WARPS);
// CHUNKS == 0: any width, read again in each pass. `width` is a multiple of
// E; q is E-byte aligned. Every thread of the team returns the scale.
template <int CHUNKS, int WARPS, typename Src>
__device__ __forceinline__ float quantize_row(Src src, int width, int8_t* q, const RowTeam<WARPS>& team) {
  constexpr int E = Src::E;
  constexpr int kThreads = WARPS * 32;
  constexpr bool kCached = CHUNKS > 0;
  constexpr int N = kCached ? CHUNKS : 1;
  static_assert(!kCached || N * E <= 32, "one mask bit per value");
  const int tid = team.index(), chunks = width / E;
  float v[N * E];
  if constexpr (kCached) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float c4[E];
      const int c = tid + j * kThreads;
      if (c < chunks) src.raw(c, c4);
#pragma unroll
      for (int i = 0; i < E; ++i) v[j * E + i] = c < chunks ? c4[i] : 0.0f;
    }
    if constexpr (Src::kLayerNorm) src.template stats<RowTeam<WARPS>, N>(team, kThreads, v, chunks);
  } else {
    if constexpr (Src::kLayerNorm) src.stats_streamed(team, kThreads, chunks);
  }
  // f(first register, chunk) for every chunk of this thread
  auto each = [&](auto&& f, bool compute) {
    if constexpr (kCached) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = tid + j * kThreads;
        if (c < chunks) {
          float(&c4)[E] = *reinterpret_cast<float(*)[E]>(v + j * E);
          if (compute) src.value(c, c4);
          f(c4, c, j * E);
        }
      }
    } else {
      for (int c = tid; c < chunks; c += kThreads) {
        float(&c4)[E] = *reinterpret_cast<float(*)[E]>(v);
        src.raw(c, c4);
        src.value(c, c4);
        f(c4, c, 0);
      }
    }
  };
  // column of mask bit `bit` (cached rows)
  auto column = [&](int bit) { return (tid + (bit / E) * kThreads) * E + bit % E; };

  float low = 0.0f;  // a lower bound on the row's maximum
  bool bad = false;
  each([&](const float(&c4)[E], int, int) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float a = fabsf(c4[i]);
      bad |= !(a <= 3.402823466e38f);
      low = fmaxf(low, a - (src.rel * a + src.abs));
    }
  }, true);
  auto zeros = [&] {
    for (int c = tid; c < chunks; c += kThreads)
#pragma unroll
      for (int i = 0; i < E; i += 4) *reinterpret_cast<uint32_t*>(q + c * E + i) = 0u;
  };
  if (team.any(bad)) {  // an infinity or a NaN in the row: no scale, no values
    zeros();
    return __int_as_float(0x7fc00000);
  }
  low = team.max(low);
  float s;
  if constexpr (Src::kExact) {
    s = low / 127.0f;
  } else {
    double top = 0.0;
    uint32_t near = 0;
    each([&](const float(&c4)[E], int c, int bit) {
      uint32_t here = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float a = fabsf(c4[i]);
        if (a + (src.rel * a + src.abs) >= low) here |= 1u << i;
      }
      if constexpr (kCached) {
        near |= here << bit;
      } else {
        for (; here; here &= here - 1) top = fmax(top, ::fabs(src.exact(c * E + __ffs(here) - 1)));
      }
    }, false);
    for (; near; near &= near - 1) top = fmax(top, ::fabs(src.exact(column(__ffs(near) - 1))));
    s = static_cast<float>(team.max(top) / 127.0);
  }
  if (s == 0.0f) {  // a row of zeros, or of values too small for a scale
    zeros();
    return 0.0f;
  }
  const double s64 = static_cast<double>(s);
  const float inv = 1.0f / s;
  // below this, 1 / s may leave fp32's range: every quotient in fp64
  const bool all_exact = s < 0x1p-100f;
  const float tol_rel = src.rel + 0x1p-22f, tol_abs = src.abs * inv;
  auto exact_q = [&](int col) {
    return static_cast<int8_t>(static_cast<int>(fmin(fmax(rint(src.exact(col) / s64), -127.0), 127.0)));
  };
  uint32_t fix = 0;
  each([&](const float(&c4)[E], int c, int bit) {
    uint32_t here = 0, m[E], word[E / 4];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      // adding 1.5 x 2^23 rounds to an integer (nearest even) and leaves it in the low bits
      const float t = c4[i] * inv, big = t + 12582912.0f, r = big - 12582912.0f;
      m[i] = __float_as_uint(big);
      // not (|t - r| below the border by more than the error), NaN included
      if (!(fabsf(t - r) < 0.5f - fmaf(fabsf(t), tol_rel, tol_abs)) || all_exact) here |= 1u << i;
    }
#pragma unroll
    for (int i = 0; i < E; i += 4)
      word[i >> 2] = __byte_perm(__byte_perm(m[i], m[i + 1], 0x0040), __byte_perm(m[i + 2], m[i + 3], 0x0040), 0x5410);
    if constexpr (E == 4) {
      *reinterpret_cast<uint32_t*>(q + c * E) = word[0];
    } else {
      *reinterpret_cast<uint2*>(q + c * E) = make_uint2(word[0], word[E / 4 - 1]);
    }
    if constexpr (kCached) {
      fix |= here << bit;
    } else {
      for (; here; here &= here - 1) {
        const int col = c * E + __ffs(here) - 1;
        q[col] = exact_q(col);
      }
    }
  }, false);
  for (; fix; fix &= fix - 1) {
    const int col = column(__ffs(fix) - 1);
    q[col] = exact_q(col);
  }
  return s;
}

constexpr int kRowThreads = 256;

// Rows of a [rows, width] matrix (row stride ld elements), each quantised by
// a team of WARPS warps: a warp per row up to 1024 columns, the CTA's eight
// warps up to 8192 (the row stays in registers in both), and past that the
// CTA reads the row again in each pass. NORM: LayerNorm first.
template <typename T, int CHUNKS, int WARPS, bool NORM>
__global__ void __launch_bounds__(kRowThreads)
    quantize_rows_kernel(const T* __restrict__ x, long long ld, const float* __restrict__ w,
                         const float* __restrict__ b, double eps, int8_t* __restrict__ q, float* __restrict__ scale,
                         int rows, int width, int vec) {
  __shared__ double team_smem[WARPS];
  constexpr int kTeams = kRowThreads / (32 * WARPS);
  const RowTeam<WARPS> team{team_smem};
  griddep_wait();    // x is the previous kernel's output
  griddep_launch();  // only now: what the next kernel reads ahead of its own wait is then older than this kernel
  const int first = static_cast<int>(blockIdx.x) * kTeams + static_cast<int>(threadIdx.x) / (32 * WARPS);
  for (long long row = first; row < rows; row += static_cast<long long>(gridDim.x) * kTeams) {
    const T* xr = x + row * ld;
    int8_t* qr = q + row * width;
    float s;
    if constexpr (NORM) {
      LayerNormSource<T> src;
      src.x = xr;
      src.vec = vec != 0;
      src.w = w;
      src.b = b;
      src.eps = eps;
      s = quantize_row<CHUNKS, WARPS>(src, width, qr, team);
    } else {
      PlainSource<T> src;
      src.x = xr;
      src.vec = vec != 0;
      s = quantize_row<CHUNKS, WARPS>(src, width, qr, team);
    }
    if (team.index() == 0) scale[row] = s;
  }
}

}  // namespace pq8
