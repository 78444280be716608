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

#include <type_traits>

#include "pq8_block.cuh"
#include "pq8_device.cuh"

namespace pq8 {

// ---------------------------------------------------------------------------
// Element types (PQ8_TYPE_F32, PQ8_TYPE_F16, PQ8_TYPE_BF16)
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
// `E` consecutive floats of a parameter vector (E a multiple of 4; column of
// a chunk, so 16-byte aligned when the vector is).
template <int E>
__device__ __forceinline__ void load_params(const float* p, bool vec, float (&v)[E]) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(p + i));
      v[i] = u.x;
      v[i + 1] = u.y;
      v[i + 2] = u.z;
      v[i + 3] = u.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = __ldg(p + i);
  }
}
// The largest |b[i]| of a vector, by every thread of the CTA for itself.
__device__ __forceinline__ float cta_max_abs(const float* b, int n, float* smem /* a float per warp */) {
  float top = 0.0f;
  for (int i = threadIdx.x; i < n; i += blockDim.x) top = fmaxf(top, fabsf(b[i]));
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = top;
  __syncthreads();
  top = smem[0];
  for (int i = 1; i < static_cast<int>(blockDim.x >> 5); ++i) top = fmaxf(top, smem[i]);
  return top;
}

// Two fp32 values per instruction (packed operands of sm_100).
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float* a, float* b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(v));
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 1 + e^-z of two values.
__device__ __forceinline__ f32x2 sigmoid_divisors(f32x2 z) {
  float x0, x1;
  unpack2(mul2(z, pack2(-1.44269504f, -1.44269504f)), &x0, &x1);
  return add2(pack2(exp2_approx(x0), exp2_approx(x1)), pack2(1.0f, 1.0f));
}
// Sigmoids of two values of at least kSigmoidLeast. 1 / d, d = 1 + e^-z, takes an exponential
// and a reciprocal from the special-function unit, which bounds epilogues with few
// other operations; here two values share one reciprocal: 1 / d0 = d1 / (d0 d1), a
// product below 2^125.
constexpr float kSigmoidLeast = -43.0f;
__device__ __forceinline__ f32x2 sigmoid2(f32x2 z) {
  float d0, d1;
  unpack2(sigmoid_divisors(z), &d0, &d1);
  const float r = rcp_approx(d0 * d1);
  return mul2(pack2(r, r), pack2(d1, d0));
}
// The same over the whole range: apart where the pair's product is so large that its reciprocal is
// no normal number (or a NaN), and e^z from d > 2^126 on (0 below z = -87.4). SiLU multiplies
// it by z and a GLU by the value, so that any floor would show in the output.
__device__ __forceinline__ f32x2 sigmoid2_apart(f32x2 z) {
  float d[2], x[2];
  unpack2(sigmoid_divisors(z), &d[0], &d[1]);
  const float p = d[0] * d[1], r = rcp_approx(p);
  if (p <= 0x1p126f) return mul2(pack2(r, r), pack2(d[1], d[0]));
  unpack2(z, &x[0], &x[1]);
#pragma unroll
  for (int i = 0; i < 2; ++i) d[i] = d[i] <= 0x1p126f ? rcp_approx(d[i]) : exp2_approx(x[i] * 1.44269504f);
  return pack2(d[0], d[1]);
}
// Callers look at many values at once, by their least (NaN if one is), and take them all
// again by sigmoid2_apart if that is below kSigmoidLeast. (24,000 x 1024 x 4096 with SiLU: 109 us; with a
// test per pair, which the compiler turned into predicated instructions, 119.)
__device__ __forceinline__ void take_least(f32x2 z, float& least) {
  float z0, z1;
  unpack2(z, &z0, &z1);
  asm("min.NaN.f32 %0, %0, %1, %2;" : "+f"(least) : "f"(z0), "f"(z1));
}
template <bool APART>
__device__ __forceinline__ f32x2 sigmoid2(f32x2 z) {
  if constexpr (APART) return sigmoid2_apart(z);
  else return sigmoid2(z);
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
// Of values >= 0, whose bit patterns are ordered as they are: the high words
// first, then the low words of the lanes that have the highest.
__device__ __forceinline__ double warp_max_f64(double v) {
  const unsigned hi = static_cast<unsigned>(__double2hiint(v)), top = __reduce_max_sync(0xffffffffu, hi);
  const unsigned lo = __reduce_max_sync(0xffffffffu, hi == top ? static_cast<unsigned>(__double2loint(v)) : 0u);
  return __hiloint2double(static_cast<int>(top), static_cast<int>(lo));
}

// Reductions over the WARPS warps that share a row. Sums are added in a fixed
// order (lanes by butterfly, then warps in turn).
template <int WARPS>
struct RowTeam {
  double* smem;  // 2 WARPS doubles, when WARPS > 1
  __device__ __forceinline__ int index() const { return WARPS == 1 ? (threadIdx.x & 31) : static_cast<int>(threadIdx.x); }
  __device__ __forceinline__ void sum2(double& a, double& b) const {
    a = warp_sum_f64(a);
    b = warp_sum_f64(b);
    if constexpr (WARPS > 1) {
      __syncthreads();  // the previous reduction has been read
      if ((threadIdx.x & 31) == 0) {
        smem[2 * (threadIdx.x >> 5)] = a;
        smem[2 * (threadIdx.x >> 5) + 1] = b;
      }
      __syncthreads();
      a = smem[0];
      b = smem[1];
#pragma unroll
      for (int i = 1; i < WARPS; ++i) {
        a += smem[2 * i];
        b += smem[2 * i + 1];
      }
    }
  }
  __device__ __forceinline__ double max(double v) const {
    v = warp_max_f64(v);
    if constexpr (WARPS > 1) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
      __syncthreads();
      v = smem[0];
#pragma unroll
      for (int i = 1; i < WARPS; ++i) v = fmax(v, smem[i]);
    }
    return v;
  }
  // of values >= 0 (infinity included), whose bit patterns are ordered as they are
  __device__ __forceinline__ float max(float v) const {
    v = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
    if constexpr (WARPS > 1) {
      float* f = reinterpret_cast<float*>(smem);
      __syncthreads();
      if ((threadIdx.x & 31) == 0) f[threadIdx.x >> 5] = v;
      __syncthreads();
      v = f[0];
#pragma unroll
      for (int i = 1; i < WARPS; ++i) v = fmaxf(v, f[i]);
    }
    return v;
  }
};

// max(z, 0) that a NaN passes (fmaxf would make it 0 and hide a bad row).
__device__ __forceinline__ float relu_f32(float z) {
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(z));
  return r;
}
__device__ __forceinline__ double act_f64(double z, int epi) {
  if (epi == PQ8_EPI_RELU) return z < 0.0 ? 0.0 : z;
  if (epi == PQ8_EPI_SILU) return z / (1.0 + exp(-z));
  return z;
}
// SiLU by the fast exponential and quotient: within 4 x 2^-23 |y| + 2^-23 of the
// exact one (the exponential's error grows with |z|, where e^z shrinks faster).
__device__ __forceinline__ float act_f32(float z, int epi) {
  if (epi == PQ8_EPI_RELU) return relu_f32(z);
  if (epi == PQ8_EPI_SILU) return __fdividef(z, 1.0f + __expf(-z));
  return z;
}

// ---------------------------------------------------------------------------
// Where a row's values come from (VEC: by 16-byte loads, of the row and of the
// norm's parameters). A source gives, for a chunk of columns, the
// fp32 values, whose error against the exact ones is at
// most error(h) for values up to h; and the exact value of one column in fp64.

// The row itself: nothing to compute, no error.
template <typename T, bool VEC>
struct PlainSource {
  static constexpr bool kExact = true, kLayerNorm = false;
  static constexpr int E = kChunk<T>;
  const T* x;
  __device__ __forceinline__ void raw(int c, float (&v)[E]) const { load_chunk<T, E>(x + c * E, VEC, v); }
  __device__ __forceinline__ void value(int, float (&)[E]) const {}
  __device__ __forceinline__ double exact(int col) const { return static_cast<double>(to_f32(x[col])); }
  __device__ __forceinline__ float error(float) const { return 0.0f; }
};

// LayerNorm of the row. fp32 error: the deviation (x - mean_hi) - mean_lo is
// rounded twice relative to its own size (the mean's own rounding is in
// mean_lo), then one rounding each for rstd, the product and the multiply-add:
// under 6 x 2^-24 (|h| + |b|), taken as 2^-21.
template <typename T, bool VEC>
struct LayerNormSource {
  static constexpr bool kExact = false, kLayerNorm = true;
  static constexpr int E = kChunk<T>;
  const T* x;
  const float* w;
  const float* b;
  double eps, inv_width;
  float top_b;  // max|b|
  double mean, rstd;
  float mean_hi, mean_lo, rs;
  __device__ __forceinline__ void raw(int c, float (&v)[E]) const { load_chunk<T, E>(x + c * E, VEC, v); }
  // Sums of x - first and its square: with a value of the row taken off, the
  // square of the mean is at most `width` times the variance, so their
  // difference keeps all but three or four of fp64's digits.
  __device__ __forceinline__ void add(const float (&v)[E], double first, double& s, double& q) const {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const double d = static_cast<double>(v[i]) - first;
      s += d;
      q += d * d;
    }
  }
  template <typename Team>
  __device__ __forceinline__ void finish(const Team& team, double first, double s, double q) {
    team.sum2(s, q);
    const double m = s * inv_width;
    mean = first + m;
    rstd = rsqrt(fmax(q * inv_width - m * m, 0.0) + eps);
    mean_hi = static_cast<float>(mean);
    mean_lo = static_cast<float>(mean - static_cast<double>(mean_hi));
    rs = static_cast<float>(rstd);
  }
  __device__ __forceinline__ void value(int c, float (&v)[E]) const {
    float g[E], h[E];
    load_params<E>(w + c * E, VEC, g);
    load_params<E>(b + c * E, VEC, h);
    const f32x2 hi = pack2(-mean_hi, -mean_hi), lo = pack2(-mean_lo, -mean_lo), r2 = pack2(rs, rs);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const f32x2 d = mul2(add2(add2(pack2(v[i], v[i + 1]), hi), lo), r2);
      unpack2(fma2(d, pack2(g[i], g[i + 1]), pack2(h[i], h[i + 1])), &v[i], &v[i + 1]);
    }
  }
  __device__ __forceinline__ double exact(int col) const {
    return (static_cast<double>(to_f32(x[col])) - mean) * rstd * static_cast<double>(w[col]) +
           static_cast<double>(b[col]);
  }
  __device__ __forceinline__ float error(float h) const { return 0x1p-21f * (h + top_b); }
};

// Group norm with its activation; mean and 1 / sqrt(var + eps) of the row's
// window come from tables indexed by group. The error bound adds the
// activation's: |act'| <= 1.1, and SiLU's own rounding.
struct GroupStat {
  double mean, rstd;
};
template <typename T, bool VEC>
struct GroupNormSource {
  static constexpr bool kExact = false, kLayerNorm = false;
  static constexpr int E = kChunk<T>;
  const T* x;
  const float* w;
  const float* b;
  const GroupStat* stat;  // [groups], shared memory
  const float4* fast;     // [groups], shared memory: mean's high and low part, 1 / deviation in fp32
  int group_width;
  float inv_width;        // 1 / group_width
  bool whole;             // a chunk lies within one group
  int epi;
  float top_b;  // max|b|
  // col / group_width for columns below 2^20: the quotient of col + 1/2 is at
  // least 1 / (2 group_width) from a whole number, more than the product's error
  __device__ __forceinline__ int group(int col) const {
    return static_cast<int>((static_cast<float>(col) + 0.5f) * inv_width);
  }
  __device__ __forceinline__ void raw(int c, float (&v)[E]) const { load_chunk<T, E>(x + c * E, VEC, v); }
  __device__ __forceinline__ void value(int c, float (&v)[E]) const {
    float g[E], h[E];
    load_params<E>(w + c * E, VEC, g);
    load_params<E>(b + c * E, VEC, h);
    if (whole) {
      const float4 f = fast[group(c * E)];
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = fmaf(((v[i] - f.x) - f.y) * f.z, g[i], h[i]);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float4 f = fast[group(c * E + i)];
        v[i] = fmaf(((v[i] - f.x) - f.y) * f.z, g[i], h[i]);
      }
    }
    if (epi == PQ8_EPI_SILU) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = act_f32(v[i], PQ8_EPI_SILU);
    } else if (epi == PQ8_EPI_RELU) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = act_f32(v[i], PQ8_EPI_RELU);
    }
  }
  __device__ __forceinline__ double exact(int col) const {
    const GroupStat s = stat[col / group_width];
    const double z = (static_cast<double>(to_f32(x[col])) - s.mean) * s.rstd * static_cast<double>(w[col]) +
                     static_cast<double>(b[col]);
    return act_f64(z, epi);
  }
  __device__ __forceinline__ float error(float h) const { return 0x1p-20f * (h + top_b + 1.0f); }
};

// ---------------------------------------------------------------------------
// One row, by a team of WARPS warps. CHUNKS > 0: each thread holds up to CHUNKS
// chunks of the row in registers (width <= CHUNKS * E * 32 * WARPS);
// CHUNKS == 0: any width, read again in each pass. FULL: the width is exactly
// that of CHUNKS chunks per thread, so that no chunk has to be checked for.
// `width` is a multiple of E; q is E-byte aligned. Every thread of the team
// returns the scale.
//
// Per value, the common path is a multiply-add that rounds (adding 1.5 x
// 2^23 leaves the nearest integer in the low bits), its remainder, and a
// running maximum of the remainders: a thread looks its values through for
// the ones next to a border only when that maximum says there is one.
template <int CHUNKS, int WARPS, bool FULL, typename Src>
__device__ __forceinline__ float quantize_row(Src src, int width, int8_t* q, const RowTeam<WARPS>& team) {
  constexpr int E = Src::E;
  constexpr int kThreads = WARPS * 32;
  constexpr bool kCached = CHUNKS > 0;
  constexpr int N = kCached ? CHUNKS : 1;
  const int tid = team.index(), chunks = FULL ? CHUNKS * kThreads : width / E;
  auto has = [&](int c) { return FULL || c < chunks; };
  static_assert(N * E <= 32, "a mask bit per value");
  float v[N][E];
  if constexpr (kCached) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = tid + j * kThreads;
      if (has(c)) src.raw(c, v[j]);
    }
  }
  // f(values, chunk) for every chunk of this thread; `compute`: from the raw
  // ones (rows that are not cached always start from those)
  auto each = [&](auto&& f, bool compute) {
    if constexpr (kCached) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = tid + j * kThreads;
        if (has(c)) {
          if (compute) src.value(c, v[j]);
          f(v[j], c);
        }
      }
    } else {
      for (int c = tid; c < chunks; c += kThreads) {
        src.raw(c, v[0]);
        src.value(c, v[0]);
        f(v[0], c);
      }
    }
  };
  // f(column) for the columns of this thread whose value `pick`s: those are
  // found in registers, then taken one at a time
  auto columns = [&](auto&& pick, auto&& f) {
    uint32_t found = 0;
    auto pick_chunk = [&](const float(&u)[E]) {
      uint32_t here = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) here |= pick(u[i]) ? 1u << i : 0u;
      return here;
    };
    if constexpr (kCached) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (has(tid + j * kThreads)) found |= pick_chunk(v[j]) << (j * E);
      for (; found; found &= found - 1) {
        const int bit = __ffs(found) - 1;
        f((tid + (bit / E) * kThreads) * E + bit % E);
      }
    } else {
#pragma unroll 1
      for (int c = tid; c < chunks; c += kThreads) {
        src.raw(c, v[0]);
        src.value(c, v[0]);
        for (found = pick_chunk(v[0]); found; found &= found - 1) f(c * E + __ffs(found) - 1);
      }
    }
  };
  if constexpr (Src::kLayerNorm) {
    const double first = static_cast<double>(to_f32(src.x[0]));
    double s = 0.0, sq = 0.0;
    if constexpr (kCached) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (has(tid + j * kThreads)) src.add(v[j], first, s, sq);
    } else {
      for (int c = tid; c < chunks; c += kThreads) {
        src.raw(c, v[0]);
        src.add(v[0], first, s, sq);
      }
    }
    src.finish(team, first, s, sq);
  }

  float mine = 0.0f, bad = 0.0f;
  float chunk_top[N];  // cached rows: the largest of each chunk
  each([&](const float(&u)[E], int c) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      m = fmaxf(m, fabsf(u[i]));
      bad = fmaf(u[i], 0.0f, bad);  // NaN from an infinity or a NaN on
    }
    mine = fmaxf(mine, m);
    if constexpr (kCached) chunk_top[(c - tid) / kThreads] = m;
  }, true);
  const float top = team.max(bad == 0.0f ? mine : INFINITY);
  float s = top / 127.0f;
  if constexpr (!Src::kExact) {
    if (top < INFINITY) {
      // the values that may be the largest, exactly (looked for only in chunks that
      // reach the bound; whole chunks in fp64 took 35 us for 24,000 x 1024 bf16)
      const float least = top - 2.5f * src.error(top);
      double t64 = 0.0;
      if (mine >= least) {
        if constexpr (kCached) {
          uint32_t found = 0;
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (has(tid + j * kThreads) && chunk_top[j] >= least) {
#pragma unroll
              for (int i = 0; i < E; ++i) found |= fabsf(v[j][i]) >= least ? 1u << (j * E + i) : 0u;
            }
          for (; found; found &= found - 1) {
            const int bit = __ffs(found) - 1;
            t64 = fmax(t64, ::fabs(src.exact((tid + (bit / E) * kThreads) * E + bit % E)));
          }
        } else {
          columns([&](float u) { return fabsf(u) >= least; },
                  [&](int col) { t64 = fmax(t64, ::fabs(src.exact(col))); });
        }
      }
      s = static_cast<float>(team.max(t64) * (1.0 / 127.0));
    }
  }
  if (!(top < INFINITY) || s == 0.0f) {
    // an infinity or a NaN in the row: no scale, no values; a row of zeros, or
    // of values too small for a scale: zeros
    for (int c = tid; c < chunks; c += kThreads)
#pragma unroll
      for (int i = 0; i < E; i += 4) *reinterpret_cast<uint32_t*>(q + c * E + i) = 0u;
    return top < INFINITY ? 0.0f : __int_as_float(0x7fc00000);
  }
  const float inv = __fdividef(1.0f, s);  // off by at most 2^-22: in `border`
  constexpr float kBig = 12582912.0f;
  // below this, 1 / s may leave fp32's range: every quotient in fp64
  const bool all = s < 0x1p-100f;
  // |remainder| from which a quotient may lie on the other side of a border:
  // the value's error, and that of the reciprocal and the product
  const float border = 0.5f - (128.0f * 0x1p-21f + src.error(top) * inv);
  float worst = 0.0f;
  each([&](const float(&u)[E], int c) {
    uint32_t m[E], word[E / 4];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float big = fmaf(u[i], inv, kBig);
      m[i] = __float_as_uint(big);
      worst = fmaxf(worst, fabsf(fmaf(u[i], inv, kBig - big)));  // what the rounding took off
    }
#pragma unroll
    for (int i = 0; i < E; i += 4)
      word[i >> 2] = __byte_perm(__byte_perm(m[i], m[i + 1], 0x0040), __byte_perm(m[i + 2], m[i + 3], 0x0040), 0x5410);
    if constexpr (E == 4) {
      *reinterpret_cast<uint32_t*>(q + c * E) = word[0];
    } else {
      *reinterpret_cast<uint2*>(q + c * E) = make_uint2(word[0], word[E / 4 - 1]);
    }
  }, false);
  if (worst >= border || all) {
    const double s64 = static_cast<double>(s);
    columns(
        [&](float u) {
          const float big = fmaf(u, inv, kBig);
          return all || fabsf(fmaf(u, inv, kBig - big)) >= border;
        },
        [&](int col) {
          q[col] = static_cast<int8_t>(static_cast<int>(fmin(fmax(rint(src.exact(col) / s64), -127.0), 127.0)));
        });
  }
  return s;
}

constexpr int kRowThreads = 256;

// Rows of a [rows, width] matrix (row stride ld elements), each quantised by
// a team of WARPS warps: a warp per row up to 1024 columns, the CTA's eight
// warps up to 8192 (the row stays in registers in both), and past that, or
// where 16-byte loads do not fit, the CTA reads the row again in each pass.
// NORM: LayerNorm first. Bound by HBM for fp32 rows as they are (24,000 x
// 1024: 19.5 us, 6.3 TB/s), by instruction issue otherwise: bf16 18 us (the same
// instructions over half the bytes), after a LayerNorm 30 us fp32, 29 us bf16 (fp64
// sums, and the long chain of reductions of a row, at 24 warps an SM).
template <typename T, int CHUNKS, int WARPS, bool FULL, bool NORM, bool VEC>
__global__ void __launch_bounds__(kRowThreads, NORM ? 3 : 4)
    quantize_rows_kernel(const T* __restrict__ x, long long ld, const float* __restrict__ w,
                         const float* __restrict__ b, double eps, int8_t* __restrict__ q, float* __restrict__ scale,
                         int rows, int width) {
  __shared__ double team_smem[2 * WARPS];
  __shared__ float top_smem[kRowThreads / 32];
  constexpr int kTeams = kRowThreads / (32 * WARPS);
  const RowTeam<WARPS> team{team_smem};
  griddep_wait();    // x is the previous kernel's output
  griddep_launch();  // only now: what the next kernel reads ahead of its own wait is then older than this kernel
  std::conditional_t<NORM, LayerNormSource<T, VEC>, PlainSource<T, VEC>> src;
  if constexpr (NORM) {
    src.w = w;
    src.b = b;
    src.eps = eps;
    src.inv_width = 1.0 / width;
    src.top_b = cta_max_abs(b, width, top_smem);
  }
  const int first = static_cast<int>(blockIdx.x) * kTeams + static_cast<int>(threadIdx.x) / (32 * WARPS);
  for (long long row = first; row < rows; row += static_cast<long long>(gridDim.x) * kTeams) {
    src.x = x + row * ld;
    const float s = quantize_row<CHUNKS, WARPS, FULL>(src, width, q + row * width, team);
    if (team.index() == 0) scale[row] = s;
  }
}

}  // namespace pq8
