// Group norm with an activation, channels last (pq8_group_norm,
// pq8_group_norm_quantize): rows of `channels` values, windows of consecutive
// rows; mean and variance over the rows of one window and the channels of one
// group,
//   y = act((x - mean) / sqrt(var + eps) * w + b).
// Sums are fp64, taken of x minus the group's first value of the window, so
// that neither a large common offset nor a long window costs digits; they are
// added in a fixed order.
//
// Two forms. Where a window's rows of a few groups fit the shared memory of a
// cluster, one launch reads x once: every CTA holds its rows there, the
// cluster's CTAs exchange their sums, and each normalises what it holds.
// Otherwise (long windows of wide groups, rows that 16-byte loads do not fit)
// partial sums go through a workspace and a second launch reads x again.
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
  int chunks;      // two launches: row chunks per window of the sums
  int slab;        // whole groups per CTA; their columns are whole units
  int hold;        // one launch: rows a CTA holds in shared memory
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

// The rows of part `c` of `parts` equal parts of [lo, hi).
__device__ __forceinline__ void part_rows(int lo, int hi, int c, int parts, int* r0, int* r1) {
  const int per = (hi - lo + parts - 1) / parts;
  *r0 = static_cast<int>(min(static_cast<long long>(lo) + static_cast<long long>(c) * per, static_cast<long long>(hi)));
  *r1 = min(*r0 + per, hi);
}

constexpr int kNormThreads = 256;

// How columns are taken: one at a time; 16-byte units that lie within one
// group; 16-byte units of which some straddle two groups (group width at
// least a unit).
enum NormUnits { kScalar = 0, kWhole = 1, kStraddle = 2 };

// A CTA's threads over the rows of a slab: thread (x, y) has unit x (and, in
// a slab of one group wider than the CTA, x + tx, ...) of rows y, y + ty, ...
template <int E>
struct SlabShape {
  int units, tx, ty, x, y;
  __device__ __forceinline__ explicit SlabShape(int cols) {
    units = cols / E;
    tx = min(units, kNormThreads);
    ty = kNormThreads / tx;
    x = static_cast<int>(threadIdx.x) % tx;
    y = static_cast<int>(threadIdx.x) / tx;
  }
};

struct GroupSum {
  double s, q;  // sums of x - first and its square
};
struct GroupSum2 {
  GroupSum a, b;  // of a unit's first group and of the next
};

// Where a unit lies: its first group (of the slab), and how many of its
// elements belong to it.
template <int UNITS, int E>
__device__ __forceinline__ void unit_group(int u, int cg, int* g, int* split) {
  *g = u * E / cg;
  *split = UNITS == kStraddle ? min((*g + 1) * cg - u * E, E) : E;
}

template <int UNITS, int E>
__device__ __forceinline__ void add_unit(GroupSum2& acc, const float (&v)[E], int split, double fa, double fb) {
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (UNITS != kStraddle || i < split) {
      const double d = static_cast<double>(v[i]) - fa;
      acc.a.s += d;
      acc.a.q += d * d;
    } else {
      const double d = static_cast<double>(v[i]) - fb;
      acc.b.s += d;
      acc.b.q += d * d;
    }
  }
}

// The threads' sums of the slab's ng groups to out[g], a warp per group, in a
// fixed order. All threads of the CTA; red: kNormThreads entries.
template <int UNITS, int E>
__device__ __forceinline__ void reduce_groups(const SlabShape<E>& sh, const GroupSum2& acc, int cg, int ng,
                                              GroupSum2* red, GroupSum* out) {
  __syncthreads();  // red has been read
  red[threadIdx.x] = acc;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int g = warp; g < ng; g += kNormThreads / 32) {
    // units with elements of group g (a slab of one group: every x)
    const int u0 = ng > 1 ? g * cg / E : 0, u1 = ng > 1 ? ((g + 1) * cg - 1) / E + 1 : sh.tx, nu = u1 - u0;
    double s = 0.0, q = 0.0;
    for (int i = lane; i < nu * sh.ty; i += 32) {
      const int u = u0 + i % nu;
      const GroupSum2& t = red[(i / nu) * sh.tx + u];
      const GroupSum& part = (UNITS == kStraddle && u * E / cg != g) ? t.b : t.a;
      s += part.s;
      q += part.q;
    }
    s = warp_sum_f64(s);
    q = warp_sum_f64(q);
    if (lane == 0) out[g] = GroupSum{s, q};
  }
}

__device__ __forceinline__ GroupStat group_stat(const GroupSum& t, double first, double n, double eps) {
  const double m = t.s / n;
  return GroupStat{first + m, 1.0 / sqrt(fmax(t.q / n - m * m, 0.0) + eps)};
}

// The first value of slab group g in the window (0 for an empty window).
template <typename T>
__device__ __forceinline__ double first_value(const GroupNormParams& p, int lo, int hi, int g0, int g, int cg) {
  if (lo >= hi) return 0.0;
  return static_cast<double>(
      to_f32(static_cast<const T*>(p.x)[static_cast<size_t>(lo) * p.channels + static_cast<size_t>(g0 + g) * cg]));
}

// Normalisation of one unit: mean and 1 / deviation in fp32 (the mean in two
// parts, so that x - mean is rounded relative to its own size), weight, bias.
template <int UNITS, int E>
struct UnitNorm {
  float hi_a, lo_a, rs_a, hi_b, lo_b, rs_b;  // of the unit's first group and of the next
  float g[E], h[E];
  int split;
  __device__ __forceinline__ UnitNorm(const GroupNormParams& p, const GroupStat* stat, int u, int cg, int ng, int col) {
    int first;
    unit_group<UNITS, E>(u, cg, &first, &split);
    set(stat[first], &hi_a, &lo_a, &rs_a);
    if constexpr (UNITS == kStraddle) set(stat[min(first + 1, ng - 1)], &hi_b, &lo_b, &rs_b);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      g[i] = p.w[col + i];
      h[i] = p.b[col + i];
    }
  }
  __device__ __forceinline__ static void set(const GroupStat& st, float* hi, float* lo, float* rs) {
    *hi = static_cast<float>(st.mean);
    *lo = static_cast<float>(st.mean - static_cast<double>(*hi));
    *rs = static_cast<float>(st.rstd);
  }
  __device__ __forceinline__ void apply(float (&v)[E], int epi, int round_out) const {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const bool next = UNITS == kStraddle && i >= split;
      v[i] = fmaf(((v[i] - (next ? hi_b : hi_a)) - (next ? lo_b : lo_a)) * (next ? rs_b : rs_a), g[i], h[i]);
    }
    if (epi == PQ8_EPI_SILU) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = act_f32(v[i], PQ8_EPI_SILU);
    } else if (epi == PQ8_EPI_RELU) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = act_f32(v[i], PQ8_EPI_RELU);
    }
    if (round_out) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = tf32_round(v[i]);
    }
  }
};

template <typename T, int UNITS>
constexpr int kUnit = UNITS == kScalar ? 1 : kChunk<T>;

template <typename T, int UNITS>
__device__ __forceinline__ void load_unit(const T* p, float (&v)[kUnit<T, UNITS>]) {
  if constexpr (UNITS == kScalar) v[0] = to_f32(p[0]);
  else load_chunk<T, kChunk<T>>(p, true, v);
}
template <typename T, int UNITS>
__device__ __forceinline__ void store_unit(T* p, const float (&v)[kUnit<T, UNITS>]) {
  if constexpr (UNITS == kScalar) p[0] = from_f32<T>(v[0]);
  else store_chunk<T, kChunk<T>>(p, true, v);
}

// ---------------------------------------------------------------------------
// One launch: cluster (window, slab), its CTAs the window's parts. Grid x: the
// cluster's CTAs, y: windows, z: slabs.
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ double ld_cluster_f64(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}

template <typename T, int UNITS>
__global__ void __launch_bounds__(kNormThreads)
    group_norm_kernel(const GroupNormParams p, T* __restrict__ y) {
  constexpr int E = kUnit<T, UNITS>;
  extern __shared__ uint4 held[];  // [rows][units]; then the slab's sums and statistics
  __shared__ GroupSum2 red[kNormThreads];
  const int cg = p.channels / p.groups, g0 = static_cast<int>(blockIdx.z) * p.slab, ng = min(p.slab, p.groups - g0);
  const SlabShape<E> sh(ng * cg);
  GroupSum* const sums = reinterpret_cast<GroupSum*>(held + static_cast<size_t>(p.hold) * (p.slab * cg / E));
  GroupStat* const stat = reinterpret_cast<GroupStat*>(sums + p.slab);
  const int parts = static_cast<int>(gridDim.x), part = static_cast<int>(blockIdx.x);
  griddep_wait();
  griddep_launch();
  int lo, hi, r0, r1;
  window_rows(p, blockIdx.y, &lo, &hi);
  part_rows(lo, hi, part, parts, &r0, &r1);
  const int held_end = min(r1, r0 + p.hold);
  const T* const x = static_cast<const T*>(p.x) + static_cast<size_t>(g0) * cg;
  const bool active = sh.y < sh.ty;
  // a thread reads back only what it has put there itself
  if (active) {
    for (int u = sh.x; u < sh.units; u += sh.tx)
      for (int r = r0 + sh.y; r < held_end; r += sh.ty)
        cp_async16(held + static_cast<size_t>(r - r0) * sh.units + u, x + static_cast<size_t>(r) * p.channels + u * E);
  }
  GroupSum2 acc{{0.0, 0.0}, {0.0, 0.0}};
  if (active) {
    for (int u = sh.x; u < sh.units; u += sh.tx) {
      int g, split;
      unit_group<UNITS, E>(u, cg, &g, &split);
      const double fa = first_value<T>(p, lo, hi, g0, g, cg);
      const double fb = UNITS == kStraddle && split < E ? first_value<T>(p, lo, hi, g0, g + 1, cg) : 0.0;
      float v[E];
      for (int r = held_end + sh.y; r < r1; r += sh.ty) {
        load_unit<T, UNITS>(x + static_cast<size_t>(r) * p.channels + u * E, v);
        add_unit<UNITS, E>(acc, v, split, fa, fb);
      }
      cp_async_wait_all();
#pragma unroll 4
      for (int r = r0 + sh.y; r < held_end; r += sh.ty) {
        load_unit<T, UNITS>(reinterpret_cast<const T*>(held + static_cast<size_t>(r - r0) * sh.units + u), v);
        add_unit<UNITS, E>(acc, v, split, fa, fb);
      }
    }
  }
  cp_async_wait_all();
  reduce_groups<UNITS, E>(sh, acc, cg, ng, red, sums);
  // every CTA adds the parts' sums in the same order
  if (parts > 1) cluster_sync();
  else __syncthreads();
  for (int g = threadIdx.x; g < ng; g += kNormThreads) {
    GroupSum t{0.0, 0.0};
    if (parts > 1) {
      for (int c = 0; c < parts; ++c) {
        const uint32_t at = map_to_rank(&sums[g], static_cast<uint32_t>(c));
        t.s += ld_cluster_f64(at);
        t.q += ld_cluster_f64(at + 8);
      }
    } else {
      t = sums[g];
    }
    stat[g] = group_stat(t, first_value<T>(p, lo, hi, g0, g, cg), static_cast<double>(max(hi - lo, 1)) * cg, p.eps);
  }
  __syncthreads();
  if (parts > 1) cluster_arrive_relaxed();  // this CTA has read the others' sums
  if (active) {
    for (int u = sh.x; u < sh.units; u += sh.tx) {
      const int col = g0 * cg + u * E;
      const UnitNorm<UNITS, E> norm(p, stat, u, cg, ng, col);
      T* const yu = y + col;
      float v[E];
#pragma unroll 2
      for (int r = r0 + sh.y; r < held_end; r += sh.ty) {
        load_unit<T, UNITS>(reinterpret_cast<const T*>(held + static_cast<size_t>(r - r0) * sh.units + u), v);
        norm.apply(v, p.epi, p.round_out);
        store_unit<T, UNITS>(yu + static_cast<size_t>(r) * p.channels, v);
      }
      for (int r = held_end + sh.y; r < r1; r += sh.ty) {
        load_unit<T, UNITS>(x + static_cast<size_t>(r) * p.channels + u * E, v);
        norm.apply(v, p.epi, p.round_out);
        store_unit<T, UNITS>(yu + static_cast<size_t>(r) * p.channels, v);
      }
    }
  }
  if (parts > 1) {
    __syncwarp();
    cluster_wait();  // nobody leaves while its sums may still be read
  }
}

// ---------------------------------------------------------------------------
// Two launches. Partial sums of one row chunk of one window for the groups of
// one slab: partial[window][chunk][group].
template <typename T, int UNITS>
__global__ void __launch_bounds__(kNormThreads)
    group_stats_kernel(const GroupNormParams p, GroupSum* __restrict__ partial) {
  constexpr int E = kUnit<T, UNITS>;
  __shared__ GroupSum2 red[kNormThreads];
  griddep_wait();
  griddep_launch();
  const int cg = p.channels / p.groups, g0 = static_cast<int>(blockIdx.z) * p.slab, ng = min(p.slab, p.groups - g0);
  const SlabShape<E> sh(ng * cg);
  const T* const x = static_cast<const T*>(p.x) + static_cast<size_t>(g0) * cg;
  for (int w = blockIdx.y; w < p.windows; w += gridDim.y) {
    int lo, hi, r0, r1;
    window_rows(p, w, &lo, &hi);
    part_rows(lo, hi, blockIdx.x, p.chunks, &r0, &r1);
    GroupSum2 acc{{0.0, 0.0}, {0.0, 0.0}};
    if (sh.y < sh.ty) {
      for (int u = sh.x; u < sh.units; u += sh.tx) {
        int g, split;
        unit_group<UNITS, E>(u, cg, &g, &split);
        const double fa = first_value<T>(p, lo, hi, g0, g, cg);
        const double fb = UNITS == kStraddle && split < E ? first_value<T>(p, lo, hi, g0, g + 1, cg) : 0.0;
        const T* const xu = x + u * E;
        constexpr int kAhead = 4;  // rows whose loads are issued together
        int r = r0 + sh.y;
        for (; r + (kAhead - 1) * sh.ty < r1; r += kAhead * sh.ty) {
          float v[kAhead][E];
#pragma unroll
          for (int k = 0; k < kAhead; ++k)
            load_unit<T, UNITS>(xu + static_cast<size_t>(r + k * sh.ty) * p.channels, v[k]);
#pragma unroll
          for (int k = 0; k < kAhead; ++k) add_unit<UNITS, E>(acc, v[k], split, fa, fb);
        }
        for (; r < r1; r += sh.ty) {
          float v[E];
          load_unit<T, UNITS>(xu + static_cast<size_t>(r) * p.channels, v);
          add_unit<UNITS, E>(acc, v, split, fa, fb);
        }
      }
    }
    reduce_groups<UNITS, E>(sh, acc, cg, ng, red,
                            partial + (static_cast<size_t>(w) * p.chunks + blockIdx.x) * p.groups + g0);
  }
}

// Statistics of groups [g0, g0 + ng) of a window, from its chunks' sums added
// in chunk order, into `stat` (shared memory). All threads.
template <typename T>
__device__ __forceinline__ void group_finish(const GroupNormParams& p, const GroupSum* partial, int w, int lo, int hi,
                                             int g0, int ng, GroupStat* stat) {
  const int cg = p.channels / p.groups;
  __syncthreads();  // stat has been read (previous window)
  for (int g = threadIdx.x; g < ng; g += blockDim.x) {
    GroupSum t{0.0, 0.0};
    const GroupSum* at = partial + static_cast<size_t>(w) * p.chunks * p.groups + g0 + g;
#pragma unroll 4
    for (int c = 0; c < p.chunks; ++c) {
      const GroupSum part = at[static_cast<size_t>(c) * p.groups];
      t.s += part.s;
      t.q += part.q;
    }
    stat[g] = group_stat(t, first_value<T>(p, lo, hi, g0, g, cg), static_cast<double>(max(hi - lo, 1)) * cg, p.eps);
  }
  __syncthreads();
}

// Normalise and activate the rows of one part of one window, one slab.
template <typename T, int UNITS>
__global__ void __launch_bounds__(kNormThreads)
    group_apply_kernel(const GroupNormParams p, const GroupSum* __restrict__ partial, T* __restrict__ y) {
  constexpr int E = kUnit<T, UNITS>;
  extern __shared__ GroupStat stat[];
  griddep_wait();
  griddep_launch();
  const int cg = p.channels / p.groups, g0 = static_cast<int>(blockIdx.z) * p.slab, ng = min(p.slab, p.groups - g0);
  const SlabShape<E> sh(ng * cg);
  for (int w = blockIdx.y; w < p.windows; w += gridDim.y) {
    int lo, hi, r0, r1;
    window_rows(p, w, &lo, &hi);
    part_rows(lo, hi, blockIdx.x, gridDim.x, &r0, &r1);
    group_finish<T>(p, partial, w, lo, hi, g0, ng, stat);
    if (sh.y >= sh.ty) continue;
    for (int u = sh.x; u < sh.units; u += sh.tx) {
      const int col = g0 * cg + u * E;
      const UnitNorm<UNITS, E> norm(p, stat, u, cg, ng, col);
      const T* const xu = static_cast<const T*>(p.x) + col;
      T* const yu = y + col;
      constexpr int kAhead = 4;
      int r = r0 + sh.y;
      for (; r + (kAhead - 1) * sh.ty < r1; r += kAhead * sh.ty) {
        float v[kAhead][E];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          load_unit<T, UNITS>(xu + static_cast<size_t>(r + k * sh.ty) * p.channels, v[k]);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          norm.apply(v[k], p.epi, p.round_out);
          store_unit<T, UNITS>(yu + static_cast<size_t>(r + k * sh.ty) * p.channels, v[k]);
        }
      }
      for (; r < r1; r += sh.ty) {
        float v[E];
        load_unit<T, UNITS>(xu + static_cast<size_t>(r) * p.channels, v);
        norm.apply(v, p.epi, p.round_out);
        store_unit<T, UNITS>(yu + static_cast<size_t>(r) * p.channels, v);
      }
    }
  }
}

// Normalise, activate and quantise the rows of one part of one window: rows
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
    part_rows(lo, hi, blockIdx.x, gridDim.x, &r0, &r1);
    if (r0 >= r1) continue;  // the whole CTA
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
