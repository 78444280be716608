// Group norm with an activation, channels last (pq8_group_norm,
// pq8_group_norm_quantize): rows of `channels` values, windows of consecutive
// rows; mean and variance over the rows of one window and the channels of one
// group,
//   y = act((x - mean) / sqrt(var + eps) * w + b).
// Sums are taken of x minus a nearby value, so that neither a large common
// offset nor a long window costs digits, and added in a fixed order: per
// column over at most 32 rows of a thread in fp32 (minus the first of them;
// two columns per instruction, no conversions), everything above in fp64
// (minus the group's first value of the window). Where the result is
// quantised every value goes to fp64 at once: integers next to a border need
// the statistics to more digits.
//
// Two forms of each. Where a window's rows of a few groups fit the shared memory of a
// cluster, one launch reads x once: every CTA holds its rows there, the
// cluster's CTAs exchange their sums, and each normalises what it holds.
// Otherwise (long windows of wide groups, rows that 16-byte loads do not fit)
// partial sums go through a workspace and a second launch reads x again.
//
// Measured (bytes of x and y over the time): 8 x 375 x 1024 fp32, 32 groups,
// one launch 8.6 to 10 us (2.5 TB/s: one wave of CTAs that load, sum, meet and store in
// turn, 14,000 cycles), 64 windows 45.9 us (4.3 TB/s); 64 x 375 x 1024 bf16 in one
// group 37.3 us (2.6 TB/s). There two CTAs an SM took 34,000 cycles a wave when it was
// 39.6 us: 11,000 to load, 4000 to sum, 3000 to exchange, 14,000 to normalise and store (8000
// without SiLU: the special-function unit). 13 ragged windows of 7969 x 1000 fp16
// in two launches 23.5 us. Quantised, 8 x 375 x 1024: 18 us, of which the second launch 8.
// With SiLU of values below -43 (weights of 60, say) those rows are normalised twice: 46 -> 66 us.
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
  int block;       // two launches: rows a CTA of the sums takes, whatever windows they belong to
  int row_block;   // two launches: the same in the second launch
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

// A thread's sums of one unit's columns over its rows, into acc by flush().
// EXACT: every value in fp64 at once.
template <int UNITS, int E, bool EXACT>
struct UnitSum {
  static constexpr int kRun = 32;  // rows in fp32
  static constexpr int H = E > 1 ? E / 2 : 1;
  int split, run = 0;
  double fa, fb;  // first values of the unit's first group and of the next
  f32x2 minus[H], s[H], q[H];  // minus the run's first row; sums of the differences and of their squares
  __device__ __forceinline__ UnitSum(int split_, double fa_, double fb_) : split(split_), fa(fa_), fb(fb_) {}
  __device__ __forceinline__ void add(GroupSum2& acc, const float (&v)[E]) {
    if constexpr (EXACT) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const bool next = UNITS == kStraddle && i >= split;
        const double d = static_cast<double>(v[i]) - (next ? fb : fa);
        if (next) {
          acc.b.s += d;
          acc.b.q += d * d;
        } else {
          acc.a.s += d;
          acc.a.q += d * d;
        }
      }
    } else {
      if (run == 0) {
#pragma unroll
        for (int i = 0; i < H; ++i) {
          minus[i] = pack2(-v[2 * i], E > 1 ? -v[2 * i + (E > 1)] : 0.0f);
          s[i] = q[i] = 0;
        }
      }
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const f32x2 d = add2(pack2(v[2 * i], E > 1 ? v[2 * i + (E > 1)] : 0.0f), minus[i]);
        s[i] = add2(s[i], d);
        q[i] = fma2(d, d, q[i]);
      }
      if (++run == kRun) flush(acc);
    }
  }
  __device__ __forceinline__ void flush(GroupSum2& acc) {
    if constexpr (!EXACT) {
      if (run == 0) return;
      const double n = run;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        float m[2], ss[2], qq[2];
        unpack2(minus[i / 2], &m[0], &m[1]);
        unpack2(s[i / 2], &ss[0], &ss[1]);
        unpack2(q[i / 2], &qq[0], &qq[1]);
        const bool next = UNITS == kStraddle && i >= split;
        // off: the run's reference value minus the group's
        const double off = -static_cast<double>(m[i % 2]) - (next ? fb : fa), sd = static_cast<double>(ss[i % 2]);
        const double ds = sd + n * off, dq = static_cast<double>(qq[i % 2]) + off * (2.0 * sd + n * off);
        if (next) {
          acc.b.s += ds;
          acc.b.q += dq;
        } else {
          acc.a.s += ds;
          acc.a.q += dq;
        }
      }
      run = 0;
    }
  }
};

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

// Squares that left fp32's range (possible where values are over 2^60 apart) leave no statistics: NaN.
__device__ __forceinline__ GroupStat group_stat(const GroupSum& t, double first, double n, double eps) {
  const double m = t.s / n;
  return GroupStat{first + m, t.q < INFINITY ? 1.0 / sqrt(fmax(t.q / n - m * m, 0.0) + eps) : NAN};
}

// The first value of slab group g in the window (0 for an empty window).
template <typename T>
__device__ __forceinline__ double first_value(const GroupNormParams& p, int lo, int hi, int g0, int g, int cg) {
  if (lo >= hi) return 0.0;
  return static_cast<double>(
      to_f32(static_cast<const T*>(p.x)[static_cast<size_t>(lo) * p.channels + static_cast<size_t>(g0 + g) * cg]));
}

// Normalisation of one unit's columns: y = act((x - hi) a + c) with hi the mean
// rounded to fp32 (x - hi is rounded relative to its own size, whatever the
// mean), a = w / deviation, and c = b minus what is left of the mean.
template <int UNITS, int E>
struct UnitNorm {
  float hi_a, hi_b;  // of the unit's first group and of the next
  float a[E], c[E];
  int split;
  __device__ __forceinline__ UnitNorm(const GroupNormParams& p, const GroupStat* stat, int u, int cg, int ng, int col) {
    int first;
    unit_group<UNITS, E>(u, cg, &first, &split);
    const GroupStat sa = stat[first], sb = UNITS == kStraddle ? stat[min(first + 1, ng - 1)] : sa;
    hi_a = static_cast<float>(sa.mean);
    hi_b = static_cast<float>(sb.mean);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const bool next = UNITS == kStraddle && i >= split;
      const double rest = next ? sb.mean - static_cast<double>(hi_b) : sa.mean - static_cast<double>(hi_a);
      const double scale = (next ? sb.rstd : sa.rstd) * static_cast<double>(p.w[col + i]);
      a[i] = static_cast<float>(scale);
      c[i] = static_cast<float>(static_cast<double>(p.b[col + i]) - rest * scale);
    }
  }
  // `least`: of all values before a SiLU so far; APART: with sigmoid2_apart.
  template <bool APART = false>
  __device__ __forceinline__ void apply(float (&v)[E], int epi, int round_out, float& least) const {
    if constexpr (E == 1) {
      v[0] = fmaf(v[0] - hi_a, a[0], c[0]);
      if (epi == PQ8_EPI_SILU) v[0] = act_f32(v[0], PQ8_EPI_SILU);
    } else {
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const f32x2 hi = pack2(-(UNITS == kStraddle && i >= split ? hi_b : hi_a),
                               -(UNITS == kStraddle && i + 1 >= split ? hi_b : hi_a));
        f32x2 z = fma2(add2(pack2(v[i], v[i + 1]), hi), pack2(a[i], a[i + 1]), pack2(c[i], c[i + 1]));
        if (epi == PQ8_EPI_SILU) {
          if constexpr (!APART) take_least(z, least);
          z = mul2(z, sigmoid2<APART>(z));
        }
        unpack2(z, &v[i], &v[i + 1]);
      }
    }
    if (epi == PQ8_EPI_RELU) {
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
// E values of a unit, rounded to T once.
template <typename T, int E>
__device__ __forceinline__ void store_values(T* p, const float (&v)[E]) {
  constexpr int C = kChunk<T>;
  if constexpr (E == 1) {
    p[0] = from_f32<T>(v[0]);
  } else {
#pragma unroll
    for (int i = 0; i < E; i += C) {
      float u[C];
#pragma unroll
      for (int j = 0; j < C; ++j) u[j] = v[i + j];
      store_chunk<T, C>(p + i, true, u);
    }
  }
}

// Rows r0, r0 + step, ... below r1 of one unit once more, where a sigmoid was out of the fast form's range.
template <typename T, int UNITS, typename Out>
__device__ __forceinline__ void norm_rows_apart(const GroupNormParams& p, const UnitNorm<UNITS, kUnit<T, UNITS>>& norm,
                                                const T* xu, Out* yu, int r0, int r1, int step, float least) {
  if (least >= kSigmoidLeast) return;
#pragma unroll 1
  for (int r = r0; r < r1; r += step) {
    float v[kUnit<T, UNITS>];
    load_unit<T, UNITS>(xu + static_cast<size_t>(r) * p.channels, v);
    norm.template apply<true>(v, p.epi, p.round_out, least);
    store_values(yu + static_cast<size_t>(r) * p.channels, v);
  }
}

// ---------------------------------------------------------------------------
// One launch: cluster (window, slab), its CTAs the window's parts. Grid x: the
// cluster's CTAs, y: windows, z: slabs.
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ double ld_cluster_f64(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}

// QUANT: the first half of the quantised form. Its rows need every channel for
// their scale, which no CTA here has: the values go to a workspace in fp32, with
// the statistics for the ones next to a border (group_rows_kernel).
struct GroupNormExtra {
  GroupStat* stat;  // [windows][groups]
  float* top_b;     // max|b|
};
template <typename T, int UNITS, bool QUANT>
__global__ void __launch_bounds__(kNormThreads)
    group_norm_kernel(const GroupNormParams p, std::conditional_t<QUANT, float, T>* __restrict__ y,
                      const GroupNormExtra extra) {
  using Out = std::conditional_t<QUANT, float, T>;
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
  // A thread reads back only what it has put there itself, so no barrier. Its
  // rows arrive in four groups; the sums of one are taken while the next are
  // under way.
  const int mine = active && held_end > r0 + sh.y ? (held_end - r0 - sh.y + sh.ty - 1) / sh.ty : 0;
  const int quarter = (mine + 3) / 4;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    for (int i = k * quarter; i < min(mine, (k + 1) * quarter); ++i) {
      const int r = r0 + sh.y + i * sh.ty;
      for (int u = sh.x; u < sh.units; u += sh.tx)
        cp_async16(held + static_cast<size_t>(r - r0) * sh.units + u, x + static_cast<size_t>(r) * p.channels + u * E);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  GroupSum2 acc{{0.0, 0.0}, {0.0, 0.0}};
  int g, split;
  unit_group<UNITS, E>(min(sh.x, sh.units - 1), cg, &g, &split);  // the same for all of a thread's units
  UnitSum<UNITS, E, QUANT> sum(split, first_value<T>(p, lo, hi, g0, g, cg),
                               UNITS == kStraddle && split < E ? first_value<T>(p, lo, hi, g0, g + 1, cg) : 0.0);
  if (sh.units <= sh.tx) {  // one unit per thread
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k == 0) asm volatile("cp.async.wait_group 3;" ::: "memory");
      else if (k == 1) asm volatile("cp.async.wait_group 2;" ::: "memory");
      else if (k == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
      else asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll 2
      for (int i = k * quarter; i < min(mine, (k + 1) * quarter); ++i) {
        float v[E];
        load_unit<T, UNITS>(reinterpret_cast<const T*>(held + static_cast<size_t>(sh.y + i * sh.ty) * sh.units + sh.x), v);
        sum.add(acc, v);
      }
    }
    if (active)
      for (int r = held_end + sh.y; r < r1; r += sh.ty) {
        float v[E];
        load_unit<T, UNITS>(x + static_cast<size_t>(r) * p.channels + sh.x * E, v);
        sum.add(acc, v);
      }
  } else {  // a group wider than the CTA: unit by unit, so that a run has the rows of one column
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll 1
    for (int u = sh.x; u < sh.units; u += sh.tx) {
      sum.flush(acc);
#pragma unroll 1
      for (int r = r0 + sh.y; r < r1; r += sh.ty) {
        float v[E];
        load_unit<T, UNITS>(r < held_end ? reinterpret_cast<const T*>(held + static_cast<size_t>(r - r0) * sh.units + u)
                                         : x + static_cast<size_t>(r) * p.channels + u * E, v);
        sum.add(acc, v);
      }
    }
  }
  sum.flush(acc);
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
    if (QUANT && part == 0) extra.stat[static_cast<size_t>(blockIdx.y) * p.groups + g0 + g] = stat[g];
  }
  if (QUANT && part == 0 && blockIdx.y == 0 && blockIdx.z == 0) {
    __shared__ float warp_top[kNormThreads / 32];
    const float top = cta_max_abs(p.b, p.channels, warp_top);
    if (threadIdx.x == 0) *extra.top_b = top;
  }
  __syncthreads();
  if (parts > 1) cluster_arrive_relaxed();  // this CTA has read the others' sums
  if (active) {
    for (int u = sh.x; u < sh.units; u += sh.tx) {
      const int col = g0 * cg + u * E;
      const UnitNorm<UNITS, E> norm(p, stat, u, cg, ng, col);
      Out* const yu = y + col;
      float v[E], least = 0.0f;
#pragma unroll 2
      for (int r = r0 + sh.y; r < held_end; r += sh.ty) {
        load_unit<T, UNITS>(reinterpret_cast<const T*>(held + static_cast<size_t>(r - r0) * sh.units + u), v);
        norm.apply(v, p.epi, p.round_out, least);
        store_values(yu + static_cast<size_t>(r) * p.channels, v);
      }
      for (int r = held_end + sh.y; r < r1; r += sh.ty) {
        load_unit<T, UNITS>(x + static_cast<size_t>(r) * p.channels + u * E, v);
        norm.apply(v, p.epi, p.round_out, least);
        store_values(yu + static_cast<size_t>(r) * p.channels, v);
      }
      norm_rows_apart<T, UNITS>(p, norm, x + u * E, yu, r0 + sh.y, r1, sh.ty, least);
    }
  }
  if (parts > 1) {
    __syncwarp();
    cluster_wait();  // nobody leaves while its sums may still be read
  }
}

// ---------------------------------------------------------------------------
// Two launches. CTAs take blocks of rows of the whole buffer, so that windows
// of any lengths keep them equally busy; a block's rows are worked through
// window by window. The sums of block b and window w go to partial[b + w]
// (blocks and windows both follow the rows, so no two pairs meet there).

// The first window from w on that ends after row r, or p.windows: a search in which
// every thread of the CTA looks at one window (up to 256 windows in one step, 2^24 in
// three). Every thread takes part.
__device__ __forceinline__ int window_after(const GroupNormParams& p, int w, int r) {
  int n = p.windows - w;  // it is one of [w, w + n]
  while (n > 0) {
    const int step = (n + kNormThreads - 1) / kNormThreads;
    const int i = w + (static_cast<int>(threadIdx.x) + 1) * step - 1;
    const int before = step * __syncthreads_count(i < w + n && p.offsets[i + 1] <= r);
    w += before;
    n = min(step - 1, n - before);
  }
  return w;
}

// f(window, its rows [lo, hi), those within [b0, b1)) for the windows with
// rows in [b0, b1). Every thread of the CTA takes part. Windows of no rows are passed over by
// search, as there may be millions of them.
template <typename F>
__device__ __forceinline__ void block_windows(const GroupNormParams& p, int b0, int b1, F&& f) {
  static_assert(kNormThreads == kRowThreads, "both kinds of kernel search with all their threads");
  int w = p.offsets == nullptr ? b0 / (p.rows / p.windows) : 0;
  bool search = p.offsets != nullptr;
  for (int after = b0;; ++w) {
    if (search) w = window_after(p, w, after);
    if (w >= p.windows) break;
    int lo, hi;
    window_rows(p, w, &lo, &hi);
    if (lo >= b1) break;
    const int r0 = max(lo, b0), r1 = min(hi, b1);
    search = r0 >= r1;
    after = r0;
    if (!search) f(w, lo, hi, r0, r1);
  }
}

// Sums of one block of rows for the groups of one slab.
template <typename T, int UNITS, bool EXACT>
__global__ void __launch_bounds__(kNormThreads)
    group_stats_kernel(const GroupNormParams p, GroupSum* __restrict__ partial, float* __restrict__ top_b) {
  constexpr int E = kUnit<T, UNITS>;
  __shared__ GroupSum2 red[kNormThreads];
  griddep_wait();
  griddep_launch();
  if (EXACT && blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) {  // max|b|, for the quantisation's error bound
    __shared__ float warp_top[kNormThreads / 32];
    const float top = cta_max_abs(p.b, p.channels, warp_top);
    if (threadIdx.x == 0) *top_b = top;
  }
  const int cg = p.channels / p.groups, g0 = static_cast<int>(blockIdx.y) * p.slab, ng = min(p.slab, p.groups - g0);
  const SlabShape<E> sh(ng * cg);
  const T* const x = static_cast<const T*>(p.x) + static_cast<size_t>(g0) * cg;
  const int b0 = static_cast<int>(blockIdx.x) * p.block;
  const int b1 = static_cast<int>(min(static_cast<long long>(b0) + p.block, static_cast<long long>(p.rows)));
  block_windows(p, b0, b1, [&](int w, int lo, int hi, int r0, int r1) {
    GroupSum2 acc{{0.0, 0.0}, {0.0, 0.0}};
    if (sh.y < sh.ty) {
      for (int u = sh.x; u < sh.units; u += sh.tx) {
        int g, split;
        unit_group<UNITS, E>(u, cg, &g, &split);
        UnitSum<UNITS, E, EXACT> sum(
            split, first_value<T>(p, lo, hi, g0, g, cg),
            UNITS == kStraddle && split < E ? first_value<T>(p, lo, hi, g0, g + 1, cg) : 0.0);
        const T* const xu = x + u * E;
        constexpr int kAhead = 4;  // rows whose loads are issued together
        int r = r0 + sh.y;
        for (; r + (kAhead - 1) * sh.ty < r1; r += kAhead * sh.ty) {
          float v[kAhead][E];
#pragma unroll
          for (int k = 0; k < kAhead; ++k)
            load_unit<T, UNITS>(xu + static_cast<size_t>(r + k * sh.ty) * p.channels, v[k]);
#pragma unroll
          for (int k = 0; k < kAhead; ++k) sum.add(acc, v[k]);
        }
        for (; r < r1; r += sh.ty) {
          float v[E];
          load_unit<T, UNITS>(xu + static_cast<size_t>(r) * p.channels, v);
          sum.add(acc, v);
        }
        sum.flush(acc);
      }
    }
    reduce_groups<UNITS, E>(sh, acc, cg, ng, red, partial + (static_cast<size_t>(blockIdx.x) + w) * p.groups + g0);
  });
}

// Statistics of groups [g0, g0 + ng) of window w, from its blocks' sums added
// in a fixed order, into `stat` (shared memory). All threads.
template <typename T>
__device__ __forceinline__ void group_finish(const GroupNormParams& p, const GroupSum* partial, int w, int lo, int hi,
                                             int g0, int ng, GroupStat* stat) {
  const int cg = p.channels / p.groups, first_block = lo / p.block, blocks = (hi - 1) / p.block - first_block + 1;
  const int lane = threadIdx.x & 31;
  const GroupSum* at = partial + (static_cast<size_t>(first_block) + w) * p.groups + g0;
  __syncthreads();  // stat has been read (previous window)
  // a warp per group, its lanes every 32nd block; or, for a few blocks, a thread per group
  if (blocks <= 8) {
    for (int g = threadIdx.x; g < ng; g += blockDim.x) {
      GroupSum t{0.0, 0.0};
      for (int c = 0; c < blocks; ++c) {
        const GroupSum part = at[static_cast<size_t>(c) * p.groups + g];
        t.s += part.s;
        t.q += part.q;
      }
      stat[g] = group_stat(t, first_value<T>(p, lo, hi, g0, g, cg), static_cast<double>(hi - lo) * cg, p.eps);
    }
  } else {
    for (int g = threadIdx.x >> 5; g < ng; g += blockDim.x >> 5) {
      const double first = first_value<T>(p, lo, hi, g0, g, cg);
      GroupSum t{0.0, 0.0};
      for (int c = lane; c < blocks; c += 32) {
        const GroupSum part = at[static_cast<size_t>(c) * p.groups + g];
        t.s += part.s;
        t.q += part.q;
      }
      t.s = warp_sum_f64(t.s);
      t.q = warp_sum_f64(t.q);
      if (lane == 0) stat[g] = group_stat(t, first, static_cast<double>(hi - lo) * cg, p.eps);
    }
  }
  __syncthreads();
}

// Normalise and activate one block of rows, one slab.
template <typename T, int UNITS>
__global__ void __launch_bounds__(kNormThreads)
    group_apply_kernel(const GroupNormParams p, const GroupSum* __restrict__ partial, T* __restrict__ y) {
  constexpr int E = kUnit<T, UNITS>;
  extern __shared__ GroupStat stat[];
  griddep_wait();
  griddep_launch();
  const int cg = p.channels / p.groups, g0 = static_cast<int>(blockIdx.y) * p.slab, ng = min(p.slab, p.groups - g0);
  const SlabShape<E> sh(ng * cg);
  const int b0 = static_cast<int>(blockIdx.x) * p.row_block;
  const int b1 = static_cast<int>(min(static_cast<long long>(b0) + p.row_block, static_cast<long long>(p.rows)));
  block_windows(p, b0, b1, [&](int w, int lo, int hi, int r0, int r1) {
    group_finish<T>(p, partial, w, lo, hi, g0, ng, stat);
    if (sh.y < sh.ty) {
      for (int u = sh.x; u < sh.units; u += sh.tx) {
        const int col = g0 * cg + u * E;
        const UnitNorm<UNITS, E> norm(p, stat, u, cg, ng, col);
        const T* const xu = static_cast<const T*>(p.x) + col;
        T* const yu = y + col;
        constexpr int kAhead = 4;
        int r = r0 + sh.y;
        float least = 0.0f;
        for (; r + (kAhead - 1) * sh.ty < r1; r += kAhead * sh.ty) {
          float v[kAhead][E];
#pragma unroll
          for (int k = 0; k < kAhead; ++k)
            load_unit<T, UNITS>(xu + static_cast<size_t>(r + k * sh.ty) * p.channels, v[k]);
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            norm.apply(v[k], p.epi, p.round_out, least);
            store_values(yu + static_cast<size_t>(r + k * sh.ty) * p.channels, v[k]);
          }
        }
        for (; r < r1; r += sh.ty) {
          float v[E];
          load_unit<T, UNITS>(xu + static_cast<size_t>(r) * p.channels, v);
          norm.apply(v, p.epi, p.round_out, least);
          store_values(yu + static_cast<size_t>(r) * p.channels, v);
        }
        norm_rows_apart<T, UNITS>(p, norm, xu, yu, r0 + sh.y, r1, sh.ty, least);
      }
    }
  });
}

// A row of no window, for a team of THREADS threads: integers and scale 0, so
// that a product that follows adds nothing there.
template <int THREADS>
__device__ __forceinline__ void zero_row(const GroupNormParams& p, int row, int8_t* q, float* scale, int index) {
  uint4* const at = reinterpret_cast<uint4*>(q + static_cast<size_t>(row) * p.channels);
  for (int c = index; c < p.channels / 16; c += THREADS) at[c] = make_uint4(0, 0, 0, 0);
  if (index == 0) scale[row] = 0.0f;
}

// Normalise, activate and quantise one block of rows: rows whole, as their
// scale needs every channel.
template <typename T, int CHUNKS, int WARPS, bool VEC>
__global__ void __launch_bounds__(kRowThreads, 2)
    group_quantize_kernel(const GroupNormParams p, const GroupSum* __restrict__ partial,
                          const float* __restrict__ top_b, int8_t* __restrict__ q, float* __restrict__ scale) {
  extern __shared__ GroupStat stat[];  // [groups], then their fp32 form
  float4* const fast = reinterpret_cast<float4*>(stat + p.groups);
  __shared__ double team_smem[2 * WARPS];
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
  src.inv_width = 1.0f / src.group_width;
  src.epi = p.epi;
  src.top_b = __ldg(top_b);
  const int b0 = static_cast<int>(blockIdx.x) * p.row_block;
  const int b1 = static_cast<int>(min(static_cast<long long>(b0) + p.row_block, static_cast<long long>(p.rows)));
  if constexpr (WARPS == 1) {  // this warp's first row on its way to L1 while the statistics are put together
    const int r = b0 + (static_cast<int>(threadIdx.x) >> 5);
    const T* const x = static_cast<const T*>(p.x) + static_cast<size_t>(r) * p.channels;
    if (r < b1)
      for (int c = (threadIdx.x & 31) * 128 / static_cast<int>(sizeof(T)); c < p.channels; c += 32 * 128 / static_cast<int>(sizeof(T)))
        asm volatile("prefetch.global.L1 [%0];" ::"l"(x + c));
  }
  const int my_team = static_cast<int>(threadIdx.x) / (32 * WARPS);
  int done = b0;  // the block's rows that are written, or in a window
  auto zero_up_to = [&](int end) {
    for (int r = done + my_team; r < end; r += kTeams) zero_row<32 * WARPS>(p, r, q, scale, team.index());
    done = max(done, end);
  };
  block_windows(p, b0, b1, [&](int w, int lo, int hi, int r0, int r1) {
    zero_up_to(r0);
    done = max(done, r1);
    group_finish<T>(p, partial, w, lo, hi, 0, p.groups, stat);
    for (int g = threadIdx.x; g < p.groups; g += blockDim.x) {
      const float m = static_cast<float>(stat[g].mean);
      fast[g] = make_float4(m, static_cast<float>(stat[g].mean - static_cast<double>(m)),
                            static_cast<float>(stat[g].rstd), 0.0f);
    }
    __syncthreads();
    for (int r = r0 + my_team; r < r1; r += kTeams) {
      src.x = static_cast<const T*>(p.x) + static_cast<size_t>(r) * p.channels;
      const float s = quantize_row<CHUNKS, WARPS, false>(src, p.channels, q + static_cast<size_t>(r) * p.channels, team);
      if (team.index() == 0) scale[r] = s;
    }
  });
  zero_up_to(b1);
}

// The second half of the quantised form where the first was one launch: rows of
// normalised fp32 values (error within error()) to integers; exact values
// from x and the statistics.
template <typename T>
struct NormedSource {
  static constexpr bool kExact = false, kLayerNorm = false;
  static constexpr int E = 4;
  const float* y;
  const T* x;
  const float* w;
  const float* b;
  const GroupStat* stat;  // of the row's window
  float inv_width;        // groups / channels
  int epi;
  float top_b;
  __device__ __forceinline__ void raw(int c, float (&v)[E]) const { load_chunk<float, E>(y + c * E, true, v); }
  __device__ __forceinline__ void value(int, float (&)[E]) const {}
  __device__ __forceinline__ double exact(int col) const {
    const GroupStat s = stat[static_cast<int>((static_cast<float>(col) + 0.5f) * inv_width)];
    const double z = (static_cast<double>(to_f32(x[col])) - s.mean) * s.rstd * static_cast<double>(w[col]) +
                     static_cast<double>(b[col]);
    return act_f64(z, epi);
  }
  __device__ __forceinline__ float error(float h) const { return 0x1p-20f * (h + top_b + 1.0f); }
};

// Window of row r, or -1.
__device__ __forceinline__ int row_window(const GroupNormParams& p, int r) {
  if (p.offsets == nullptr) return r / (p.rows / p.windows);
  int a = 0, b = p.windows;  // the first window that ends after r is in [a, b]
  while (a < b) {
    const int mid = (a + b) >> 1;
    if (__ldg(p.offsets + mid + 1) <= r) a = mid + 1;
    else b = mid;
  }
  return a < p.windows && __ldg(p.offsets + a) <= r ? a : -1;
}

template <typename T, int CHUNKS, int WARPS, bool FULL>
__global__ void __launch_bounds__(kRowThreads, 3)
    group_rows_kernel(const GroupNormParams p, const float* __restrict__ y, const GroupNormExtra extra,
                      int8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ double team_smem[2 * WARPS];
  constexpr int kTeams = kRowThreads / (32 * WARPS);
  const RowTeam<WARPS> team{team_smem};
  griddep_wait();
  griddep_launch();
  NormedSource<T> src;
  src.w = p.w;
  src.b = p.b;
  src.inv_width = 1.0f / static_cast<float>(p.channels / p.groups);
  src.epi = p.epi;
  src.top_b = __ldg(extra.top_b);
  const int first = static_cast<int>(blockIdx.x) * kTeams + static_cast<int>(threadIdx.x) / (32 * WARPS);
  for (int row = first; row < p.rows; row += static_cast<int>(gridDim.x) * kTeams) {
    const int w = row_window(p, row);
    if (w < 0) {  // the whole team
      zero_row<32 * WARPS>(p, row, q, scale, team.index());
      continue;
    }
    const size_t at = static_cast<size_t>(row) * p.channels;
    src.y = y + at;
    src.x = static_cast<const T*>(p.x) + at;
    src.stat = extra.stat + static_cast<size_t>(w) * p.groups;
    const float s = quantize_row<CHUNKS, WARPS, FULL>(src, p.channels, q + at, team);
    if (team.index() == 0) scale[row] = s;
  }
}

}  // namespace pq8
