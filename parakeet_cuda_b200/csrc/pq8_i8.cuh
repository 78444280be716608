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
#include "pq8_schedule.h"

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
// A few tokens (m <= 8): the weights are read once, 16 bytes per lane, by
// dp4a; latency- and HBM-bound. A warp takes R channels over the whole of K, a
// lane every 32nd 16-byte chunk; the lanes' sums meet in one reduction per
// output. With FUSED the tokens arrive in floating point and every CTA
// quantises them for itself into shared memory (the same few KB from L2 for
// all of them), which saves the launch and the round trip of a pass of its own:
// 1 x 1024 x 4096 (tokens x K x channels) from fp32 in 2.6 us against 5.0 in two
// launches, 8 x 640 x 8198 in 5.6 against 11.8 (in a graph). Product alone: 1 x
// 1024 x 4096 2.0 us (2.1 TB/s of weights: launch and one round trip to memory),
// 8 x 640 x 8198 4.2 (1.3 TB/s: eight dp4a sums per weight word).
constexpr int kI8GemvThreads = 256;
constexpr int kI8GemvMaxM = 8;

// Tokens in floating point, for the FUSED form.
struct I8Tokens {
  const void* x;
  long long ld;
  const float* norm_w;  // LayerNorm first, or NULL
  const float* norm_b;
  double eps;
  int type;
};

// One value of type `type` (PQ8_TYPE_*) at element `i` of p.
__device__ __forceinline__ float load_as_f32(const void* p, int type, size_t i) {
  return type == PQ8_TYPE_F32   ? static_cast<const float*>(p)[i]
         : type == PQ8_TYPE_F16 ? __half2float(static_cast<const __half*>(p)[i])
                                : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_from_f32(void* p, int type, size_t i, float v) {
  if (type == PQ8_TYPE_F32) static_cast<float*>(p)[i] = v;
  else if (type == PQ8_TYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// FUSED: tokens of type T, after a LayerNorm with NORM. One token is quantised by
// the whole CTA (up to 8192 columns), several by a warp each (up to 1024).
template <int M, int R, bool FUSED, typename T, bool NORM>
__global__ void __launch_bounds__(kI8GemvThreads, 2) i8_gemv_kernel(const I8Params p, const I8Tokens tokens, int y_type) {
  extern __shared__ int4 q_smem[];  // FUSED: [m][k] int8
  __shared__ float scale_smem[M];
  constexpr int kWarps = kI8GemvThreads / 32, kTeam = M == 1 ? kWarps : 1;
  __shared__ double team_smem[2 * kTeam];
  __shared__ float top_smem[kWarps];
  const int lane = threadIdx.x & 31;
  const int unit = static_cast<int>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const bool glu = p.epi == PQ8_EPI_GLU;
  const int half = p.n >> 1;
  // channel of local row r: consecutive ones, or for GLU the pairs (j, j + n / 2)
  constexpr int P = R > 1 ? R / 2 : 1;
  const int j0 = unit * (glu ? P : R);
  auto channel = [&](int r) { return glu ? (r < P ? j0 + r : half + j0 + r - P) : j0 + r; };
  auto valid = [&](int r) { return glu ? j0 + r % P < half : j0 + r < p.n; };
  const int chunks = p.k >> 4;
  const int4* wrow[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    wrow[r] = reinterpret_cast<const int4*>(p.w + static_cast<size_t>(valid(r) ? channel(r) : 0) * p.k);
  griddep_wait();
  griddep_launch();
  // The first weights are on their way while the tokens are quantised.
  constexpr int kAhead = 2;
  int4 ahead[kAhead][R];
#pragma unroll
  for (int a = 0; a < kAhead; ++a)
#pragma unroll
    for (int r = 0; r < R; ++r)
      ahead[a][r] = lane + 32 * a < chunks ? __ldg(wrow[r] + lane + 32 * a) : make_int4(0, 0, 0, 0);
  if constexpr (FUSED) {
    int8_t* q = reinterpret_cast<int8_t*>(q_smem);
    std::conditional_t<NORM, LayerNormSource<T, true>, PlainSource<T, true>> src;
    if constexpr (NORM) {
      src.w = tokens.norm_w;
      src.b = tokens.norm_b;
      src.eps = tokens.eps;
      src.inv_width = 1.0 / p.k;
      src.top_b = cta_max_abs(tokens.norm_b, p.k, top_smem);
    }
    const RowTeam<kTeam> team{team_smem};
    const int r = kTeam > 1 ? 0 : threadIdx.x >> 5;
    if (r < p.m) {
      src.x = static_cast<const T*>(tokens.x) + r * tokens.ld;
      const float s = quantize_row<32 / kChunk<T>, kTeam, false>(src, p.k, q + r * p.k, team);
      if (team.index() == 0) scale_smem[r] = s;
    }
    __syncthreads();
  }
  if (j0 >= p.out_cols) return;
  // lane i finishes the outputs of token i; what it needs besides the sums
  const int row = lane < M ? min(lane, p.m - 1) : 0;
  const float s = FUSED ? scale_smem[row] : p.x_scale[row];
  float t[R], b[R], res[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = valid(r) ? channel(r) : 0;
    t[r] = p.w_scale[j];
    b[r] = p.bias ? p.bias[j] : 0.0f;
    res[r] = p.epi == PQ8_EPI_RESIDUAL ? load_as_f32(p.resid, y_type, static_cast<size_t>(row) * p.out_cols + j) : 0.0f;
  }
  int acc[R][M];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < M; ++i) acc[r][i] = 0;
  auto add = [&](const int4(&wv)[R], int c) {
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int at = min(i, p.m - 1);
      const int4 xv = FUSED ? q_smem[at * chunks + c]
                            : __ldg(reinterpret_cast<const int4*>(p.x + static_cast<size_t>(at) * p.k) + c);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        acc[r][i] = __dp4a(wv[r].x, xv.x, acc[r][i]);
        acc[r][i] = __dp4a(wv[r].y, xv.y, acc[r][i]);
        acc[r][i] = __dp4a(wv[r].z, xv.z, acc[r][i]);
        acc[r][i] = __dp4a(wv[r].w, xv.w, acc[r][i]);
      }
    }
  };
#pragma unroll
  for (int a = 0; a < kAhead; ++a)
    if (lane + 32 * a < chunks) add(ahead[a], lane + 32 * a);
#pragma unroll 2
  for (int c = lane + 32 * kAhead; c < chunks; c += 32) {
    int4 wv[R];
#pragma unroll
    for (int r = 0; r < R; ++r) wv[r] = __ldg(wrow[r] + c);
    add(wv, c);
  }
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
  if (lane >= M || lane >= p.m) return;
  float z[R];
#pragma unroll
  for (int r = 0; r < R; ++r) z[r] = i8_scaled(mine[r], s, t[r], b[r]);
  const size_t y0 = static_cast<size_t>(row) * p.out_cols + j0;
  if (glu) {
#pragma unroll
    for (int r = 0; r < P; ++r)
      if (valid(r)) store_from_f32(p.y, y_type, y0 + r, __fdividef(z[r], 1.0f + __expf(-z[R > 1 ? r + P : 0])));
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (valid(r))
        store_from_f32(p.y, y_type, y0 + r,
                       p.epi == PQ8_EPI_RESIDUAL ? fmaf(p.alpha, z[r], res[r]) : act_f32(z[r], p.epi));
  }
}

// ---------------------------------------------------------------------------
// More tokens: 5th-generation tensor cores, tcgen05.mma kind::i8 (8-bit operands from
// shared memory, 32-bit integer sums in tensor memory).
//
// As in pq8_gemm, the MMA's M dimension is 128 weight rows and its N dimension BN
// tokens, so an epilogue thread owns one output channel (its scale and bias
// stay in registers) and a warp's store covers 32 consecutive channels of one
// token: coalesced for any n, without a staging tile (tiles staged for TMA
// stores measured no faster: 24000 x 1024 x 4096 to fp32 in 110 us against 104). Both operands are
// K-major 128-byte rows, brought by TMA into 128-byte swizzled stages of 128
// values of K; K past its end and rows past n or m arrive as zeros.
//
// PAIR: two CTAs share each MMA (cta_group::2, 256 weight rows): each loads
// its own 128 weight rows and half of the tokens. Single CTAs may split K:
// the S = 2, 4 or 8 CTAs of a cluster each sum a range of K, stage their sums
// in shared memory, and add them up by bulk reductions into one another's
// shared memory, CTA s finishing rows [s, s + 1) BN / S of the tile.
//
// Two accumulators let the next tile's products run under a tile's epilogue.
//
// Measured: 8192^3 350 us (3.14e15 operations/s, 0.93 of the rate taken for 8 bits:
// twice the bf16 product's); 24,000 x 1024 x 4096 with SiLU to bf16 101 us (2.0e15;
// the chip is at its power limit there, 990 W at 1.5 to 1.65 GHz, and the products
// alone take 66); 3000 x 4096 x 1024 15.3 to 17.6 us (64 pair tiles on 74 pairs);
// 375 x 1024 x 2048 GLU 5.6 us (3 us of launch, set-up and first loads).
//
// Warps: 0 and 2 TMA producers, 1 MMA issuer (and tensor-memory owner), 3
// scheduler of the MMA issuer, 4 on: epilogue.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  if constexpr (PAIR) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
// TMA load into this CTA's shared memory, counted on a barrier of the pair's leader.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const void* tmap, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];" ::"r"(smem_addr(dst)),
      "l"(tmap), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d_pair(void* dst, const void* tmap, int c0, int c1, int c2, int c3,
                                                 uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3, %4, %5}], [%6];" ::"r"(smem_addr(dst)),
      "l"(tmap), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
// Adds 32-bit integers of this CTA's shared memory to those at `dst` in a CTA of the cluster.
__device__ __forceinline__ void bulk_add_s2s_cluster(uint32_t dst, const void* src, uint32_t bytes, uint32_t mbar) {
  asm volatile(
      "cp.reduce.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes.add.s32 [%0], [%1], %2, [%3];" ::
          "r"(dst),
      "r"(smem_addr(src)), "r"(bytes), "r"(mbar)
      : "memory");
}

struct I8GemmParams {
  I8Params p;
  int n_tiles, m_tiles, k_blocks;  // 128-row weight tiles, BN-token tiles, 128-value K blocks
  int k_splits;
  int glu_blocks;  // GLU: tmap_w is [n / 32][2][16][k], so that a tile's rows come in one load
};

template <int BN_, bool PAIR_>
struct I8Cfg {
  static constexpr int STAGES = BN_ >= 128 ? 6 : 8;
  static constexpr int kRelease = 2;  // K blocks per meeting of the scheduler and the MMA warp
  static constexpr int BN = BN_, kCtas = PAIR_ ? 2 : 1;
  static constexpr bool PAIR = PAIR_;
  static constexpr int kTokens = BN / kCtas;  // token rows a CTA loads
  static constexpr int kABytes = 128 * 128, kBBytes = kTokens * 128, kStageBytes = kABytes + kBBytes;
  // Epilogue: kGroups groups of 4 warps (one per TMEM lane quarter), each with
  // kCols of the tile's tokens, E at a time. Sixteen warps for wide tiles: with
  // eight, two to a scheduler, the epilogue's chains of dependent operations left
  // most issue slots empty and it took longer than the products.
  static constexpr int kGroups = BN >= 64 ? 4 : 2, kEpiWarps = 4 * kGroups, kCols = BN / kGroups;
  static constexpr int E = kCols >= 16 ? 16 : 8;  // accumulator columns per tcgen05.ld
  static constexpr int kChunks = kCols / E;
  static constexpr int kScaleOff = STAGES * kStageBytes;  // token scales of each epilogue warp's part
  static constexpr int kBarOff = kScaleOff + kEpiWarps * kCols * 4;
  static constexpr int kNumBars = 2 * STAGES + 4 + 2;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kSmemBytes = kMiscOff + 16 + 1024;
  static constexpr int kTmemCols = 2 * BN <= 32 ? 32 : 2 * BN <= 64 ? 64 : 2 * BN <= 128 ? 128 : 2 * BN <= 256 ? 256 : 512;
  static constexpr int kThreads = (4 + kEpiWarps) * 32;
  static_assert(kTokens % 8 == 0 && BN % (PAIR ? 32 : 16) == 0 && BN <= 256 && kCols % E == 0, "tile shape");
  static_assert(kSmemBytes <= 227 * 1024, "shared memory overflow");
  static_assert(STAGES % 2 == 0, "the producers take stages in turn");
  static_assert(PAIR || BN * 128 * 4 <= STAGES * kStageBytes, "split K stages its sums in the ring");
};

template <int E>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&v)[E]) {
  if constexpr (E == 16) tmem_ld16(taddr, v);
  else tmem_ld8(taddr, v);
}

// f(the epilogue as a type): one test per chunk instead of one per output.
template <int V>
struct EpilogueTag {
  static constexpr int value = V;
};
template <typename F>
__device__ __forceinline__ void i8_epilogue(int epi, F&& f) {
  if (epi == PQ8_EPI_NONE) f(EpilogueTag<PQ8_EPI_NONE>{});
  else if (epi == PQ8_EPI_SILU) f(EpilogueTag<PQ8_EPI_SILU>{});
  else if (epi == PQ8_EPI_RESIDUAL) f(EpilogueTag<PQ8_EPI_RESIDUAL>{});
  else if (epi == PQ8_EPI_GLU) f(EpilogueTag<PQ8_EPI_GLU>{});
  else f(EpilogueTag<PQ8_EPI_RELU>{});
}

// The outputs of one channel for `cnt` <= E tokens (0: this lane stores
// nothing) from their sums v, token scales sx, channel scale t and bias b;
// `cols` elements apart at y. Every lane of the warp takes part. GLU: lanes
// 0-15 have a value channel and lanes 16-31 its gate; of each two tokens
// the lower lane finishes the first and the upper lane the second. least: of the values before
// a sigmoid so far. APART: with sigmoid2_apart.
template <typename T, int E, int EPI, bool APART = false>
__device__ __forceinline__ void i8_finish(const uint32_t (&v)[E], const T (&rv)[E], const float* sx, float t, float b,
                                          float alpha, T* y, int cols, int cnt, float& least) {
  constexpr bool kGlu = EPI == PQ8_EPI_GLU;
  constexpr int N = kGlu ? E / 2 : E;  // outputs of this lane
  const bool upper = (threadIdx.x & 16) != 0;
  const f32x2 t2 = pack2(t, t), b2 = pack2(b, b);
  float out[N];
  float a_prev = 0.0f, g_prev = 0.0f;  // GLU: the first of two outputs' value and gate
#pragma unroll
  for (int j = 0; j < E; j += 2) {
    const f32x2 s = *reinterpret_cast<const f32x2*>(sx + j);
    f32x2 z = fma2(mul2(pack2(static_cast<float>(static_cast<int>(v[j])), static_cast<float>(static_cast<int>(v[j + 1]))), s), t2, b2);
    if constexpr (kGlu) {
      float z0, z1;
      unpack2(z, &z0, &z1);
      const float other = __shfl_xor_sync(0xffffffffu, upper ? z0 : z1, 16);
      const float a = upper ? other : z0, gate = upper ? z1 : other;
      if (j % 4 == 0) {
        a_prev = a;
        g_prev = gate;
      } else {
        take_least(pack2(g_prev, gate), least);
        unpack2(mul2(pack2(a_prev, a), sigmoid2<APART>(pack2(g_prev, gate))), &out[j / 2 - 1], &out[j / 2]);
      }
    } else {
      if constexpr (EPI == PQ8_EPI_RESIDUAL) z = fma2(pack2(alpha, alpha), z, pack2(to_f32(rv[j]), to_f32(rv[j + 1])));
      if constexpr (EPI == PQ8_EPI_SILU) {
        take_least(z, least);
        z = mul2(z, sigmoid2<APART>(z));
      }
      unpack2(z, &out[j], &out[j + 1]);
      if constexpr (EPI == PQ8_EPI_RELU) {
        out[j] = relu_f32(out[j]);
        out[j + 1] = relu_f32(out[j + 1]);
      }
    }
  }
  constexpr int kStep = E / N;
  T* const y0 = y + (kGlu && upper ? cols : 0);
  const int mine = kGlu && upper ? cnt - 1 : cnt;  // GLU: tokens 1, 3, ... of the upper lanes
  if (cnt == E) {
#pragma unroll
    for (int j = 0; j < N; ++j) y0[static_cast<size_t>(j * kStep) * cols] = from_f32<T>(out[j]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j * kStep < mine) y0[static_cast<size_t>(j * kStep) * cols] = from_f32<T>(out[j]);
  }
}

// Residuals of `cnt` <= E tokens from m0 on of one channel.
template <typename T, int E>
__device__ __forceinline__ void i8_load_resid(T (&rv)[E], const T* res, int m0, int cols, int cnt) {
#pragma unroll
  for (int j = 0; j < E; ++j) rv[j] = j < cnt ? res[static_cast<size_t>(m0 + j) * cols] : from_f32<T>(0.0f);
}

template <typename T, int BN, bool PAIR>
__global__ void __launch_bounds__(I8Cfg<BN, PAIR>::kThreads, 1)
    i8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                   const __grid_constant__ I8GemmParams g) {
  using C = I8Cfg<BN, PAIR>;
  constexpr int STAGES = C::STAGES;
  const I8Params& p = g.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;   // [2]
  uint64_t* drain = acc_empty + 2;
  uint64_t* red_full = drain + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kMiscOff + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  const bool leader = rank == 0;
  const int S = PAIR ? 1 : g.k_splits;
  const bool split = S > 1;
  int* const status = p.status;
  const bool glu = p.epi == PQ8_EPI_GLU;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], C::kEpiWarps * C::kCtas);  // one arrival per epilogue warp
    }
    mbar_init(drain, 1);
    mbar_init(red_full, 1);
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_x);
  }
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the peer's barriers exist before anything arrives on them
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_slot, C::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, C::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Tiles: channel units fastest, then token tiles; the K splits of a tile are one cluster.
  const int n_units = (g.n_tiles + C::kCtas - 1) / C::kCtas;
  const int num_tiles = n_units * g.m_tiles;
  const int tile0 = static_cast<int>(blockIdx.x) / (split ? S : C::kCtas);
  const int tile_step = static_cast<int>(gridDim.x) / (split ? S : C::kCtas);
  const int my_split = split ? static_cast<int>(cluster_rank()) : 0;
  const int per_split = (g.k_blocks + S - 1) / S;
  const int kb0 = my_split * per_split, kb1 = min(kb0 + per_split, g.k_blocks);
  const ScheduleRange mine{tile0, num_tiles, tile_step, kb0, kb1};

  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------ producers
    // Two, taking K blocks (and so stages) in turn: a thread that has issued TMA
    // loads takes a few hundred cycles until its next barrier wait is answered.
    if (lane == 0) {
      const uint32_t me = warp >> 1;
      griddep_wait();
      if (me == 1) griddep_launch();
      const uint32_t full_at = PAIR ? map_to_rank(full, 0) : smem_addr(full);
      uint32_t it = 0;  // K blocks so far, of both producers
      Ring<STAGES> ring;
      ring.advance(me);
      for (int tile = tile0; tile < num_tiles; tile += tile_step) {
        const int unit = tile % n_units, token0 = (tile / n_units) * BN + static_cast<int>(rank) * C::kTokens;
        const int n_tile = unit * C::kCtas + static_cast<int>(rank);
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          if ((it & 1) != me) continue;
          if (!mbar_wait(&empty[ring.idx], ring.phase ^ 1u, abort_flag, status)) goto loads_done;
          uint8_t* a = smem + ring.idx * C::kStageBytes;
          const uint32_t bar = full_at + ring.idx * 8;
          if (leader) mbar_expect_tx(&full[ring.idx], C::kStageBytes * C::kCtas);
          auto load = [&](void* dst, const void* map, int row) {
            if constexpr (PAIR) tma_load_2d_pair(dst, map, kb * 128, row, bar);
            else tma_load_2d(dst, map, kb * 128, row, &full[ring.idx]);
          };
          if (glu) {
            // 16 rows of the first half, then the 16 gate rows of the same channels, four times
            if (g.glu_blocks) {
              if constexpr (PAIR) tma_load_4d_pair(a, &tmap_w, kb * 128, 0, 0, n_tile * 4, bar);
              else tma_load_4d(a, &tmap_w, kb * 128, 0, 0, n_tile * 4, &full[ring.idx]);
            } else {
#pragma unroll 1
              for (int i = 0; i < 8; ++i)
                load(a + i * 2048, &tmap_w, ((i & 1) ? p.n / 2 : 0) + n_tile * 64 + (i >> 1) * 16);
            }
          } else {
            load(a, &tmap_w, n_tile * 128);
          }
          load(a + C::kABytes, &tmap_x, token0);
          ring.advance(2);
        }
      }
    loads_done:
      // no copy may land in the shared memory of a CTA that has gone (the
      // leader's barriers count the peer's too, and the pair leaves together)
      if (leader)
        for (uint32_t j = it > STAGES ? it - STAGES : 0; j < it; ++j)
          if ((j & 1) == me) mbar_drain(&full[j % STAGES], (j / STAGES) & 1);
    }
    __syncwarp();
  } else if (warp == 3) {
    // ------------------------------------------------------------- scheduler
    // Waits on every barrier the products depend on and releases the MMA warp
    // through a named barrier: a shared-memory access by the warp that
    // issues tcgen05.mma is held behind the products it has queued, so its own
    // waits would drain the tensor pipe at every K block (128 x 16384 x 1024 in
    // tiles of 32: 39 us with the MMA warp waiting for itself, 35 so). A wait that gives up is
    // told to the MMA warp in the next meeting (pq8_schedule.h).
    if (leader) {
      Ring<STAGES> ring;
      schedule_products(
          mine, C::kRelease,
          [&](int local) {  // lane 0's answer; landed() makes it the warp's
            return lane != 0 || mbar_wait(&acc_empty[local & 1], ((local >> 1) & 1) ^ 1, abort_flag, status);
          },
          [&](int n, bool ok) {
            if (lane == 0)
              for (int b = 0; b < n && ok; ++b, ring.advance(1))
                ok = mbar_wait(&full[ring.idx], ring.phase, abort_flag, status);
            return __shfl_sync(0xffffffffu, ok, 0) != 0;
          },
          [&](bool bad) { return rendezvous_or(1, bad); });
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (leader) {
      constexpr uint32_t idesc = idesc_i8(128 * C::kCtas, BN);
      const uint64_t desc0 = smem_desc_sw128(smem_addr(smem));
      bool issued = false;
      Ring<STAGES> ring;
      const bool stop = issue_products(
          mine, C::kRelease, [&](bool bad) { return rendezvous_or(1, bad); },
          [&](int local, int kb, int n) {
            const int acc = local & 1;
            const uint32_t d = tmem + acc * BN;
            tc_fence_after();
            if (lane == 0) {
              for (int b = 0; b < n; ++b, ring.advance(1)) {
                const uint64_t ad = desc0 + ring.idx * (C::kStageBytes >> 4), bd = ad + (C::kABytes >> 4);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  mma_i8<PAIR>(d, ad + 2 * j, bd + 2 * j, idesc, (kb + b > kb0 || j > 0) ? 1u : 0u);
                if constexpr (PAIR) mma_commit_pair(&empty[ring.idx], 0x3);
                else mma_commit(&empty[ring.idx]);
              }
              if (kb + n == kb1) {
                if constexpr (PAIR) mma_commit_pair(&acc_full[acc], 0x3);
                else mma_commit(&acc_full[acc]);
              }
            }
            __syncwarp();
            issued = true;
          });
      if (stop && issued && lane == 0) {  // the products under way end before the CTA is torn down
        if constexpr (PAIR) mma_commit_pair(drain, 0x1);
        else mma_commit(drain);
        mbar_drain(drain, 0);
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // -------------------------------------------------------------- epilogue
    constexpr int E = C::E;
    const int q = warp & 3, group = (warp - 4) >> 2, r = q * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(q * 32) << 16;
    float* sx = reinterpret_cast<float*>(smem + C::kScaleOff) + (warp - 4) * C::kCols;
    const uint32_t acc_empty_at = PAIR ? map_to_rank(acc_empty, 0) : smem_addr(acc_empty);
    bool published = false, apart = false;
    griddep_wait();
    int local = 0;
    for (int tile = tile0; tile < num_tiles; tile += tile_step, ++local) {
      const int n_tile = (tile % n_units) * C::kCtas + static_cast<int>(rank);
      const int token0 = (tile / n_units) * BN;
      const int acc = local & 1;
      // this thread's channel: output column `col`, weight row `row`
      const int col = glu ? n_tile * 64 + q * 16 + (lane & 15) : n_tile * 128 + r;
      const int row = glu && lane >= 16 ? p.n / 2 + col : col;
      const bool valid = col < p.out_cols;
      const float t = valid ? __ldg(p.w_scale + row) : 0.0f;
      const float b = (valid && p.bias != nullptr) ? __ldg(p.bias + row) : 0.0f;
      T* const y = static_cast<T*>(p.y) + col;
      const T* const res = static_cast<const T*>(p.resid) + col;
      const int cols = p.out_cols;

      // the scales of up to kCols tokens from m0 on, for this warp
      auto load_scales = [&](int m0) {
        __syncwarp();  // the previous tile's have been read
#pragma unroll
        for (int i = 0; i < C::kCols; i += 32)
          if (i + lane < C::kCols) sx[i + lane] = m0 + i + lane < p.m ? __ldg(p.x_scale + m0 + i + lane) : 0.0f;
        __syncwarp();
      };
      if (!split) {
        const int first = token0 + group * C::kCols;
        load_scales(first);
        bool ok = true;
        // (One kind per loop: 16 registers of residuals are held where there are any.)
        i8_epilogue(p.epi, [&](auto epi) {
          constexpr int EPI = decltype(epi)::value;
          constexpr bool kSigmoid = EPI == PQ8_EPI_SILU || EPI == PQ8_EPI_GLU;
          auto release = [&] {  // every lane has read its sums: the accumulator is free
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (PAIR) mbar_arrive_cluster(acc_empty_at + acc * 8);
              else mbar_arrive(&acc_empty[acc]);
            }
          };
          T rv[E];
          if constexpr (EPI == PQ8_EPI_RESIDUAL) i8_load_resid<T, E>(rv, res, first, cols, valid ? min(E, p.m - first) : 0);
          ok = mbar_wait(&acc_full[acc], (local >> 1) & 1, abort_flag, status);
          if (!ok) return;
          tc_fence_after();
          float least = 0.0f;
          auto part = [&](auto apart) {  // this warp's part of the tile
#pragma unroll 1
            for (int cc = 0; cc < C::kChunks; ++cc) {
              const int m0 = first + cc * E, cnt = min(E, p.m - m0);
              uint32_t v[E];
              tmem_ld_cols<E>(tmem + lane_base + acc * BN + group * C::kCols + cc * E, v);
              tmem_wait_ld();
              if (!kSigmoid && cc + 1 == C::kChunks) release();
              if (cnt > 0) {
                T* const yp = y + static_cast<size_t>(m0) * cols;
                i8_finish<T, E, EPI, decltype(apart)::value>(v, rv, sx + cc * E, t, b, p.alpha, yp, cols, valid ? cnt : 0,
                                                             least);
                if constexpr (EPI == PQ8_EPI_RESIDUAL)
                  if (cc + 1 < C::kChunks) i8_load_resid<T, E>(rv, res, m0 + E, cols, valid ? min(E, p.m - m0 - E) : 0);
              }
            }
          };
          if constexpr (!kSigmoid) {
            part(std::false_type{});
          } else {
            // A sigmoid below the fast form's range: the part once more, so that the sums have
            // to stay until here, and the next tile without the fast form (values that
            // reach there in one tile do so in most: 24,000 x 1024 x 4096 with values of
            // deviation 37 in 142 us, with both forms every time 204).
            if (!apart) part(std::false_type{});
            if (apart || __any_sync(0xffffffffu, !(least >= kSigmoidLeast))) {
              least = 0.0f;
              part(std::true_type{});
              apart = __any_sync(0xffffffffu, !(least >= kSigmoidLeast));
            }
            release();
          }
        });
        if (!ok) break;
      } else {
        // K split: this CTA's sums to shared memory, [token][channel] (the
        // ring: every load has been multiplied) ...
        int* const stage = reinterpret_cast<int*>(smem);
        if (!mbar_wait(&acc_full[0], 0, abort_flag, status)) break;
        tc_fence_after();
#pragma unroll 1
        for (int cc = 0; cc < C::kChunks; ++cc) {
          const int c0 = group * C::kCols + cc * E;
          uint32_t v[E];
          tmem_ld_cols<E>(tmem + lane_base + c0, v);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < E; ++j) stage[(c0 + j) * 128 + r] = static_cast<int>(v[j]);
        }
        tc_fence_before();
        fence_proxy_async_smem();  // read and added to by the bulk-copy unit
        const int R = BN / S;      // tokens each CTA finishes
        if (warp == 4 && lane == 0) mbar_expect_tx(red_full, static_cast<uint32_t>((S - 1) * R * 512));
        __syncwarp();
        cluster_sync();  // every CTA's sums are staged
        published = true;
        // ... then added to each finishing CTA's own, one bulk reduction each
        if (warp == 4 && lane < S - 1) {
          const uint32_t d = static_cast<uint32_t>((my_split + 1 + lane) % S);
          int* src = stage + static_cast<int>(d) * R * 128;
          bulk_add_s2s_cluster(map_to_rank(src, d), src, static_cast<uint32_t>(R * 512), map_to_rank(red_full, d));
        }
        __syncwarp();
        const int rows = R / C::kGroups, off = my_split * R + group * rows;
        const int cnt_all = min(rows, p.m - token0 - off);
        load_scales(token0 + off);
        if (!mbar_wait(red_full, 0, abort_flag, status)) break;
#pragma unroll 1
        for (int c0 = 0; c0 < cnt_all; c0 += E) {
          const int cnt = min(E, cnt_all - c0), m0 = token0 + off + c0;
          i8_epilogue(p.epi, [&](auto epi) {
            constexpr int EPI = decltype(epi)::value;
            T rv[E];
            if constexpr (EPI == PQ8_EPI_RESIDUAL) i8_load_resid<T, E>(rv, res, m0, cols, valid ? cnt : 0);
            uint32_t v[E];
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = j < cnt ? static_cast<uint32_t>(stage[(off + c0 + j) * 128 + r]) : 0u;
            T* const yp = y + static_cast<size_t>(m0) * cols;
            float least = 0.0f;
            i8_finish<T, E, EPI>(v, rv, sx + c0, t, b, p.alpha, yp, cols, valid ? cnt : 0, least);
            if constexpr (EPI == PQ8_EPI_SILU || EPI == PQ8_EPI_GLU)
              if (__any_sync(0xffffffffu, !(least >= kSigmoidLeast)))
                i8_finish<T, E, EPI, true>(v, rv, sx + c0, t, b, p.alpha, yp, cols, valid ? cnt : 0, least);
          });
        }
      }
    }
    if (split && !published) {  // gave up before the sums were staged
      __syncwarp();
      cluster_sync();
    }
  }

  if (split && warp < 4) {  // these warps publish nothing, but the barrier counts every thread
    __syncwarp();
    cluster_arrive_relaxed();
    cluster_wait();
  }
  __syncthreads();
  // The pair's MMAs read both CTAs' shared memory, and a split's sums travel
  // between CTAs: nobody leaves before everybody is done.
  if (PAIR || split) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem, C::kTmemCols);
    else tmem_dealloc(tmem, C::kTmemCols);
  }
}

}  // namespace pq8
