// int8 matrix product with a scale per row of each operand:
//   C[m, n] = f((sum_k A[m, k] B[n, k]) * sa[m] * sb[n] + bias[n]),  f = identity or GELU
// A [M, K] are int8 activations with a scale per token, B [N, K] int8 weights with a scale per output
// channel.  The sum is exact in int32 (|A|, |B| <= 128 and K <= 131071), so any split of K and any order give
// the same bits; it is converted to fp32, scaled and rounded once to C's dtype.
#include "common.cuh"
#include "host_util.h"
#include "vec8.cuh"

namespace da {
namespace i8 {

constexpr int64_t kMaxK = 131071;

struct Params {
  const int8_t* a;
  const int8_t* b;
  const float* sa;
  const float* sb;
  const void* bias;
  void* c;
  int64_t lda, ldb, ldc;
  int M, N, K, bias_dtype, c_dtype, gelu;
  int turns;  // the pair kernel's epilogue warps take turns
  int tma_c;  // C's rows take TMA stores (base, stride and width in whole 16-byte words)
  int* status;
  Div31 per_group;  // the pair kernel: tiles in a group of 8 rows of tiles
};

// One output before its rounding to C's dtype: every kernel here computes exactly this.
DA_DEV float finish(int acc, float sa, float sb, float bias) { return __fmaf_rn(__fmul_rn((float)acc, sa), sb, bias); }

// The same for two neighbouring columns, whose accumulators come as bits.
DA_DEV F2 finish2(float acc0, float acc1, float sa, F2 sb, F2 bias) {
  return fma2(mul2(f2((float)__float_as_int(acc0), (float)__float_as_int(acc1)), dup(sa)), sb, bias);
}

DA_DEV float col_bias(const Params& p, int n) { return p.bias ? load1(p.bias, p.bias_dtype, n) : 0.f; }

// ----------------------------------------------------------------------------------------------- large products
// Persistent CTA pairs: a pair computes 256 x 256 tiles (each CTA 128 rows of A and, of every K stage, half of
// B's rows) with cta_group::2 kind::i8 instructions of 256 x 256 x 32; two int32 accumulators of 256 TMEM columns
// each, so that the epilogue of one tile runs under the products of the next.
// A stage holds 128 bytes of K (5 stages of 32 KB for long K; 3 stages of 64 KB measured the same; 4 leave room for the
// columns' scales where K is short, and cost 2 % where it is long).
//
// Bound: long K by the tensor pipe (79 % active; a dependent instruction takes ~180 cycles, 136 at the nominal rate):
// 8192 x 4096 x 4096 in 89 us, 3.1 POP/s, 16384 x 8192 x 8192 in 650 us, 3.4 POP/s.  Short K by the output: 32768 x 512 x
// 1536 in 30 us, its 100 MB near the 3.4 to 3.9 TB/s at which HBM takes writes alone; with GELU 42.6 us, of which the
// stores are not the bound (an earlier form at 47.4 us took 45.5 without them): the epilogue's 16 instructions a value
// fill 59 % of the issue slots, and 4 warps a scheduler, which 96 registers allow, do not cover the waits in their chains.
template <bool kTurns>  // of the epilogue warps: see the epilogue
struct Pair {
  static constexpr int kTile = 256;  // rows and columns of a pair's tile
  static constexpr int kOperand = 128 * 128;
  static constexpr int kStageBytes = 2 * kOperand;
  static constexpr int kStages = kTurns ? 5 : 4;
  static constexpr int kEpilogueWarps = 16;
  static constexpr int kOff = kStages * kStageBytes;         // an output box per epilogue warp
  static constexpr int kColumns = kOff + kEpilogueWarps * 4096;  // and the scales and biases of its columns
  static constexpr int kSmem = kColumns + (kTurns ? 0 : kEpilogueWarps * 512);
  static constexpr int kThreads = 128 + 32 * kEpilogueWarps;  // warps 0, 2 TMA; 1 MMA; 3 idle; then the epilogue
  static constexpr int kGroupM = 8;  // row tiles that run through the columns together (A and B stay in L2)
};

template <int kOut, bool kGelu, bool kTurns>
__global__ void __launch_bounds__(Pair<kTurns>::kThreads, 1) gemm_pair_kernel(const __grid_constant__ CUtensorMap ta,
                                                                              const __grid_constant__ CUtensorMap tb,
                                                                              const __grid_constant__ CUtensorMap tc,
                                                                              const Params p) {
  using C = Pair<kTurns>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[C::kStages], empty[C::kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = (int)(cluster_ctarank() & 1u);
  const int m_tiles = (p.M + C::kTile - 1) / C::kTile, n_tiles = (p.N + C::kTile - 1) / C::kTile;
  const int tiles = m_tiles * n_tiles, pairs = gridDim.x / 2, pair = blockIdx.x / 2;
  const int my_tiles = pair < tiles ? (tiles - 1 - pair) / pairs + 1 : 0;
  const int nk = (p.K + 127) / 128;
  Abort ab{&abort_flag, p.status};

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kTurns ? C::kEpilogueWarps : 2 * C::kEpilogueWarps);  // its epilogue warps in both CTAs
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<2>(&tmem_base, 2 * C::kTile);
    tmem_relinquish<2>();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  grid_dependency_wait();
  grid_launch_dependents();
  const uint32_t tmem = tmem_base;
  auto tile_mn = [&](int i, int& m0, int& n0) {
    const uint32_t t = pair + i * pairs;
    const uint32_t group = p.per_group.div(t), in = t - group * p.per_group.d;
    const uint32_t height = min(C::kGroupM, m_tiles - (int)group * C::kGroupM);
    const uint32_t n = height == C::kGroupM ? in / C::kGroupM : in / height;
    m0 = (int)(group * C::kGroupM + in - n * height) * C::kTile;
    n0 = (int)n * C::kTile;
  };

  if ((warp == 0 || warp == 2) && lane == 0) {
    // ---------------------------------------------------------------- TMA producers (alternate stages)
    const int pi = warp == 0 ? 0 : 1;
    prefetch_tmap(&ta);
    prefetch_tmap(&tb);
    bool ok = true;
    int it = 0, last = -1;
    for (int i = 0; ok && i < my_tiles; ++i) {
      int m0, n0;
      tile_mn(i, m0, n0);
      for (int kb = 0; kb < nk; ++kb, ++it) {
        if ((it & 1) != pi) continue;
        const int s = it % C::kStages;
        if (!mbar_wait(&empty[s], ((it / C::kStages) & 1u) ^ 1u, ab, 71)) { ok = false; break; }
        if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::kStageBytes);
        const uint32_t bar = mapa_shared(smem_u32(&full[s]), 0);
        uint8_t* sa = smem + s * C::kStageBytes;
        tma_load_2d_pair(&ta, bar, sa, kb * 128, m0 + rank * 128);
        tma_load_2d_pair(&tb, bar, sa + C::kOperand, kb * 128, n0 + rank * 128);
        last = it;
      }
    }
    // After a wait that gave up, this producer's loads in flight.  (Otherwise every load has been consumed before
    // the epilogue's last tile; and a stage's phase may have moved on by two, which a wait would not notice.)
    if (rank == 0 && !ok)
      for (int j = (last - C::kStages + 1 > 0 ? last - C::kStages + 1 : 0); j <= last; ++j)
        if ((j & 1) == pi) mbar_wait_drain(&full[j % C::kStages], (j / C::kStages) & 1u);
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---------------------------------------------------------------- MMA issuer (leader)
    const uint32_t idesc = idesc_i8(C::kTile, C::kTile);
    bool ok = true;
    int it = 0;
    for (int i = 0; ok && i < my_tiles; ++i) {
      const int buf = i & 1;
      if (i >= 2 && !mbar_wait(&acc_empty[buf], ((i >> 1) - 1) & 1u, ab, 72)) break;
      tc_fence_after();
      const uint32_t d = tmem + buf * C::kTile;
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = it % C::kStages;
        if (!mbar_wait(&full[s], (it / C::kStages) & 1u, ab, 73)) { ok = false; break; }
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + s * C::kStageBytes);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_i8_ss<2>(d, sdesc_sw128(sa + k * 32, 16, 1024), sdesc_sw128(sa + C::kOperand + k * 32, 16, 1024), idesc,
                       (kb > 0 || k > 0) ? 1u : 0u);
        mma_commit_pair(smem_u32(&empty[s]));
      }
      if (ok) mma_commit_pair(smem_u32(&acc_full[buf]));
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- epilogue.  All 16 warps take every tile, 32 rows
    // x 64 columns each; or, in turns, 8 warps every second tile (and accumulator), 32 x 128 each, so that one
    // group's waits lie under the other's arithmetic.
    constexpr int turns = kTurns ? 2 : 1, width = 64 * turns;
    const int quad = warp & 3, turn = kTurns ? (warp - 4) / 8 : 0, part = kTurns ? (warp - 4) / 4 & 1 : (warp - 4) / 4;
    uint8_t* box = smem + C::kOff + (warp - 4) * 4096;
    const bool vec_cols = reinterpret_cast<uintptr_t>(p.sb) % 16 == 0 &&
                          (!p.bias || (p.bias_dtype == DA_F32 && reinterpret_cast<uintptr_t>(p.bias) % 16 == 0));
    // Short K: a tile's scales and biases, fetched a tile ahead (a lane two columns) and read back from shared memory as
    // (s, s, b, b), and its column steps unrolled.  Loading them where they are used waited at every step: 32768 x 512 x
    // 1536 with GELU 48.7 us, now 46.9, unrolled 43.0; without 31.5, 29.9 and 29.6.
    float4* columns = reinterpret_cast<float4*>(smem + C::kColumns) + (warp - 4) * 32;
    float4 next = make_float4(0.f, 0.f, 0.f, 0.f);
    float next_sa = 0.f;
    const bool vec2 = reinterpret_cast<uintptr_t>(p.sb) % 8 == 0 &&
                          (!p.bias || (p.bias_dtype == DA_F32 && reinterpret_cast<uintptr_t>(p.bias) % 8 == 0));
    auto fetch = [&](int i) {
      if (i >= my_tiles) return;
      int m0, n0;
      tile_mn(i, m0, n0);
      const int row = m0 + rank * 128 + quad * 32 + lane;
      next_sa = row < p.M ? p.sa[row] : 0.f;
      if (kTurns) return;
      const int n = n0 + part * width + lane * 2;
      if (vec2 && n + 2 <= p.N) {
        const float2 t = __ldg(reinterpret_cast<const float2*>(p.sb + n));
        const float2 u = p.bias ? __ldg(reinterpret_cast<const float2*>(static_cast<const float*>(p.bias) + n))
                                : make_float2(0.f, 0.f);
        next = make_float4(t.x, t.y, u.x, u.y);
      } else {
        if (n < p.N) next.x = p.sb[n], next.z = col_bias(p, n);
        if (n + 1 < p.N) next.y = p.sb[n + 1], next.w = col_bias(p, n + 1);
      }
    };
    fetch(turn);
    constexpr int kStep = 16;  // columns at a time: what GELU and its constants need stays in 96 registers
    constexpr int per_box = kOut == DA_F32 ? 32 : 64;  // columns in 128 bytes
    bool ok = true;
    for (int i = turn; i < my_tiles; i += turns) {
      const int buf = i & 1;
      int m0, n0;
      tile_mn(i, m0, n0);
      const int row0 = m0 + rank * 128 + quad * 32;
      const float sa = next_sa;
      if constexpr (!kTurns) {
        __syncwarp();
        columns[lane] = next;
        __syncwarp();
      }
      fetch(i + turns);
      if (ok) ok = mbar_wait(&acc_full[buf], (i >> 1) & 1u, ab, 74);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      if (ok) {
#pragma unroll (kTurns ? 1 : 4)
        for (int c = 0; c < width; c += kStep) {
          const int col = n0 + part * width + c;
          float v[kStep];
          tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + buf * C::kTile + part * width + c, v);
          tmem_wait_ld();
          if (c + kStep == width) {  // the last columns of this accumulator are in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(&acc_empty[buf]), 0));
          }
          if (col >= p.N || row0 >= p.M) continue;
          F2 y[kStep / 2];
          if constexpr (!kTurns) {
#pragma unroll
            for (int e = 0; e < kStep / 2; ++e) {
              const float4 at = columns[c / 2 + e];
              y[e] = finish2(v[2 * e], v[2 * e + 1], sa, f2(at.x, at.y), f2(at.z, at.w));
            }
          } else if (vec_cols && col + kStep <= p.N) {
#pragma unroll
            for (int e = 0; e < kStep / 4; ++e) {
              const float4 s = __ldg(reinterpret_cast<const float4*>(p.sb + col) + e);
              float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
              if (p.bias) b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.bias) + col) + e);
              y[2 * e] = finish2(v[4 * e], v[4 * e + 1], sa, f2(s.x, s.y), f2(b.x, b.y));
              y[2 * e + 1] = finish2(v[4 * e + 2], v[4 * e + 3], sa, f2(s.z, s.w), f2(b.z, b.w));
            }
          } else {
#pragma unroll
            for (int e = 0; e < kStep; ++e)
              v[e] = col + e < p.N ? finish(__float_as_int(v[e]), sa, p.sb[col + e], col_bias(p, col + e)) : 0.f;
#pragma unroll
            for (int e = 0; e < kStep / 2; ++e) y[e] = f2(v[2 * e], v[2 * e + 1]);
          }
          if constexpr (kGelu) {
#pragma unroll
            for (int e = 0; e < kStep / 2; ++e) y[e] = gelu2(y[e]);
          }
          const int in_box = c % per_box;
          if (in_box == 0) {  // a free output box
            if (lane == 0) tma_store_wait_read<0>();
            __syncwarp();
          }
          const uint32_t dst = smem_u32(box);
          if constexpr (kOut == DA_F32) {
#pragma unroll
            for (int e = 0; e < kStep / 4; ++e) {
              float a0, a1, a2, a3;
              split(y[2 * e], a0, a1);
              split(y[2 * e + 1], a2, a3);
              st_shared_v4(dst + sw128_offset(lane, in_box / 4 + e), __float_as_uint(a0), __float_as_uint(a1),
                           __float_as_uint(a2), __float_as_uint(a3));
            }
          } else {
            using T = typename std::conditional<kOut == DA_BF16, __nv_bfloat16, __half>::type;
#pragma unroll
            for (int e = 0; e < kStep / 8; ++e)
              st_shared_v4(dst + sw128_offset(lane, in_box / 8 + e), narrow<T>(y[4 * e]), narrow<T>(y[4 * e + 1]),
                           narrow<T>(y[4 * e + 2]), narrow<T>(y[4 * e + 3]));
          }
          if (in_box + kStep != per_box && col + kStep < p.N) continue;  // more of the box follows
          const int col0 = col - in_box;
          if (p.tma_c) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tc, box, col0, row0);
              tma_store_commit();
            }
          } else {  // rows of C that no TMA store takes: lanes along the columns
            __syncwarp();
            const int cols = min(per_box, p.N - col0), rows = min(32, p.M - row0);
            const uint8_t* b = box;
            using E = typename std::conditional<kOut == DA_F32, float, uint16_t>::type;
            E* dst = static_cast<E*>(p.c) + (int64_t)row0 * p.ldc + col0;
            auto value = [&](int r, int e) {
              return *reinterpret_cast<const E*>(b + sw128_offset(r, e * sizeof(E) / 16) + e * sizeof(E) % 16);
            };
            if (rows == 32 && cols == per_box) {  // 8 rows' reads before their writes
#pragma unroll 1
              for (int r0 = 0; r0 < 32; r0 += 8) {
                E v[8][per_box / 32];
#pragma unroll
                for (int r = 0; r < 8; ++r)
#pragma unroll
                  for (int e = 0; e < per_box / 32; ++e) v[r][e] = value(r0 + r, lane + 32 * e);
#pragma unroll
                for (int r = 0; r < 8; ++r, dst += p.ldc)
#pragma unroll
                  for (int e = 0; e < per_box / 32; ++e) dst[lane + 32 * e] = v[r][e];
              }
            } else {
              for (int r = 0; r < rows; ++r, dst += p.ldc)
                for (int e = lane; e < cols; e += 32) dst[e] = value(r, e);
            }
            __syncwarp();
          }
        }
      }
    }
    if (lane == 0) tma_store_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) tmem_dealloc<2>(tmem, 2 * C::kTile);
}

template <int kOut, bool kGelu, bool kTurns>
int launch_pair(const Params& p, cudaStream_t st) {
  using C = Pair<kTurns>;
  constexpr int elem = kOut == DA_F32 ? 4 : 2;
  CUtensorMap ta, tb, tc;
  if (int rc = make_tmap_2d(&ta, p.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.K, p.M, p.lda, 128, 128)) return rc;
  if (int rc = make_tmap_2d(&tb, p.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.K, p.N, p.ldb, 128, 128)) return rc;
  tc = ta;
  if (p.tma_c) {
    const CUtensorMapDataType dt = kOut == DA_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : kOut == DA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if (int rc = make_tmap_2d(&tc, p.c, dt, elem, p.N, p.M, (uint64_t)p.ldc * elem, 128 / elem, 32)) return rc;
  }
  constexpr auto kern = gemm_pair_kernel<kOut, kGelu, kTurns>;
  if (int rc = allow_smem<kern>(C::kSmem + 1024)) return rc;
  const int64_t tiles = (int64_t)((p.M + C::kTile - 1) / C::kTile) * ((p.N + C::kTile - 1) / C::kTile);
  const int pairs = tiles < sm_count() / 2 ? (int)tiles : sm_count() / 2;
  return launch_kernel(kern, dim3(2 * pairs), dim3(C::kThreads), C::kSmem + 1024, st, true, ta, tb, tc, p);
}

template <int kOut>
int dispatch_pair(const Params& p, cudaStream_t st) {
  if (p.turns) return p.gelu ? launch_pair<kOut, true, true>(p, st) : launch_pair<kOut, false, true>(p, st);
  return p.gelu ? launch_pair<kOut, true, false>(p, st) : launch_pair<kOut, false, false>(p, st);
}

// ----------------------------------------------------------------------------------------------- few tokens
// Up to a few hundred tokens the weights' bytes and the length of one CTA's chain of K stages set the time, not the
// products.  Here the output channels are the instruction's 128 rows and the tokens its columns (kTn of them, so
// one token costs a 128 x 16 instruction, not 128 x 256), and the K stages of a tile are split over a cluster of
// up to 8 CTAs: each leaves its int32 sums in shared memory, and after a cluster barrier every CTA adds all of the
// cluster's sums for its share of the tokens through distributed shared memory (exact, so in any order) and
// stores them.
//
// Bound: latency.  1 x 512 x 1536 with GELU in 3.7 us.  Over 24 layers' weights in turn, which L2 does not hold:
// 1 x 4096 x 4096 in 6.9 us (2.4 TB/s of weights), 24 x 4096 x 4096 in 7.7 us, 128 x 4096 x 4096 in 10.4 us, 16 x 8192 x 8192 in
// 14.7 us (4.6 TB/s).  With weights that stay in L2 5.5, 6.1 and 9.1 us for the first three.
template <int kTn>
struct Few {
  static constexpr int kStageBytes = (128 + kTn) * 128;
  static constexpr int kStages = kTn == 128 ? 6 : 8;
  static constexpr int kSumBytes = kTn * 128 * 4;  // aliases the stages, which every product has read by then
  static constexpr int kSmem = kStages * kStageBytes;
  static constexpr int kCols = kTn < 32 ? 32 : kTn;  // TMEM columns
  static constexpr int kThreads = 192;               // warp 0 TMA, 1 MMA, 2-5 epilogue
  static_assert(kSumBytes <= kSmem);
};

template <int kTn, int kSplits>
__global__ void __launch_bounds__(Few<kTn>::kThreads, 1) gemm_few_kernel(const __grid_constant__ CUtensorMap ta,
                                                                         const __grid_constant__ CUtensorMap tb,
                                                                         const Params p) {
  using C = Few<kTn>;
  constexpr int splits = kSplits;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[C::kStages], empty[C::kStages], done;
  __shared__ float scale[kTn];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  const int n_tiles = (p.N + 127) / 128;
  const int n0 = tile % n_tiles * 128, m0 = tile / n_tiles * kTn;
  const int nk_all = (p.K + 127) / 128, per = (nk_all + splits - 1) / splits;
  const int kb0 = rank * per, nk = max(0, min(per, nk_all - kb0));
  Abort ab{&abort_flag, p.status};

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<1>(&tmem_base, C::kCols);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dependency_wait();
  grid_launch_dependents();
  const uint32_t tmem = tmem_base;
  int ch_n = p.N;  // an epilogue thread's first channel, the scales and biases of its two
  float s0 = 0.f, s1 = 0.f, b0 = 0.f, b1 = 0.f;

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int kb = 0;
      for (; kb < nk; ++kb) {
        const int s = kb % C::kStages;
        if (!mbar_wait(&empty[s], ((kb / C::kStages) & 1u) ^ 1u, ab, 75)) { ok = false; break; }
        mbar_arrive_expect_tx(&full[s], C::kStageBytes);
        tma_load_2d(&tb, &full[s], smem + s * C::kStageBytes, (kb0 + kb) * 128, n0);
        tma_load_2d(&ta, &full[s], smem + s * C::kStageBytes + 128 * 128, (kb0 + kb) * 128, m0);
      }
      for (int j = max(0, kb - C::kStages); !ok && j < kb; ++j)
        mbar_wait_drain(&full[j % C::kStages], (j / C::kStages) & 1u);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      bool ok = true;
      for (int kb = 0; kb < nk; ++kb) {
        const int s = kb % C::kStages;
        ok = mbar_wait(&full[s], (kb / C::kStages) & 1u, ab, 76);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sw = smem_u32(smem + s * C::kStageBytes), sx = sw + 128 * 128;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_i8_ss<1>(tmem, sdesc_sw128(sw + k * 32, 16, 1024), sdesc_sw128(sx + k * 32, 16, 1024), idesc_i8(128, kTn),
                       (kb > 0 || k > 0) ? 1u : 0u);
        mma_commit<1>(smem_u32(&empty[s]));
      }
      mma_commit<1>(smem_u32(&done));
      if (!ok) mbar_wait_drain(&done, 0);
    }
  } else {
    const int quad = warp & 3, t = threadIdx.x - 64;
    // what the stores need, fetched under the products
    for (int i = t; i < kTn; i += 128) scale[i] = m0 + i < p.M ? p.sa[m0 + i] : 0.f;
    ch_n = n0 + t % 64 * 2;
    if (ch_n < p.N) {
      s0 = p.sb[ch_n];
      b0 = col_bias(p, ch_n);
    }
    if (ch_n + 1 < p.N) {
      s1 = p.sb[ch_n + 1];
      b1 = col_bias(p, ch_n + 1);
    }
    bool ok = mbar_wait(&done, 0, ab, 77);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    // sums [token][channel]
    int* sums = reinterpret_cast<int*>(smem);
#pragma unroll 1
    for (int c = 0; c < kTn; c += 16) {
      float v[16];
      tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + c, v);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 16; ++e) sums[(c + e) * 128 + quad * 32 + lane] = ok && nk > 0 ? __float_as_int(v[e]) : 0;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (splits > 1) cluster_sync();
  if (warp >= 2 && ch_n < p.N) {
    // a thread takes two neighbouring channels of every second token of this CTA's share, kAtOnce tokens together
    constexpr int kAtOnce = kSplits == 8 ? 2 : 4;
    const int t = threadIdx.x - 64;
    const int tokens = min(kTn, p.M - m0), share = (tokens + splits - 1) / splits;
    const int last = min(tokens, (rank + 1) * share);
    const int elem = p.c_dtype == DA_F32 ? 4 : 2;
    const bool two = ch_n + 1 < p.N;
    const bool pair = two && p.ldc % 2 == 0 && reinterpret_cast<uintptr_t>(p.c) % (2 * elem) == 0;
    uint32_t peer[kSplits];
#pragma unroll
    for (int r = 0; r < kSplits; ++r) {
      const uint32_t own = smem_u32(smem) + t % 64 * 8;
      peer[r] = kSplits > 1 ? mapa_shared(own, (uint32_t)(rank + r) % kSplits) : own;
    }
    for (int tok0 = rank * share + t / 64; tok0 < last; tok0 += 2 * kAtOnce) {
      int a0[kAtOnce] = {}, a1[kAtOnce] = {};
#pragma unroll
      for (int r = 0; r < kSplits; ++r)
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const int tok = min(tok0 + 2 * u, kTn - 1);
          int x, y;
          asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(peer[r] + tok * 512));
          a0[u] += x;
          a1[u] += y;
        }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int tok = tok0 + 2 * u;
        if (tok >= last) break;
        const float sa = scale[tok];
        float y0 = finish(a0[u], sa, s0, b0), y1 = two ? finish(a1[u], sa, s1, b1) : 0.f;
        if (p.gelu) split(gelu2(f2(y0, y1)), y0, y1);
        const int64_t at = (int64_t)(m0 + tok) * p.ldc + ch_n;
        if (pair) {
          if (p.c_dtype == DA_F32) *reinterpret_cast<float2*>(static_cast<float*>(p.c) + at) = make_float2(y0, y1);
          else *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.c) + at) =
                   p.c_dtype == DA_BF16 ? pack_bf16x2(y0, y1) : pack_f16x2(y0, y1);
        } else {
          store1(p.c, p.c_dtype, at, y0);
          if (two) store1(p.c, p.c_dtype, at + 1, y1);
        }
      }
    }
  }
  __syncthreads();
  if (splits > 1) cluster_sync();  // peers may still read this CTA's sums
  if (warp == 1) tmem_dealloc<1>(tmem, C::kCols);
}

template <int kTn, int kSplits>
int launch_few(const Params& p, cudaStream_t st) {
  using C = Few<kTn>;
  CUtensorMap ta, tb;
  if (int rc = make_tmap_2d(&ta, p.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.K, p.M, p.lda, 128, kTn)) return rc;
  if (int rc = make_tmap_2d(&tb, p.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.K, p.N, p.ldb, 128, 128)) return rc;
  constexpr auto kern = gemm_few_kernel<kTn, kSplits>;
  if (int rc = allow_smem<kern>(C::kSmem + 1024)) return rc;
  const int64_t tiles = (int64_t)((p.N + 127) / 128) * ((p.M + kTn - 1) / kTn);
  return launch_cluster(kern, dim3((unsigned)(tiles * kSplits)), dim3(C::kThreads), C::kSmem + 1024, st, kSplits, ta, tb,
                        p);
}
template <int kTn>
int dispatch_few(const Params& p, int splits, cudaStream_t st) {
  switch (splits) {
    case 1: return launch_few<kTn, 1>(p, st);
    case 2: return launch_few<kTn, 2>(p, st);
    case 4: return launch_few<kTn, 4>(p, st);
    default: return launch_few<kTn, 8>(p, st);
  }
}

// The few-token kernel where every tile gets two CTAs or more, or there are at most 256 tokens and its tiles fit on
// the SMs at once.  Measured (us, few against pair, weights in L2): 1 x 4096 x 4096 5.8 / 14.0, 128 x 4096 x 4096 9.6 / 14.7,
// 256 x 4096 x 4096 12.7 / 14.9, 512 x 4096 x 4096 17.4 / 15.9, 1024 x 512 x 1536 12.8 / 10.0.
int dispatch(const Params& p, cudaStream_t st) {
  const int tn = p.M <= 16 ? 16 : p.M <= 32 ? 32 : p.M <= 64 ? 64 : 128;
  const int64_t tiles = (int64_t)((p.N + 127) / 128) * ((p.M + tn - 1) / tn);
  const int sms = sm_count();
  if (2 * tiles > sms && (p.M > 256 || tiles > sms)) return p.c_dtype == DA_F16    ? dispatch_pair<DA_F16>(p, st)
                                                                    : p.c_dtype == DA_BF16 ? dispatch_pair<DA_BF16>(p, st)
                                                                                           : dispatch_pair<DA_F32>(p, st);
  // as many K ranges as fill the SMs, none shorter than 2 stages
  const int nk = (p.K + 127) / 128;
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= sms && nk >= splits * 2 * 2) splits *= 2;
  switch (tn) {
    case 16: return dispatch_few<16>(p, splits, st);
    case 32: return dispatch_few<32>(p, splits, st);
    case 64: return dispatch_few<64>(p, splits, st);
    default: return dispatch_few<128>(p, splits, st);
  }
}

}  // namespace i8
}  // namespace da

extern "C" int da_gemm_i8(const int8_t* A, int64_t lda, const float* a_scale, const int8_t* B, int64_t ldb,
                          const float* b_scale, const void* bias, int bias_dtype, int gelu, void* C, int64_t ldc,
                          int c_dtype, int64_t M, int64_t N, int64_t K, int* status, void* stream) {
  using namespace da;
  if (!A || !B || !a_scale || !b_scale || !C || !status) return DA_ERR_NULL;
  // (the tile count stays an int)
  if (M <= 0 || N <= 0 || K <= 0 || K > i8::kMaxK || M > 0x3fffffffLL || N > 0x3fffffffLL || lda < K || ldb < K ||
      ldc < N || ((M + 255) / 256) * ((N + 255) / 256) > 0x3fffffffLL)
    return DA_ERR_SHAPE;
  if (c_dtype < DA_F16 || c_dtype > DA_F32 || (bias && (bias_dtype < DA_F16 || bias_dtype > DA_F32)))
    return DA_ERR_DTYPE;
  if (lda % 16 || ldb % 16 || reinterpret_cast<uintptr_t>(A) % 16 || reinterpret_cast<uintptr_t>(B) % 16)
    return DA_ERR_ALIGN;
  if (int rc = bind_device(A)) return rc;
  const int elem = c_dtype == DA_F32 ? 4 : 2;
  // A long K loop hides the wait of a turn for its next accumulator, a short one does not.  Measured (us, all warps on
  // every tile against turns): 32768 x 512 x 1536 29.9 / 36.0, with GELU 42.4 / 52.0; 32768 x 768 x 1536 39.2 / 41.1, 45.9
  // / 56.2; 32768 x 1024 x 1536 49.2 / 46.8, 53.0 / 60.1; 32768 x 1536 x 1536 with GELU 72.5 / 71.7; 8192 x 4096 x 4096 93.8
  // / 88.8.
  const int turns = K >= (gelu ? 1536 : 1024);
  // A TMA store writes whole 16-byte words: where a row of C ends inside one, it would write into what lies behind.
  const int tma_c = reinterpret_cast<uintptr_t>(C) % 16 == 0 && ldc * elem % 16 == 0 && N * elem % 16 == 0;
  const i8::Params p{A,      B,      a_scale, b_scale,    bias,    C,    lda,   ldb,   ldc,
                     (int)M, (int)N, (int)K,  bias_dtype, c_dtype, gelu, turns, tma_c, status,
                     Div31((uint32_t)((N + 255) / 256 * 8))};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return i8::dispatch(p, st);
}
