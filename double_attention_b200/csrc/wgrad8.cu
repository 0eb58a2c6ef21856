// Weight gradient of a Linear from the 8-bit checkpoint of its input:
//   dW[n, k] = sum_t dY[t, n] X[t, k],  X[t, k] = q[t, k] 2^e[t, k / 32]
// X is exact in dY's 16-bit dtype (q has 7 bits, the scale is a power of two), so the product runs on 16-bit
// tensor cores with fp32 accumulation and nothing is rounded before the sum.
//
// Persistent CTA pairs: a pair computes a 256 x 256 tile of dW over a range of rows with cta_group::2 instructions;
// each CTA brings its 128 columns of dY (TMA, 64 rows a stage) and 128 columns of q, which 16 warps, 4 a stage, turn
// into X in the tensor core's layout in shared memory.  (Above 768 output columns X is expanded in memory first.)
//
// The tensor core cuts each sum into its accumulator to fp32 instead of rounding it: measured, a chain over 43690
// rows comes out 3.1e-5 low (1.1e-8 for each of its instructions), 70 times the error of a plain fp32 product.  So the
// accumulator (double-buffered in TMEM) is taken over after every 1024 rows and added, rounded, into a second sum
// that the same 16 warps keep in registers, 64 values a thread.
//
// dY whose rows are not on 16-byte words is first copied to rows that are: 50000 rows, 1333 x 1001 in 193 us, 1336 x
// 1000 in 146.
//
// Where there are fewer tiles than pairs the rows are split over pairs and the partial sums added in split order.
//
// Measured: 262144 rows, 1536 x 512 (X expanded in memory first, see plan_for) 387 us, 60 of them the expansion, the
// product at 1.3 PFLOP/s (61 % of the tensor pipe: ~200 cycles a dependent instruction); 8192 rows, 4096 x 4096 243 us,
// 1.13 PFLOP/s; converting in the kernel, 262144 rows, 512 x 1536 417 us and 128 x 512 77 us (2.7 TB/s).  The converting
// form is bound by the latency of its barriers: without the conversion's arithmetic it keeps 88 % of its time.
#include "common.cuh"
#include "host_util.h"
#include "vec8.cuh"

namespace da {
namespace wg8 {

constexpr int kTile = 256;
constexpr int kRows = 64;                     // rows (the sum's index) per stage
constexpr int kStages = 6;                    // dY boxes and converted X tiles
constexpr int kRawStages = 4;                 // q boxes
constexpr int kChunk = 16;                    // stages accumulated in TMEM at a time
constexpr int kHalfTile = kRows * 128 * 2;    // 128 columns of 16 bits
constexpr int kRaw = kRows * 128;
constexpr int kOffX = kStages * kHalfTile;
constexpr int kOffRaw = 2 * kStages * kHalfTile;
constexpr int kSmem = kOffRaw + kRawStages * kRaw;
constexpr int kGroups = 4;                    // conversion groups of 4 warps, each a stage at a time
constexpr int kThreads = 128 + kGroups * 128;  // warps 0, 3 dY; 1 MMA; 2 q; 4-19 conversion and sums

struct Params {
  const int8_t* e;
  void* out;        // dW, or the partial sums where the rows are split
  int64_t ldo;
  int rows, split_rows, N, K, splits, blocks;
  int vec;  // rows of `out` take 16-byte stores
  int* status;
};

// Four bytes of q, as two 16-bit pairs times `unit` (a pair of the block's scale): exact.
template <typename T>
DA_DEV uint2 expand4(uint32_t w, uint32_t unit);
template <>
DA_DEV uint2 expand4<__nv_bfloat16>(uint32_t w, uint32_t unit) {
  // 0x4300 is 128 with a last place of 1: 0x4300 | (q & 127) is 128 + (q & 127), 0x4300 | (q & 128) is 128 or 256,
  // and their difference is q
  const uint32_t lo = __byte_perm(w, 0x43434343u, 0x4140), hi = __byte_perm(w, 0x43434343u, 0x4342);
  auto value = [&](uint32_t t) {
    const uint32_t a = t & 0xff7fff7fu, b = t & 0xff80ff80u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    const __nv_bfloat162 r = __hmul2(d, *reinterpret_cast<const __nv_bfloat162*>(&unit));
    return *reinterpret_cast<const uint32_t*>(&r);
  };
  return make_uint2(value(lo), value(hi));
}
template <>
DA_DEV uint2 expand4<__half>(uint32_t w, uint32_t unit) {
  // 0x6400 is 1024 with a last place of 1: 0x6400 | (q xor 128) is 1024 + 128 + q
  w ^= 0x80808080u;
  const uint32_t lo = __byte_perm(w, 0x64646464u, 0x4140), hi = __byte_perm(w, 0x64646464u, 0x4342);
  auto value = [&](uint32_t t) {
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&t), __half2half2(__ushort_as_half(0x6480)));
    const __half2 r = __hmul2(d, *reinterpret_cast<const __half2*>(&unit));
    return *reinterpret_cast<const uint32_t*>(&r);
  };
  return make_uint2(value(lo), value(hi));
}
// The pair (2^e, 2^e).  The code -128 of a block that was not finite gives an infinity (bf16) or a NaN, which its
// values, all 0, turn into NaN.
template <typename T>
DA_DEV uint32_t unit_pair(int e) {
  uint32_t u;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    u = (uint32_t)(e + 127) << 7;  // -128: 0xff80
  } else {
    u = e >= -14 ? (uint32_t)(e + 15) << 10 : e >= -24 ? 1u << (e + 24) : 0x7fffu;
  }
  return __byte_perm(u, 0, 0x1010);
}

// Partial sums lie as the threads hold them, a row each: [split][tile][CTA of the pair][4 columns][128 rows], so that a
// warp stores 512 bytes at once (row-major, 16 bytes a row, the stores of a split took 4 us).
DA_DEV float4* partial_at(void* base, int tiles, int split, int tile, int rank, int col4, int row) {
  return static_cast<float4*>(base) + ((((int64_t)split * tiles + tile) * 2 + rank) * (kTile / 4) + col4) * 128 + row;
}

// kExpanded: X comes expanded from memory (tx is its map, not q's) and no warp converts.
template <typename T, typename TO, bool kExpanded>
__global__ void __launch_bounds__(kThreads, 1) wgrad_kernel(const __grid_constant__ CUtensorMap ty,
                                                            const __grid_constant__ CUtensorMap tx, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t y_full[kStages], x_full[kStages], empty[kStages], raw_full[kRawStages], raw_empty[kRawStages];
  __shared__ uint64_t acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = (int)(cluster_ctarank() & 1u);
  const int k_tiles = (p.K + kTile - 1) / kTile, n_tiles = (p.N + kTile - 1) / kTile;
  const int items = k_tiles * n_tiles * p.splits, pairs = gridDim.x / 2, pair = blockIdx.x / 2;
  const int my_items = pair < items ? (items - 1 - pair) / pairs + 1 : 0;
  Abort ab{&abort_flag, p.status};

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&y_full[s], 1);
      mbar_init(&x_full[s], 2 * 4);  // one group's 4 warps of both CTAs
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kRawStages; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], 4);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * kGroups * 4);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<2>(&tmem_base, 2 * kTile);
    tmem_relinquish<2>();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  grid_dependency_wait();
  grid_launch_dependents();
  const uint32_t tmem = tmem_base;
  // item -> first column of dY, first column of X, first row, stages of rows
  auto item_at = [&](int i, int& n0, int& k0, int& z, int& t0, int& nt) {
    const int w = pair + i * pairs;
    const int tile = w / p.splits;
    z = w - tile * p.splits;
    n0 = tile / k_tiles * kTile;
    k0 = tile % k_tiles * kTile;
    t0 = z * p.split_rows;
    nt = (min(p.split_rows, p.rows - t0) + kRows - 1) / kRows;
  };

  if ((warp == 0 || warp == 3) && lane == 0) {
    // ---------------------------------------------------------------- dY producers (alternate stages)
    const int pi = warp == 0 ? 0 : 1;
    prefetch_tmap(&ty);
    if (kExpanded) prefetch_tmap(&tx);
    bool ok = true;
    int it = 0, last = -1;
    for (int i = 0; ok && i < my_items; ++i) {
      int n0, k0, z, t0, nt;
      item_at(i, n0, k0, z, t0, nt);
      for (int t = 0; t < nt; ++t, ++it) {
        if ((it & 1) != pi) continue;
        const int s = it % kStages;
        if (!mbar_wait(&empty[s], ((it / kStages) & 1u) ^ 1u, ab, 81)) { ok = false; break; }
        if (rank == 0) mbar_arrive_expect_tx(&y_full[s], (kExpanded ? 4 : 2) * kHalfTile);
        const uint32_t bar = mapa_shared(smem_u32(&y_full[s]), 0);
        uint8_t* dst = smem + s * kHalfTile;
        const int x = n0 + rank * 128, y = t0 + t * kRows;
        tma_load_2d_pair(&ty, bar, dst, x, y);
        tma_load_2d_pair(&ty, bar, dst + kRows * 128, x + 64, y);
        if constexpr (kExpanded) {
          dst += kOffX;
          tma_load_2d_pair(&tx, bar, dst, k0 + rank * 128, y);
          tma_load_2d_pair(&tx, bar, dst + kRows * 128, k0 + rank * 128 + 64, y);
        }
        last = it;
      }
    }
    // after a wait that gave up: this producer's loads in flight (kStages is even, so its stages are its own)
    if (rank == 0 && !ok)
      for (int j = (last - kStages + 1 > 0 ? last - kStages + 1 : 0); j <= last; ++j)
        if ((j & 1) == pi) mbar_wait_drain(&y_full[j % kStages], (j / kStages) & 1u);
  } else if (!kExpanded && warp == 2 && lane == 0) {
    // ---------------------------------------------------------------- q producer
    prefetch_tmap(&tx);
    bool ok = true;
    int it = 0;
    for (int i = 0; ok && i < my_items; ++i) {
      int n0, k0, z, t0, nt;
      item_at(i, n0, k0, z, t0, nt);
      for (int t = 0; t < nt; ++t, ++it) {
        const int s = it % kRawStages;
        if (!mbar_wait(&raw_empty[s], ((it / kRawStages) & 1u) ^ 1u, ab, 82)) { ok = false; break; }
        mbar_arrive_expect_tx(&raw_full[s], kRaw);
        tma_load_2d(&tx, &raw_full[s], smem + kOffRaw + s * kRaw, k0 + rank * 128, t0 + t * kRows);
      }
    }
    for (int j = (it - kRawStages > 0 ? it - kRawStages : 0); !ok && j < it; ++j)
      mbar_wait_drain(&raw_full[j % kRawStages], (j / kRawStages) & 1u);
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---------------------------------------------------------------- MMA issuer (leader)
    const uint32_t idesc = idesc_f16(kTile, kTile, std::is_same<T, __nv_bfloat16>::value, true, true);
    bool ok = true;
    int it = 0, chunk = 0;
    for (int i = 0; ok && i < my_items; ++i) {
      int n0, k0, z, t0, nt;
      item_at(i, n0, k0, z, t0, nt);
      for (int t = 0; t < nt; ++t, ++it) {
        const int s = it % kStages, buf = chunk & 1;
        const uint32_t parity = (it / kStages) & 1u;
        if (t % kChunk == 0 && chunk >= 2 && !mbar_wait(&acc_empty[buf], ((chunk >> 1) - 1) & 1u, ab, 83)) { ok = false; break; }
        if (!mbar_wait(&y_full[s], parity, ab, 84) || (!kExpanded && !mbar_wait(&x_full[s], parity, ab, 85))) { ok = false; break; }
        tc_fence_after();
        const uint32_t sy = smem_u32(smem + s * kHalfTile), sx = smem_u32(smem + kOffX + s * kHalfTile);
#pragma unroll
        for (int k = 0; k < kRows / 16; ++k)
          mma_f16_ss<2>(tmem + buf * kTile, sdesc_sw128(sy + k * 16 * 128, kRows * 128, 1024),
                        sdesc_sw128(sx + k * 16 * 128, kRows * 128, 1024), idesc, (t % kChunk > 0 || k > 0) ? 1u : 0u);
        mma_commit_pair(smem_u32(&empty[s]));
        if (t % kChunk == kChunk - 1 || t == nt - 1) {
          mma_commit_pair(smem_u32(&acc_full[buf]));
          ++chunk;
        }
      }
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- conversion and sums
    // A thread turns 16 columns of rows r, r + 16, r + 32 and r + 48 of its group's stages; of the sum it keeps
    // row (lane of its quadrant of TMEM) x 64 columns.
    const int group = warp / 4 - 1, quad = warp & 3, tid = threadIdx.x % 128;
    const int r = tid / 8, j = tid % 8;
    // the 32 bytes it writes per row are chunks 2 (j % 4) and + 1 of 64-column block j / 4.  Block 1 goes through them
    // in the other order, so that the 8 threads of a row write to all banks at once, and so do odd rows, so that two
    // rows read from all banks at once.
    const int swap = (j / 4) ^ (r & 1);
    const uint32_t src_off = kOffRaw + r * 128 + j * 16 + 8 * swap;
    const uint32_t dst_off = kOffX + (j / 4) * (kRows * 128) + r * 128;
    const uint32_t c0 = ((2 * (j % 4) + swap) ^ (r & 7)) << 4, c1 = ((2 * (j % 4) + (swap ^ 1)) ^ (r & 7)) << 4;
    const uint32_t base = smem_u32(smem);
    const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + group * 64;
    bool ok = true;
    int it = 0, chunk = 0;  // stages and chunks before this item
    for (int i = 0; ok && i < my_items; ++i) {
      int n0, k0, z, t0, nt;
      item_at(i, n0, k0, z, t0, nt);
      float sum[64];
#pragma unroll
      for (int c = 0; c < 64; ++c) sum[c] = 0.f;
      const int block = (k0 + rank * 128) / 32 + j / 2;
      const bool live = block < p.blocks;
      const int8_t* e_at = p.e + (int64_t)(t0 + r) * p.blocks + block;
      const int rows_left = live ? p.rows - t0 - r : 0;
      auto exponents = [&](int t) {  // of the thread's 4 rows of stage t, a byte each
        uint32_t e4 = 0;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int row = t * kRows + 16 * h;
          const int e = row < rows_left ? (int)__ldg(e_at + (int64_t)row * p.blocks) : 0;
          e4 |= (uint32_t)(e & 255) << (8 * h);
        }
        return e4;
      };
      // takes over chunk c of this item: sum += accumulator
      auto take = [&](int c) {
        const int buf = (chunk + c) & 1;
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&acc_full[buf], ((chunk + c) >> 1) & 1u, ab, 88));
        if (!ok) return;
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 64; q += 16) {
          float v[16];
          tmem_ld16(acc + buf * kTile + q, v);
          tmem_wait_ld();
#pragma unroll
          for (int x = 0; x < 16; ++x) sum[q + x] += v[x];
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(&acc_empty[buf]), 0));
      };
      const int chunks = (nt + kChunk - 1) / kChunk;
      int t = (group - it % kGroups + kGroups) % kGroups;  // the group's first stage of this item
      uint32_t e_next = kExpanded ? 0 : exponents(t), e_after = kExpanded ? 0 : exponents(t + kGroups);
      for (int c = 0; ok && c < chunks; ++c) {
        const int t_end = min(nt, (c + 1) * kChunk);
#pragma unroll 1
        for (; !kExpanded && t < t_end; t += kGroups) {
          const uint32_t e4 = e_next;
          e_next = e_after;
          e_after = exponents(t + 2 * kGroups);
          const int at = it + t, s = at % kStages, rs = at % kRawStages;
          ok = __all_sync(0xffffffffu, mbar_wait(&raw_full[rs], (at / kRawStages) & 1u, ab, 86) &&
                                           mbar_wait(&empty[s], ((at / kStages) & 1u) ^ 1u, ab, 87));
          if (!ok) break;
          const uint32_t src = base + src_off + rs * kRaw, dst = base + dst_off + s * kHalfTile;
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const uint2 w0 = ld_shared_v2(src + h * 16 * 128), w1 = ld_shared_v2((src ^ 8) + h * 16 * 128);
            const uint32_t u = unit_pair<T>((int)(int8_t)(e4 >> (8 * h)));
            const uint2 x0 = expand4<T>(w0.x, u), x1 = expand4<T>(w0.y, u);
            st_shared_v4(dst + c0 + h * 16 * 128, x0.x, x0.y, x1.x, x1.y);
            const uint2 x2 = expand4<T>(w1.x, u), x3 = expand4<T>(w1.y, u);
            st_shared_v4(dst + c1 + h * 16 * 128, x2.x, x2.y, x3.x, x3.y);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&raw_empty[rs]);
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&x_full[s]), 0));
        }
        if (ok && c > 0) take(c - 1);  // while the tensor core works on chunk c
      }
      if (ok) take(chunks - 1);
      it += nt;
      chunk += chunks;
      if (!ok) break;
      const int row = n0 + rank * 128 + quad * 32 + lane, col = k0 + group * 64;
      if (row >= p.N || col >= p.K) continue;
      if (p.splits > 1) {
        float4* dst = partial_at(p.out, k_tiles * n_tiles, z, (pair + i * pairs) / p.splits, rank, group * 16,
                                 quad * 32 + lane);
#pragma unroll
        for (int q = 0; q < 64; q += 4)
          if (col + q < p.K) dst[q / 4 * 128] = make_float4(sum[q], sum[q + 1], sum[q + 2], sum[q + 3]);
        continue;
      }
      TO* dst = static_cast<TO*>(p.out) + (int64_t)row * p.ldo + col;
      if (p.vec && col + 64 <= p.K) {
        if constexpr (std::is_same<TO, float>::value) {
#pragma unroll
          for (int q = 0; q < 64; q += 4)
            *reinterpret_cast<float4*>(dst + q) = make_float4(sum[q], sum[q + 1], sum[q + 2], sum[q + 3]);
        } else {
#pragma unroll
          for (int q = 0; q < 64; q += 8)
            *reinterpret_cast<uint4*>(dst + q) =
                make_uint4(pack2<TO>(sum[q], sum[q + 1]), pack2<TO>(sum[q + 2], sum[q + 3]),
                           pack2<TO>(sum[q + 4], sum[q + 5]), pack2<TO>(sum[q + 6], sum[q + 7]));
        }
      } else {
#pragma unroll
        for (int q = 0; q < 64; ++q)
          if (col + q < p.K) {
            if constexpr (std::is_same<TO, float>::value) dst[q] = sum[q];
            else dst[q] = from_f32<TO>(sum[q]);
          }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) tmem_dealloc<2>(tmem, 2 * kTile);
}

// dW = the splits' partial sums.  kWays warps add a range of the splits each for 32 rows x 4 columns, in order, and the first
// adds their sums in order.
template <typename TO, int kWays>
__global__ void __launch_bounds__(256) reduce_kernel(const float* partial, int splits, int k_tiles, int n_tiles, int N,
                                                     int K, TO* out, int64_t ldo) {
  __shared__ float4 part[8][32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, way = warp % kWays;
  const int piece = blockIdx.x * (8 / kWays) + warp / kWays;
  const int quad = piece % 4, col4 = piece / 4 % (kTile / 4), half = piece / kTile;  // half = tile * 2 + rank
  const int tile = half / 2, rank = half % 2;
  const int row = tile / k_tiles * kTile + rank * 128 + quad * 32 + lane, col = tile % k_tiles * kTile + col4 * 4;
  const int per = (splits + kWays - 1) / kWays, z0 = way * per, z1 = min(splits, z0 + per);
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (row < N && col < K) {
    const float4* src = partial_at(const_cast<float*>(partial), k_tiles * n_tiles, 0, tile, rank, col4, quad * 32 + lane);
    const int64_t step = (int64_t)k_tiles * n_tiles * (kTile * kTile / 4);
#pragma unroll 5
    for (int z = z0; z < z1; ++z) {
      const float4 v = src[z * step];
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
  }
  if constexpr (kWays > 1) {
    part[warp][lane] = s;
    __syncthreads();
  }
  if (way > 0 || row >= N || col >= K) return;
#pragma unroll
  for (int w = 1; w < kWays; ++w) {
    const float4 v = part[warp + w][lane];
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  TO* dst = out + row * ldo + col;
  const float v[4] = {s.x, s.y, s.z, s.w};
  if (col + 4 <= K && ldo % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0) {
    if constexpr (std::is_same<TO, float>::value) *reinterpret_cast<float4*>(dst) = s;
    else *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<TO>(s.x, s.y), pack2<TO>(s.z, s.w));
  } else {
    for (int q = 0; q < 4 && col + q < K; ++q) {
      if constexpr (std::is_same<TO, float>::value) dst[q] = v[q];
      else dst[q] = from_f32<TO>(v[q]);
    }
  }
}

// Rows of 16-bit values copied to rows on 16-byte words, which TMA needs: 8 columns a thread and item, from the two
// aligned words that hold them.  `end` is the end of src.  50000 x 1333 in 40 us (6.6 TB/s).
constexpr int kCopies = 4;
__global__ void __launch_bounds__(256) align_rows_kernel(const uint16_t* src, int64_t ld, const uint16_t* end, int items,
                                                         Div31 per_row, int N, uint16_t* dst) {
  grid_dependency_wait();
  grid_launch_dependents();
  uint4 v[kCopies];
#pragma unroll
  for (int k = 0; k < kCopies; ++k) {
    const int i = (blockIdx.x * kCopies + k) * 256 + threadIdx.x;
    if (i >= items) continue;
    const int row = (int)per_row.div((uint32_t)i), col = (i - row * (int)per_row.d) * 8;
    const uint16_t* at = src + row * ld + col;
    const int m = (int)(reinterpret_cast<uintptr_t>(at) / 2 & 7);
    if (at - m >= src && at - m + 16 <= end) {
      v[k] = shift16(*reinterpret_cast<const uint4*>(at - m), *reinterpret_cast<const uint4*>(at - m + 8), m);
    } else {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < N) w[j / 2] |= (uint32_t)at[j] << (j % 2 * 16);
      v[k] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
#pragma unroll
  for (int k = 0; k < kCopies; ++k) {
    const int i = (blockIdx.x * kCopies + k) * 256 + threadIdx.x;
    if (i < items) *reinterpret_cast<uint4*>(dst + (int64_t)i * 8) = v[k];
  }
}
int align_rows(const uint16_t* src, int64_t ld, int64_t rows, int64_t N, uint16_t* dst, cudaStream_t st) {
  const Div31 per_row((uint32_t)((N + 7) / 8));
  const uint16_t* end = src + (rows - 1) * ld + N;
  const int64_t slab = (Div31::kMax - 256 * kCopies) / per_row.d;  // (items and their index stay below 2^31)
  for (int64_t r0 = 0; r0 < rows; r0 += slab) {
    const int64_t items = (rows - r0 < slab ? rows - r0 : slab) * per_row.d;
    if (int rc = launch_kernel(align_rows_kernel, dim3((unsigned)((items + 256 * kCopies - 1) / (256 * kCopies))), dim3(256),
                               0, st, false, src + r0 * ld, ld, end, (int)items, per_row, (int)N,
                               dst + r0 * per_row.d * 8))
      return rc;
  }
  return DA_OK;
}

struct Plan {
  int splits;
  int64_t split_rows;
  bool expanded;
  int64_t x_elems, y_elems, elems;  // workspace (fp32 elements): the expanded X, dY on 16-byte rows, and the partial sums
};
// The rows are split while there are fewer tiles than CTA pairs; a split has at least 256 rows (1000 rows, 512 x 512 in
// 13.5 us; at least 128 12.9, at least 512 15.2; 256 rows 10.3, 12.0 and 10.2).
Plan plan_for(int64_t rows, int64_t N, int64_t K) {
  const int64_t n_tiles = (N + kTile - 1) / kTile, tiles = n_tiles * ((K + kTile - 1) / kTile);
  int64_t s = (sm_count() / 2) / tiles;
  const int64_t most = (rows + 255) / 256;
  if (s > most) s = most;
  if (s < 1) s = 1;
  Plan p;
  p.split_rows = (rows + s * kRows - 1) / (s * kRows) * kRows;
  p.splits = (int)((rows + p.split_rows - 1) / p.split_rows);
  // Expanding X into memory first costs 3 bytes of traffic a value and saves every row of tiles its conversion.
  // Measured (us, converting in the kernel against expanding first): 262144 rows, 1536 x 512 429 / 386 and
  // 512 x 1536 423 / 498; 8192 rows, 4096 x 4096 343 / 243; 16384 rows, 640 x 2000 69 / 64.
  p.expanded = N > 3 * kTile;
  p.x_elems = p.expanded ? (rows * ((K + 31) / 32 * 16) + 63) / 64 * 64 : 0;
  p.y_elems = N % 8 ? (rows * ((N + 7) / 8 * 4) + 63) / 64 * 64 : 0;
  p.elems = p.x_elems + p.y_elems + (p.splits > 1 ? p.splits * tiles * kTile * kTile : 0);
  return p;
}

template <typename T, typename TO, bool kExpanded>
int launch(const CUtensorMap& ty, const CUtensorMap& tx, const Params& p, cudaStream_t st) {
  constexpr auto kern = wgrad_kernel<T, TO, kExpanded>;
  if (int rc = allow_smem<kern>(kSmem + 1024)) return rc;
  const int64_t items = (int64_t)((p.N + kTile - 1) / kTile) * ((p.K + kTile - 1) / kTile) * p.splits;
  const int pairs = items < sm_count() / 2 ? (int)items : sm_count() / 2;
  return launch_kernel(kern, dim3(2 * pairs), dim3(kThreads), kSmem + 1024, st, true, ty, tx, p);
}

// The product of one 16-bit type, and the sum of the splits.
template <typename T>
int run(const void* dy, int64_t ldy, const int8_t* q, const int8_t* e, int64_t rows, int64_t N, int64_t K, void* out,
        int out_dtype, int64_t ldo, float* workspace, const Plan& plan, int* status, cudaStream_t st) {
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr CUtensorMapDataType dt = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int64_t blocks = (K + 31) / 32;
  const bool split = plan.splits > 1;
  float* partial = workspace + plan.x_elems + plan.y_elems;
  CUtensorMap ty, tx;
  if (ldy % 8 || reinterpret_cast<uintptr_t>(dy) % 16) {
    uint16_t* aligned = reinterpret_cast<uint16_t*>(workspace + plan.x_elems);
    if (int rc = align_rows(static_cast<const uint16_t*>(dy), ldy, rows, N, aligned, st)) return rc;
    dy = aligned;
    ldy = (N + 7) / 8 * 8;
  }
  if (int rc = make_tmap_2d(&ty, dy, dt, 2, N, rows, (uint64_t)ldy * 2, 64, kRows)) return rc;
  if (plan.expanded) {
    if (int rc = da_checkpoint8_restore(q, e, rows, blocks * 32, workspace, bf16 ? DA_BF16 : DA_F16, blocks * 32, st))
      return rc;
    if (int rc = make_tmap_2d(&tx, workspace, dt, 2, blocks * 32, rows, blocks * 64, 64, kRows)) return rc;
  } else {
    if (int rc = make_tmap_2d(&tx, q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, blocks * 32, rows, blocks * 32, 128, kRows, false))
      return rc;
  }
  const int vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && ldo * (out_dtype == DA_F32 ? 4 : 2) % 16 == 0;
  const Params p{e,      split ? partial : out, ldo,         (int)rows,   (int)plan.split_rows,
                 (int)N, (int)K,                plan.splits, (int)blocks, vec,
                 status};
  int rc;
  if (split || out_dtype == DA_F32)
    rc = plan.expanded ? launch<T, float, true>(ty, tx, p, st) : launch<T, float, false>(ty, tx, p, st);
  else
    rc = plan.expanded ? launch<T, T, true>(ty, tx, p, st) : launch<T, T, false>(ty, tx, p, st);
  if (rc || !split) return rc;
  const int k_tiles = (int)((K + kTile - 1) / kTile), n_tiles = (int)((N + kTile - 1) / kTile);
  // Measured (us, 2 / 8 warps a piece): 9 splits of 392 x 1000 17.2 / 19.8, 6 of 1536 x 512 15.9 / 19.7, 16 of 512 x 512
  // 14.8 / 15.0, 37 of 128 x 384 18.8 / 15.3, 74 of 128 x 128 25.7 / 19.4.
  auto sum = [&](auto* to) {
    using TO = std::remove_pointer_t<decltype(to)>;
    const unsigned pieces = (unsigned)(k_tiles * n_tiles * 2 * kTile);
    const bool few = plan.splits <= 16;
    return launch_kernel(few ? reduce_kernel<TO, 2> : reduce_kernel<TO, 8>, dim3(few ? pieces / 4 : pieces), dim3(256), 0, st,
                         false, (const float*)partial, plan.splits, k_tiles, n_tiles, (int)N, (int)K, to, ldo);
  };
  return out_dtype == DA_F32 ? sum(static_cast<float*>(out)) : sum(static_cast<T*>(out));
}

}  // namespace wg8
}  // namespace da

extern "C" int64_t da_checkpoint8_wgrad_workspace_elems(int64_t rows, int64_t N, int64_t K) {
  if (rows <= 0 || N <= 0 || K <= 0) return -1;
  return da::wg8::plan_for(rows, N, K).elems;
}

extern "C" int da_checkpoint8_wgrad(const void* dy, int dtype, int64_t ldy, const int8_t* q, const int8_t* e,
                                    int64_t rows, int64_t N, int64_t K, void* out, int out_dtype, int64_t ldo,
                                    float* workspace, int64_t workspace_elems, int* status, void* stream) {
  using namespace da;
  if (!dy || !q || !e || !out || !status) return DA_ERR_NULL;
  if (rows <= 0 || rows > 0x7fff0000LL || N <= 0 || K <= 0 || N > 0x3fffffLL || K > 0x3fffffLL || ldy < N || ldo < K)
    return DA_ERR_SHAPE;
  if ((dtype != DA_F16 && dtype != DA_BF16) || (out_dtype != DA_F32 && out_dtype != dtype)) return DA_ERR_DTYPE;
  if (N % 8 == 0 && (ldy % 8 || reinterpret_cast<uintptr_t>(dy) % 16)) return DA_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(dy) % 2 || reinterpret_cast<uintptr_t>(q) % 16) return DA_ERR_ALIGN;
  const wg8::Plan plan = wg8::plan_for(rows, N, K);
  if (plan.elems && (!workspace || workspace_elems < plan.elems)) return DA_ERR_WORKSPACE;
  if (plan.elems && reinterpret_cast<uintptr_t>(workspace) % 256) return DA_ERR_ALIGN;
  if (int rc = bind_device(dy)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == DA_BF16 ? wg8::run<__nv_bfloat16>(dy, ldy, q, e, rows, N, K, out, out_dtype, ldo, workspace, plan, status, st)
                          : wg8::run<__half>(dy, ldy, q, e, rows, N, K, out, out_dtype, ldo, workspace, plan, status, st);
}
