// Outer routed attention of long chunks of new tokens over a paged cache.
//
// The same product as paged_attn.cu's, for sequences that bring many tokens: 128 query tokens a CTA pair, scores and
// P V on paired tensor-core instructions into TMEM, laid out as attn_fwd.cu's (attn_layout.cuh).  What differs:
//   * keys and values come page by page through the table, boxes of a page's positions (up to the tile's); positions
//     that the sequence does not have are fetched past the end of the cache, where TMA fills in zeros;
//   * the softmax offset is each row's own maximum, whatever the keys' lengths.  One map: a running maximum, against
//     which outputs in TMEM are rescaled only when it has grown by more than 2^8 (they are fp32, the weights at most 2^8);
//     several maps: a first launch over the keys leaves each map's maximum and sum, a second builds the mixture
//     P = sum_s alpha_s softmax_s and needs one P V for all maps;
//   * the (query tile, key range) pieces are planned on the device from the lengths: equal key ranges of all tiles, so
//     that few or uneven tiles fill the GPU; join_kernel adds the pieces of a tile in order.
// A value behind a row's last position weighs 0, and 0 times a NaN or an infinity is NaN: such rows are found when they
// are written and computed again by the other kernel, which tells them apart.
#include <math.h>

#include "attn_layout.cuh"
#include "host_util.h"
#include "paged_chunk.h"

namespace da {
namespace paged {

using attn::kMaxK;
using attn::kMaxMaps;
using attn::kMaxPB;
using attn::kMaxSB;
using attn::kMaxV;
using attn::kRows;
using attn::Layout;

constexpr int kThreads = 320;  // warp roles as in attn_fwd.cu
constexpr int kValueWarp = 6, kPvWarp = 7, kKeyWarp2 = 8, kValueWarp2 = 9;
constexpr int kSmem = 224 * 1024;
constexpr float kGrow = 8.f;  // log2 of the growth of a row's maximum that its outputs bear

struct ChunkParams {
  Cache c;
  Plan plan;
  int H, R, D, maps, group, dtype;
  int branch0[kMaxMaps];
  int brow_k, brow_v;  // positions a box of keys, of values
  int phase;           // several maps: 1 sums, 2 outputs; one map: 0
  const float *scales, *weights;
  void* y;
  int64_t y_row;       // elements from row to row
  float* part;         // [pieces][128][D]
  float* part_ml;      // [pieces][2][128]: one map's maximum (log2) and sum
  float* stats;        // [pieces][2][maps][128]: phase 1's
  int few_most;
  int* status;
};

// Positions that some row of tile i sees.
DA_DEV int64_t tile_end(const Cache& c, const Sequence& s, int i) {
  const int64_t e = s.held + min(s.n, (i + 1) * 128);
  return e < c.capacity ? e : c.capacity;
}

// ------------------------------------------------------------------------------------------------ plan
constexpr int kPlanThreads = 1024, kLengths = 10;

// One CTA: a warp a sequence, a tile a lane.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const Cache c, const Plan plan, int few_most, int nk_shift, int pairs) {
  __shared__ int2 kept[kPlanThreads];  // the first sequences' new tokens (of chunks), and tokens that they had
  __shared__ unsigned long long units;
  __shared__ int counts[kLengths], carry[2], sums[2][32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  auto load = [&](int b) {
    const Sequence s = sequence(c, b);
    return make_int2(s.n > few_most ? s.n : 0, (int)s.held);
  };
  if (threadIdx.x < c.B) kept[threadIdx.x] = load(threadIdx.x);
  if (threadIdx.x < kLengths) counts[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    units = 0;
    carry[0] = carry[1] = 0;
  }
  __syncthreads();
  auto get = [&](int b) { return b < kPlanThreads ? kept[b] : load(b); };
  auto tiles_of = [](int2 s) { return (s.x + 127) >> 7; };
  auto keys_of = [&](int2 s, int i) {  // key tiles of query tile i
    const int64_t e = (int64_t)s.y + min(s.x, (i + 1) * 128);
    return (int)(((e < c.capacity ? e : c.capacity) + (1 << nk_shift) - 1) >> nk_shift);
  };
  unsigned long long mine = 0;
  for (int b = warp; b < c.B; b += kPlanThreads / 32) {
    const int2 s = get(b);
    for (int i = lane; i < tiles_of(s); i += 32) mine += keys_of(s, i);
  }
  if (mine) atomicAdd(&units, mine);
  __syncthreads();
  // The pieces' length: of a few that suit one or two rounds of the CTA pairs, the one that is done first, counting a
  // piece's start and end as two key tiles.
  const int64_t total = (int64_t)units;
  auto length = [&](int f) {
    const int64_t round = (int64_t)pairs * (f < 5 ? 1 : 2), base = (total + round - 1) / round;
    const int64_t more = f % 5 == 0 ? 0 : (base + (16 >> (f % 5 - 1)) - 1) / (16 >> (f % 5 - 1));  // none, a 16th, 8th, 4th, half
    const int64_t len = base + more;
    return (int)(len < 1 ? 1 : len);
  };
  int len[kLengths], n[kLengths];
#pragma unroll
  for (int f = 0; f < kLengths; ++f) {
    len[f] = length(f);
    n[f] = 0;
  }
  for (int b = warp; b < c.B; b += kPlanThreads / 32) {
    const int2 s = get(b);
    for (int i = lane; i < tiles_of(s); i += 32) {
      const int t = keys_of(s, i);
#pragma unroll
      for (int f = 0; f < kLengths; ++f) n[f] += (unsigned)(t + len[f] - 1) / (unsigned)len[f];
    }
  }
#pragma unroll
  for (int f = 0; f < kLengths; ++f) {
    n[f] = __reduce_add_sync(0xffffffffu, n[f]);
    if (lane == 0 && n[f]) atomicAdd(&counts[f], n[f]);
  }
  __syncthreads();
  int best = 1;
  int64_t best_cost = INT64_MAX;
#pragma unroll
  for (int f = 0; f < kLengths; ++f) {
    const int64_t cost = (int64_t)((counts[f] + pairs - 1) / pairs) * (len[f] + 2);
    if (cost < best_cost) {
      best_cost = cost;
      best = len[f];
    }
  }
  // tiles and pieces in order: 32 sequences a turn, one a warp
  for (int base = 0; base < c.B; base += 32) {
    const int b = base + warp;
    const int2 s = b < c.B ? get(b) : make_int2(0, 0);
    const int tiles = tiles_of(s);
    int count = 0;
    for (int i = lane; i < tiles; i += 32) count += (unsigned)(keys_of(s, i) + best - 1) / (unsigned)best;
    count = __reduce_add_sync(0xffffffffu, count);
    if (lane == 0) {
      sums[0][warp] = tiles;
      sums[1][warp] = count;
    }
    __syncthreads();
    const int t = sums[0][lane], k = sums[1][lane];
    int tile0 = carry[0] + __reduce_add_sync(0xffffffffu, lane < warp ? t : 0);
    int piece0 = carry[1] + __reduce_add_sync(0xffffffffu, lane < warp ? k : 0);
    __syncthreads();
    if (threadIdx.x == kPlanThreads - 1) {
      carry[0] = tile0 + tiles;
      carry[1] = piece0 + count;
    }
    if (b < c.B && lane == 0) plan.seq_piece[b] = piece0;
    for (int i0 = 0; i0 < tiles; i0 += 32) {
      const int i = i0 + lane, keys = i < tiles ? keys_of(s, i) : 0, own = (unsigned)(keys + best - 1) / (unsigned)best;
      int at = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += u;
      }
      const int all = __shfl_sync(0xffffffffu, at, 31), first = piece0 + at - own;
      if (i < tiles) plan.tile_piece[tile0 + i] = first;
      // (a tile's pieces side by side: the warp writes one tile after another, a piece a lane)
      for (int j = 0; j < min(32, tiles - i0); ++j) {
        const int from = __shfl_sync(0xffffffffu, first, j), many = __shfl_sync(0xffffffffu, own, j);
        const int last = __shfl_sync(0xffffffffu, keys, j);
        for (int m = lane; m < many; m += 32) {
          plan.pieces[2 * (from + m)] = make_int4(b, i0 + j, m * best, min(best, last - m * best));
          plan.pieces[2 * (from + m) + 1] = make_int4(from, many, 0, 0);
          *reinterpret_cast<int2*>(plan.odd + 2 * (from + m)) = make_int2(0, 0);
        }
      }
      piece0 += all;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    plan.seq_piece[c.B] = carry[1];
    plan.tile_piece[carry[0]] = carry[1];
    *reinterpret_cast<int4*>(plan.head) = make_int4(carry[1], carry[0], 0, 0);
  }
}

// ------------------------------------------------------------------------------------------------ attention
template <typename T, bool kMix>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(const __grid_constant__ CUtensorMap tq,
                                                            const __grid_constant__ CUtensorMap tk,
                                                            const __grid_constant__ CUtensorMap tv, const ChunkParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t q_full, o_full;
  __shared__ uint64_t k_full[kMaxK], k_empty[kMaxK], v_full[kMaxV], v_empty[kMaxV];
  __shared__ uint64_t s_full[kMaxSB], p_full[kMaxSB], p_empty[kMaxPB], pv_full[kMaxPB];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag, bad_flag;
  __shared__ float top[2][128];  // the two halves of a row tell each other their maxima

  grid_dependency_wait();  // the plan and the appended tokens are visible from here on
  grid_launch_dependents();
  const int piece = blockIdx.x / 2;
  if (piece >= p.plan.head[0]) return;
  const Layout L = attn::make_layout(p.maps, p.group, p.R, p.D, kMix, true, kSmem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank() & 1u;
  const int4 here = p.plan.pieces[2 * piece], tile = p.plan.pieces[2 * piece + 1];
  const Sequence seq = sequence(p.c, here.x);
  const int64_t end = tile_end(p.c, seq, here.y);
  const int t0 = here.y * 128;  // first token of the tile in its sequence
  const int nk = L.nk, nj = here.w;
  const int maps = kMix ? p.maps : 1;
  // (the pieces that run side by side start at different tiles of their ranges: any order gives the same rows)
  const int rot = piece % nj;
  auto ktile = [&](int j) { return here.z + (j + rot) % nj; };
  const bool outputs = !kMix || p.phase == 2;
  const int U = nj * maps;               // score units: (key tile, map)
  const int nv = outputs ? nj : 0;       // P.V key tiles
  Abort ab{&abort_flag, p.status};
  const int* table = p.c.table + here.x * p.c.table_stride;
  const int outside = p.c.pages << p.c.page_shift;  // a slot past the cache: zeros
  auto slot_of = [&](int64_t pos) -> int {
    if (pos >= end) return outside;
    const int page = table[pos >> p.c.page_shift];
    if (page < 0 || page >= p.c.pages) {
      *reinterpret_cast<volatile int*>(&bad_flag) = 1;
      return outside;
    }
    return (page << p.c.page_shift) + (int)(pos & (p.c.page - 1));
  };

  if (threadIdx.x == 0) {
    abort_flag = bad_flag = 0;
    mbar_init(&q_full, 1);
    mbar_init(&o_full, 1);
    for (int i = 0; i < kMaxK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < kMaxV; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < kMaxSB; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 2);
    }
    for (int i = 0; i < kMaxPB; ++i) {
      mbar_init(&p_empty[i], 1);
      mbar_init(&pv_full[i], 2);  // a probability tile is complete in both CTAs
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<2>(&tmem_base, L.tmem_cols);
    tmem_relinquish<2>();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  if (warp == 0 || warp == kKeyWarp2) {
    // ---------------------------------------------------------------- key producers (both CTAs): warp 0
    // takes the even key stages (and loads q), warp 8 the odd ones
    if (lane == 0) {
      const int pi = warp == 0 ? 0 : 1;
      prefetch_tmap(&tk);
      if (pi == 0) {
        prefetch_tmap(&tq);
        if (rank == 0) mbar_arrive_expect_tx(&q_full, 2 * L.q_bytes);
        const uint32_t qf = mapa_shared(smem_u32(&q_full), 0);
        const int row = (int)(seq.first + t0 + 64 * (int)rank);  // (rows past the last token are zeros)
        for (int s = 0; s < maps; ++s)
          for (int gi = 0; gi < p.group; ++gi)
            for (int kb = 0; kb < L.rpb; ++kb)
              tma_load_4d_pair(&tq, qf, smem + L.off_q + ((s * p.group + gi) * L.rpb + kb) * (kRows * 128), 0, row,
                               p.branch0[s] + gi, kb);
      }
      int kx = 0;  // key stages of both producers
      const int stage_bytes = L.kbb * L.k_stage, half = nk / 2;
      const int wide = p.brow_k == half ? L.kbb : 1;  // column blocks a box
      for (int u = 0; u < U; ++u) {
        const int j = u / maps, s = u % maps;
        bool ok = true;
        for (int c = 0; c < L.kchunks; c += L.kbb, ++kx) {
          if (kx % 2 != pi) continue;
          const int st = kx % L.kslots;
          if (!mbar_wait(&k_empty[st], ((kx / L.kslots) & 1u) ^ 1u, ab, 71)) { ok = false; break; }
          if (rank == 0) mbar_arrive_expect_tx(&k_full[st], 2 * stage_bytes);
          const uint32_t kf = mapa_shared(smem_u32(&k_full[st]), 0);
          const int gi = c / L.rpb, kb = c % L.rpb;  // kbb divides rpb: a stage never spans two branches
          const int block = (p.branch0[s] + gi) * L.rpb + kb;
          const int64_t pos = (int64_t)ktile(j) * nk + (int)rank * half;
          for (int r0 = 0; r0 < half; r0 += p.brow_k) {
            const int slot = slot_of(pos + r0);
            for (int e = 0; e < L.kbb; e += wide)
              tma_load_3d_pair(&tk, kf, smem + L.off_k + st * stage_bytes + e * L.k_stage + r0 * 128, 0, slot, block + e);
          }
        }
        if (!ok) break;
      }
      if (rank == 0) {  // drain: none of this producer's loads may be in flight at teardown
        if (pi == 0) mbar_wait_drain(&q_full, 0);
        for (int c = (kx > L.kslots ? kx - L.kslots : 0); c < kx; ++c)
          if (c % 2 == pi) mbar_wait_drain(&k_full[c % L.kslots], (c / L.kslots) & 1u);
      }
    }
  } else if (warp == kValueWarp || warp == kValueWarp2) {
    // ---------------------------------------------------------------- value producers: warp 6 even
    // stages, warp 9 odd ones
    int vc = 0;
    const int pi = warp == kValueWarp ? 0 : 1;
    if (lane == 0) {
      prefetch_tmap(&tv);
      for (int v = 0; v < nv; ++v) {
        bool ok = true;
        for (int c = 0; c < nk / 64; ++c, ++vc) {
          if (vc % 2 != pi) continue;
          const int st = vc % L.nvs;
          if (!mbar_wait(&v_empty[st], ((vc / L.nvs) & 1u) ^ 1u, ab, 72)) { ok = false; break; }
          if (rank == 0) mbar_arrive_expect_tx(&v_full[st], 2 * L.v_stage);
          const uint32_t vf = mapa_shared(smem_u32(&v_full[st]), 0);
          const int64_t pos = (int64_t)ktile(v) * nk + c * 64;
          uint8_t* dst = smem + L.off_v + st * L.v_stage;
          for (int r0 = 0; r0 < 64; r0 += p.brow_v) {
            const int slot = slot_of(pos + r0);
            if (p.brow_v == 64) {  // one box: this CTA's per column blocks of each of the npv value groups
              tma_load_4d_pair(&tv, vf, dst, 0, slot, (int)rank * L.per, 0);
            } else {
              for (int i = 0; i < L.npv; ++i)
                for (int e = 0; e < L.per; ++e)
                  tma_load_4d_pair(&tv, vf, dst + ((i * L.per + e) * 64 + r0) * 128, 0, slot, (int)rank * L.per + e, i);
            }
          }
        }
        if (!ok) break;
      }
    }
    __syncwarp();
    if (outputs) named_bar_sync(2, 192);  // bad_flag is final
    if (lane == 0 && rank == 0)
      for (int c = (vc > L.nvs ? vc - L.nvs : 0); c < vc; ++c)
        if (c % 2 == pi) mbar_wait_drain(&v_full[c % L.nvs], (c / L.nvs) & 1u);
  } else if (warp == 1 || warp == kPvWarp) {
    // ---------------------------------------------------------------- MMA issuers (leader): scores on warp 1,
    // P.V on warp 7
    if (rank == 0 && lane == 0) {
      constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
      const uint32_t idesc_s = idesc_f16(128, nk, bf16, false, false);
      const uint32_t idesc_o = idesc_f16(128, L.nc, bf16, false, true);  // B = V, MN-major
      const uint32_t qa = smem_u32(smem + L.off_q);
      bool ok = mbar_wait(&q_full, 0, ab, 73);
      tc_fence_after();
      if (warp == 1) {
        // S units in order; a score buffer is reused once the softmax has consumed its previous unit.
        int kx = 0, st = 0;  // key stages consumed, current slot
        for (int u = 0; ok && u < U; ++u) {
          const int sb = u % L.nsb, s = u % maps;
          if (u >= L.nsb && !mbar_wait(&p_full[sb], ((u - L.nsb) / L.nsb) & 1u, ab, 74)) { ok = false; break; }
          const uint32_t d = tmem + L.tmem_s + (uint32_t)(sb * L.s_cols);
          for (int c = 0; ok && c < L.kchunks; ++c) {
            const int cib = c % L.kbb;  // chunk inside the current stage
            if (cib == 0) {
              st = kx % L.kslots;
              if (!mbar_wait(&k_full[st], (kx / L.kslots) & 1u, ab, 75)) { ok = false; break; }
              tc_fence_after();
            }
            const uint64_t ad0 = sdesc_sw128(qa + (s * L.kchunks + c) * (kRows * 128), 16, 1024);
            const uint64_t bd0 =
                sdesc_sw128(smem_u32(smem + L.off_k + (st * L.kbb + cib) * L.k_stage), 16, 1024);
#pragma unroll
            for (int kin = 0; kin < 4; ++kin)  // +32 B per K step of 16 = +2 in the encoded address
              mma_f16_ss<2>(d, ad0 + 2 * kin, bd0 + 2 * kin, idesc_s, (c | kin) ? 1u : 0u);
            if (cib == L.kbb - 1) {
              mma_commit_pair(smem_u32(&k_empty[st]));
              ++kx;
            }
          }
          if (!ok) break;
          mma_commit_pair(smem_u32(&s_full[sb]));
        }
        if (!outputs) {
          mma_commit_pair(smem_u32(&o_full));
          mbar_wait_drain(&o_full, 0);  // every score product has completed
        }
      } else if (outputs) {
        // P.V per key tile, as soon as its probability tile and value rows are in shared memory.
        int vc = 0;
        for (int v = 0; ok && v < nv; ++v) {
          const int pb = v % L.npb;
          if (!mbar_wait(&pv_full[pb], (v / L.npb) & 1u, ab, 76)) { ok = false; break; }
          tc_fence_after();
          const uint32_t pa = smem_u32(smem + L.off_p + pb * L.p_bytes);
          for (int c = 0; ok && c < nk / 64; ++c, ++vc) {
            const int st = vc % L.nvs;
            if (!mbar_wait(&v_full[st], (vc / L.nvs) & 1u, ab, 77)) { ok = false; break; }
            tc_fence_after();
            const uint32_t va = smem_u32(smem + L.off_v + st * L.v_stage);
            // MN-major V: rows are keys (K), 128 B = 64 value columns (N);
            // LBO = distance between 64-column boxes, SBO = 8 key rows.
            const uint64_t ad0 = sdesc_sw128(pa + c * (kRows * 128), 16, 1024);
            const uint64_t bd0 = sdesc_sw128(va, 64 * 128, 1024), bd1 = sdesc_sw128(va + L.per * (64 * 128), 64 * 128, 1024);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {  // K step of 16 keys: A +32 B (+2), B +16 rows x 128 B (+128)
              mma_f16_ss<2>(tmem, ad0 + 2 * kk, bd0 + 128 * kk, idesc_o, (v | c | kk) ? 1u : 0u);
              if (L.npv == 2)  // the two groups' products in turn: neither waits for its own last one
                mma_f16_ss<2>(tmem + (uint32_t)(L.nc / 2), ad0 + 2 * kk, bd1 + 128 * kk, idesc_o, (v | c | kk) ? 1u : 0u);
            }
            mma_commit_pair(smem_u32(&v_empty[st]));
          }
          if (!ok) break;
          mma_commit_pair(smem_u32(&p_empty[pb]));
        }
        mma_commit_pair(smem_u32(&o_full));
        mbar_wait_drain(&o_full, 0);  // every P.V product (and so every score product) has completed
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax + epilogue (warps 2 to 5)
    const int quad = warp & 3;
    const int l = quad * 32 + lane;
    const int r = l & 63, half = l >> 6;
    const int trow = 64 * (int)rank + r;  // row of the tile
    const int t = t0 + trow;              // token of the sequence
    const bool live = t < seq.n;
    const int64_t sees = min(seq.held + t + 1, end);
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    const uint32_t pf_leader = mapa_shared(smem_u32(&p_full[0]), 0);
    const uint32_t pv_leader = mapa_shared(smem_u32(&pv_full[0]), 0);
    const bool arriver = (warp == 2 && lane == 0);
    const float kLog2e = 1.4426950408889634f;
    const int hc = nk / 2;  // key columns per thread per tile
    float scale2[kMaxMaps];
#pragma unroll
    for (int s = 0; s < kMaxMaps; ++s) scale2[s] = s < maps ? p.scales[s] * rsqrtf((float)p.group) * kLog2e : 0.f;
    bool ok = true;

    // Number of visible keys among the 32 columns starting at position k0.
    auto key_limit = [&](int64_t k0) -> int { return (int)clamp64(sees - k0, 0, 32); };
    // pb >= 0: this unit completed probability tile buffer pb
    auto finish_unit = [&](int u, int pb) {
      if (pb >= 0) fence_proxy_async();
      tc_fence_before();
      named_bar_sync(1, 128);
      if (arriver) {
        mbar_arrive_cluster_relaxed(pf_leader + (u % L.nsb) * 8);  // score buffer read
        if (pb >= 0) mbar_arrive_remote(pv_leader + pb * 8);         // probability tile written
      }
    };
    // One thread's 32 weights of a tile, columns half * hc + ch * 32 and on.
    auto store_weights = [&](uint32_t pa, int ch, const float* e) {
      const int kc = half * hc + ch * 32;
      const uint32_t box = pa + (kc >> 6) * (kRows * 128);
      const int cb = (kc & 63) >> 3;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        st_shared_v4(box + sw128_offset(r, cb + i), pack2<T>(e[8 * i], e[8 * i + 1]), pack2<T>(e[8 * i + 2], e[8 * i + 3]),
                     pack2<T>(e[8 * i + 4], e[8 * i + 5]), pack2<T>(e[8 * i + 6], e[8 * i + 7]));
    };

    float factor = 1.f;              // of the outputs in TMEM
    float ref = -INFINITY, sum = 0.f;  // one map: offset of the weights, this half's sum
    if constexpr (kMix) {
      if (p.phase == 1) {
        // ---- each map's maximum and sum of its weights against it
        float mx[kMaxMaps], sm[kMaxMaps];
#pragma unroll
        for (int s = 0; s < kMaxMaps; ++s) {
          mx[s] = -INFINITY;
          sm[s] = 0.f;
        }
        for (int u = 0; u < U; ++u) {
          const int j = u / maps, s = u % maps, sb = u % L.nsb;
          if (ok) ok = mbar_wait(&s_full[sb], (u / L.nsb) & 1u, ab, 78);
          ok = __all_sync(0xffffffffu, ok);
          if (ok) {
            tc_fence_after();
            float m = mx[s], a = sm[s];
            const float sc = scale2[s];
            for (int ch = 0; ch < hc / 32; ++ch) {
              float v[32];
              tmem_ld32(tmem + lane_base + L.tmem_s + (uint32_t)(sb * L.s_cols + ch * 32), v);
              tmem_wait_ld();
              const int lim = key_limit((int64_t)ktile(j) * nk + half * hc + ch * 32);
              float big = -INFINITY;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                v[i] = i < lim ? v[i] * sc : -INFINITY;
                big = fmaxf(big, v[i]);
              }
              const float next = fmaxf(m, big), at = next == -INFINITY ? 0.f : next;
              a *= m == -INFINITY ? 1.f : ex2(m - at);  // (a is 0 then, or NaN)
              m = next;
#pragma unroll
              for (int i = 0; i < 32; ++i) a += ex2(v[i] - at);
            }
            mx[s] = m;
            sm[s] = a;
          }
          finish_unit(u, -1);
        }
        for (int s = 0; s < maps; ++s) {
          top[0][l] = mx[s];
          top[1][l] = sm[s];
          named_bar_sync(1, 128);
          const float m1 = top[0][l ^ 64], a1 = top[1][l ^ 64], m = fmaxf(mx[s], m1), at = m == -INFINITY ? 0.f : m;
          const float a = sm[s] * (mx[s] == -INFINITY ? 1.f : ex2(mx[s] - at)) + a1 * (m1 == -INFINITY ? 1.f : ex2(m1 - at));
          if (half == 0) {
            float* dst = p.stats + ((size_t)piece * 2 * maps + s) * 128 + trow;
            dst[0] = m;
            dst[(size_t)maps * 128] = ok ? a : NAN;
          }
          named_bar_sync(1, 128);
        }
      } else {
        // ---- the pieces' sums of this row; offsets so that the mixture's largest weight is near 1
        float off2[kMaxMaps], al[kMaxMaps], shift = -INFINITY;
#pragma unroll
        for (int s = 0; s < kMaxMaps; ++s) {
          off2[s] = al[s] = 0.f;
          if (s < maps) {
            const float* src = p.stats + ((size_t)tile.x * 2 * maps + s) * 128 + trow;
            const size_t next = (size_t)2 * maps * 128;
            float m = -INFINITY, a = 0.f;
            for (int i = 0; i < tile.y; ++i) m = fmaxf(m, src[i * next]);
            const float at = m == -INFINITY ? 0.f : m;
            for (int i = 0; i < tile.y; ++i) {
              const float mi = src[i * next], ai = src[i * next + (size_t)maps * 128];
              a += ai * (mi == -INFINITY ? 1.f : ex2(mi - at));
            }
            al[s] = p.weights ? p.weights[s] : 1.f;
            off2[s] = m + log2f(a);
            shift = fmaxf(shift, log2f(fabsf(al[s])) - log2f(a));
          }
        }
        shift = fminf(fmaxf(shift, -100.f), 100.f);
        factor = ex2(shift);
        float pm[64];
        for (int v = 0; v < nv; ++v) {
          const int pb = v % L.npb;
          const uint32_t pa = smem_u32(smem + L.off_p + pb * L.p_bytes);
          for (int s = 0; s < maps; ++s) {
            const int u = v * maps + s, sb = u % L.nsb;
            if (ok) ok = mbar_wait(&s_full[sb], (u / L.nsb) & 1u, ab, 78);
            if (ok && s == 0 && v >= L.npb) ok = mbar_wait(&p_empty[pb], ((v - L.npb) / L.npb) & 1u, ab, 79);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
              tc_fence_after();
              const float sc = scale2[s], off = off2[s] + shift, w = al[s];
              for (int ch = 0; ch < hc / 32; ++ch) {
                float sv[32];
                tmem_ld32(tmem + lane_base + L.tmem_s + (uint32_t)(sb * L.s_cols + ch * 32), sv);
                tmem_wait_ld();
                const int lim = key_limit((int64_t)ktile(v) * nk + half * hc + ch * 32);
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                  const float e = i < lim ? w * ex2(sv[i] * sc - off) : 0.f;
                  pm[ch * 32 + i] = s == 0 ? e : pm[ch * 32 + i] + e;
                }
              }
              if (s == maps - 1)
                for (int ch = 0; ch < hc / 32; ++ch) store_weights(pa, ch, pm + ch * 32);
            }
            finish_unit(u, s == maps - 1 ? pb : -1);
          }
        }
      }
    } else {
      // ---- one map: weights against a maximum that follows the row
      for (int v = 0; v < nv; ++v) {
        const int pb = v % L.npb, sb = v % L.nsb;
        const uint32_t pa = smem_u32(smem + L.off_p + pb * L.p_bytes);
        const uint32_t scores = tmem + lane_base + L.tmem_s + (uint32_t)(sb * L.s_cols);
        const int64_t k0 = (int64_t)ktile(v) * nk + half * hc;
        if (ok) ok = mbar_wait(&s_full[sb], (v / L.nsb) & 1u, ab, 78);
        if (ok && v >= L.npb) ok = mbar_wait(&p_empty[pb], ((v - L.npb) / L.npb) & 1u, ab, 79);
        ok = __all_sync(0xffffffffu, ok);
        float big = -INFINITY;
        if (ok) {
          tc_fence_after();
          for (int ch = 0; ch < hc / 32; ++ch) {
            float s[32];
            tmem_ld32(scores + ch * 32, s);
            tmem_wait_ld();
            const int lim = key_limit(k0 + ch * 32);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < lim) big = fmaxf(big, s[i] * scale2[0]);
          }
        }
        top[v & 1][l] = big;
        named_bar_sync(1, 128);
        big = fmaxf(big, top[v & 1][l ^ 64]);
        const bool grown = big > ref + kGrow || (ref == -INFINITY && big > ref);
        if (__any_sync(0xffffffffu, grown)) {
          const float next = grown ? big : ref;
          const float c = !grown || ref == -INFINITY ? 1.f : ex2(ref - next);
          ref = next;
          sum *= c;
          if (v > 0 && ok) {  // the outputs so far, once the products into them are done
            ok = mbar_wait(&p_empty[(v - 1) % L.npb], ((v - 1) / L.npb) & 1u, ab, 80);
            ok = __all_sync(0xffffffffu, ok);
            if (ok && __any_sync(0xffffffffu, c != 1.f)) {
              tc_fence_after();
              for (int col = 0; col < p.D / 2; col += 32) {
                float o[32];
                tmem_ld32(tmem + lane_base + (uint32_t)col, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] *= c;
                tmem_st32(tmem + lane_base + (uint32_t)col, o);
              }
              tmem_wait_st();
            }
          }
        }
        if (ok) {
          const float at = ref == -INFINITY ? 0.f : ref;
          for (int ch = 0; ch < hc / 32; ++ch) {
            float s[32];
            tmem_ld32(scores + ch * 32, s);
            tmem_wait_ld();
            const int lim = key_limit(k0 + ch * 32);
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              s[i] = i < lim ? ex2(s[i] * scale2[0] - at) : 0.f;
              part += s[i];
            }
            sum += part;
            store_weights(pa, ch, s);
          }
        }
        finish_unit(v, pb);
      }
    }

    // ---- epilogue
    if (outputs) {
      named_bar_sync(2, 192);
      const bool wrong = !seq.fits || *reinterpret_cast<volatile int*>(&bad_flag);
      if (wrong && arriver) atomicOr(p.status, DA_DEV_BAD_PAGE);
      if (!kMix) {
        top[0][l] = sum;
        named_bar_sync(1, 128);
        sum += top[0][l ^ 64];
      }
      if (ok) ok = mbar_wait(&o_full, 0, ab, 81);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      const bool whole = tile.y == 1;
      if (!kMix && whole) factor = 1.f / sum;
      if (wrong || !ok) factor = NAN;
      float odd = 0.f;  // becomes NaN with any output that is no number
      const int64_t row = seq.first + t;
      if (ok) {
        for (int i = 0; i < L.npv; ++i) {
          const int col0 = i * L.nc + half * (L.nc / 2);
          for (int c = 0; c < L.nc / 2; c += 32) {
            float o[32];
            tmem_ld32(tmem + lane_base + (uint32_t)(i * (L.nc / 2) + c), o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              odd = fmaf(o[e], 0.f, odd);
              o[e] *= factor;
            }
            if (live && !whole) {
              float4* dst = reinterpret_cast<float4*>(p.part + ((size_t)piece * 128 + trow) * p.D + col0 + c);
#pragma unroll
              for (int e = 0; e < 8; ++e) dst[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            } else if (live) {
              uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.y) + row * p.y_row + col0 + c);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                dst[e] = make_uint4(pack2<T>(o[8 * e], o[8 * e + 1]), pack2<T>(o[8 * e + 2], o[8 * e + 3]),
                                    pack2<T>(o[8 * e + 4], o[8 * e + 5]), pack2<T>(o[8 * e + 6], o[8 * e + 7]));
            }
          }
        }
      }
      if (!kMix && live && !whole && half == 0) {
        p.part_ml[(size_t)piece * 256 + trow] = ref;
        p.part_ml[(size_t)piece * 256 + 128 + trow] = wrong || !ok ? NAN : sum;
      }
      const bool spoiled = named_bar_or(1, 128, live && !wrong && ok && odd != 0.f);
      if (arriver) p.plan.odd[2 * piece + (int)rank] |= spoiled;
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) tmem_dealloc<2>(tmem, L.tmem_cols);
}

// Adds the pieces of the tiles that have several: a warp takes 128 columns of a row.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const ChunkParams p, const bool weighted) {
  grid_dependency_wait();
  grid_launch_dependents();
  if ((int)blockIdx.x >= p.plan.head[1]) return;
  const int first = p.plan.tile_piece[blockIdx.x], pieces = p.plan.tile_piece[blockIdx.x + 1] - first;
  if (pieces < 2) return;
  const int4 here = p.plan.pieces[2 * first];
  const Sequence seq = sequence(p.c, here.x);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, parts = p.D / 128;
  const int trow = blockIdx.y * (8 / parts) + warp / parts, t = here.y * 128 + trow, col = (warp % parts) * 128 + lane * 4;
  if (t >= seq.n) return;
  const float* ml = p.part_ml + (size_t)first * 256 + trow;
  float top = -INFINITY, sum = 0.f;
  if (weighted) {
    for (int i = lane; i < pieces; i += 32) top = fmaxf(top, ml[(size_t)i * 256]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -INFINITY) top = 0.f;
  }
  const float* src = p.part + ((size_t)first * 128 + trow) * p.D + col;
  const size_t step = (size_t)128 * p.D;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int base = 0; base < pieces; base += 32) {
    float w = 1.f;
    if (weighted) {
      w = 0.f;
      if (base + lane < pieces) {
        const float m = ml[(size_t)(base + lane) * 256];
        w = m == -INFINITY ? 0.f : ex2(m - top);
        sum += ml[(size_t)(base + lane) * 256 + 128] * (m == -INFINITY ? 1.f : w);
      }
    }
    const int n = min(32, pieces - base);
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(src + (size_t)(base + i) * step);
      const float wi = __shfl_sync(0xffffffffu, w, i);
      o.x = fmaf(wi, v.x, o.x);
      o.y = fmaf(wi, v.y, o.y);
      o.z = fmaf(wi, v.z, o.z);
      o.w = fmaf(wi, v.w, o.w);
    }
  }
  float f = 1.f;
  if (weighted) {
#pragma unroll
    for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    f = 1.f / sum;
  }
  T* y = static_cast<T*>(p.y) + (seq.first + t) * p.y_row + col;
  *reinterpret_cast<uint2*>(y) = make_uint2(pack2<T>(o.x * f, o.y * f), pack2<T>(o.z * f, o.w * f));
}

// ------------------------------------------------------------------------------------------------ host
namespace {

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

// Tiles and pieces that a step can have: equal shares of at most two rounds of the CTA pairs, and one more piece a tile.
void most(int64_t tokens, int64_t B, int few_most, int64_t* tiles, int64_t* pieces) {
  const int64_t long_ones = tokens / ((int64_t)few_most + 1);
  *tiles = tokens / 128 + (B < long_ones ? B : long_ones) + 1;
  *pieces = *tiles + sm_count() + 1;
}

int64_t plan_bytes(int64_t B, int64_t tiles, int64_t pieces) {
  return 16 + round16((B + 1) * 4) + round16((tiles + 1) * 4) + pieces * 32 + round16(pieces * 8);
}

template <typename T>
int run(const ChunkArgs& a, cudaStream_t st) {
  int64_t tiles, pieces;
  most(a.c.tokens, a.c.B, a.few_most, &tiles, &pieces);
  ChunkParams p;
  p.c = a.c;
  p.plan = chunk_plan(a.workspace, a.c.tokens, a.c.B, a.few_most);
  uint8_t* at = static_cast<uint8_t*>(a.workspace) + plan_bytes(a.c.B, tiles, pieces);
  p.part = reinterpret_cast<float*>(at);
  p.part_ml = p.part + (size_t)pieces * 128 * a.D;
  p.stats = p.part_ml + (size_t)pieces * 256;
  p.H = a.H;
  p.R = a.R;
  p.D = a.D;
  p.group = a.group;
  p.dtype = a.dtype;
  p.few_most = a.few_most;
  p.status = a.status;
  const bool mix = a.maps > 1 && !a.per_map;
  p.maps = mix ? a.maps : 1;
  const Layout L = attn::make_layout(p.maps, a.group, a.R, a.D, mix, true, kSmem);
  if (L.nks < 2 || L.nsb < 2) return DA_ERR_UNSUPPORTED;
  p.brow_k = a.c.page < L.nk / 2 ? a.c.page : L.nk / 2;
  p.brow_v = a.c.page < 64 ? a.c.page : 64;
  const CUtensorMapDataType dt = a.dtype == DA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tq, tk, tv;
  {  // queries: (column in its block of 64, row, branch, block)
    const uint64_t dims[4] = {64, (uint64_t)a.c.tokens, (uint64_t)a.H, (uint64_t)a.R / 64};
    const uint64_t strides[3] = {(uint64_t)a.q_row * 2, a.H > 1 ? (uint64_t)a.q_branch * 2 : 16, 128};
    const uint32_t box[4] = {64, (uint32_t)kRows, 1, 1};
    if (int rc = make_tmap_blocks(&tq, a.q, dt, 2, 4, dims, strides, box)) return rc;
  }
  {  // keys: (column in its block, slot, block)
    const uint64_t dims[3] = {64, (uint64_t)a.c.pages * a.c.page, (uint64_t)a.H * a.R / 64};
    const uint64_t strides[2] = {(uint64_t)a.H * a.R * 2, 128};
    const uint32_t box[3] = {64, (uint32_t)p.brow_k, (uint32_t)(p.brow_k == L.nk / 2 ? L.kbb : 1)};
    if (int rc = make_tmap_blocks(&tk, a.key_pages, dt, 2, 3, dims, strides, box)) return rc;
  }
  {  // values: (column in its block, slot, block inside an nc-wide group, group)
    const uint64_t dims[4] = {64, (uint64_t)a.c.pages * a.c.page, (uint64_t)L.nc / 64, (uint64_t)a.D / L.nc};
    const uint64_t strides[3] = {(uint64_t)a.D * 2, 128, (uint64_t)L.nc * 2};
    const bool whole = p.brow_v == 64;
    const uint32_t box[4] = {64, (uint32_t)p.brow_v, (uint32_t)(whole ? L.per : 1), (uint32_t)(whole ? L.npv : 1)};
    if (int rc = make_tmap_blocks(&tv, a.value_pages, dt, 2, 4, dims, strides, box)) return rc;
  }
  if (int rc = launch_kernel(plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, false, a.c, p.plan, a.few_most,
                             L.nk == 256 ? 8 : 7, sm_count() / 2))
    return rc;
  const int smem = L.smem + 1024;
  const dim3 grid((unsigned)(2 * pieces)), block(kThreads);
  if (int rc = mix ? allow_smem<chunk_kernel<T, true>>(kSmem + 1024) : allow_smem<chunk_kernel<T, false>>(kSmem + 1024)) return rc;
  for (int s = 0; s < (a.per_map ? a.maps : 1); ++s) {
    for (int m = 0; m < kMaxMaps; ++m) {
      const int map = a.per_map ? s : m;
      p.branch0[m] = m < p.maps ? (a.H >= a.maps ? map * a.group : map * a.H / a.maps) : 0;
    }
    p.scales = a.scales + (a.per_map ? s : 0);
    p.weights = a.per_map ? nullptr : a.weights;
    p.y = static_cast<T*>(a.y) + (a.per_map ? (int64_t)s * a.D : 0);
    p.y_row = a.per_map ? (int64_t)a.maps * a.D : a.D;
    p.phase = 0;
    if (mix) {
      p.phase = 1;
      if (int rc = launch_kernel(chunk_kernel<T, true>, grid, block, smem, st, true, tq, tk, tv, p)) return rc;
      p.phase = 2;
      if (int rc = launch_kernel(chunk_kernel<T, true>, grid, block, smem, st, true, tq, tk, tv, p)) return rc;
    } else if (int rc = launch_kernel(chunk_kernel<T, false>, grid, block, smem, st, true, tq, tk, tv, p)) {
      return rc;
    }
    if (int rc = launch_kernel(join_kernel<T>, dim3((unsigned)tiles, (unsigned)(16 * a.D / 128)), dim3(256), 0, st, false, p, !mix)) return rc;
  }
  return DA_OK;
}

}  // namespace

int64_t chunk_workspace(int64_t tokens, int64_t B, int few_most, int D, int maps, bool per_map) {
  int64_t tiles, pieces;
  most(tokens, B, few_most, &tiles, &pieces);
  const int64_t stats = maps > 1 && !per_map ? (int64_t)2 * maps * 128 : 0;
  return plan_bytes(B, tiles, pieces) + pieces * (128 * (int64_t)D + 256 + stats) * (int64_t)sizeof(float);
}

Plan chunk_plan(void* workspace, int64_t tokens, int64_t B, int few_most) {
  int64_t tiles, pieces;
  most(tokens, B, few_most, &tiles, &pieces);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  Plan p;
  p.head = reinterpret_cast<int*>(at);
  at += 16;
  p.seq_piece = reinterpret_cast<int*>(at);
  at += round16((B + 1) * 4);
  p.tile_piece = reinterpret_cast<int*>(at);
  at += round16((tiles + 1) * 4);
  p.pieces = reinterpret_cast<int4*>(at);
  at += pieces * 32;
  p.odd = reinterpret_cast<int*>(at);
  p.tiles_most = (int)tiles;
  p.pieces_most = (int)pieces;
  return p;
}

int chunk_attention(const ChunkArgs& a, cudaStream_t st) {
  return a.dtype == DA_BF16 ? run<__nv_bfloat16>(a, st) : run<__half>(a, st);
}

}  // namespace paged
}  // namespace da
