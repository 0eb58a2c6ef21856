// Outer routed attention of long chunks of new tokens over a paged cache.
//
// The same product as paged_attn.cu's, for sequences that bring many tokens: 128 query tokens a CTA pair, scores and
// P V on paired tensor-core instructions into TMEM, folded as attn_fwd.cu's: a row's 64 first and 64 last keys in two lanes.  What differs:
//   * keys and values come page by page through the table, boxes of a page's positions (up to the tile's); positions
//     that the sequence does not have are fetched past the end of the cache, where TMA fills in zeros;
//   * the softmax offset is each row's own maximum, whatever the keys' lengths.  One map: a running maximum, against
//     which outputs in TMEM are rescaled only when it has grown by more than 2^8 (they are fp32, the weights at most 2^8);
//     several maps: a first launch over the keys leaves each map's maximum and sum, a second builds the mixture
//     P = sum_s alpha_s softmax_s and needs one P V for all maps;
//   * the (query tile, key range) pieces are planned on the device from the lengths: equal key ranges of all tiles, so
//     that few or uneven tiles fill the GPU; join_kernel adds the pieces of a tile in order.
// A value behind a row's last position weighs 0, and 0 times a NaN or an infinity is NaN: such rows are found when they
// are written and their sequences computed again by the other kernel, which tells them apart and reads the cache once per 16 rows
// (512 tokens behind 32768: 376 us instead of 47).  Weights are rounded to 16 bits once, as a second part would double the
// product with the values: 2.3e-3 against 64 bits in bf16, where the outputs' own rounding is 1.7e-3; 2.9e-4 and 2.1e-4 in fp16.
//
// Measured on the device, all launches of a call together: 512 tokens behind 32768 (bf16, one map of 256 columns, 512 value
// columns) 47 us, 0.55 PFLOP/s, of which this file's chunk kernel takes 35 with its tensor pipe 44 % active.  Six
// uneven chunks of up to 700 tokens behind up to 4001 (fp16, four maps of 128 columns) 87 us, 0.26 PFLOP/s: 2^x is asked for
// twice a score and map, 16 a clock, which is 41 and 35 % of the phases, issue slots 43 and 36 %.  What bounds both is latency: before
// its first product a CTA pair takes about 6000 cycles (plan, descriptors, barriers between the two, first keys), after the
// last about 4500 to leave a piece's outputs, 128 KB a CTA; between them a tile of 128 keys waits on a chain of scores,
// maxima, weights and products, of which two groups of softmax warps keep two under way (one group: 115 us instead of 105
// when that step was made).
#include <math.h>

#include "attn_common.h"
#include "host_util.h"
#include "paged_chunk.h"

namespace da {
namespace paged {

using attn::kMaxMaps;

// Warps: 0 brings keys (and the queries), 1 issues the score products, 2 brings values, 3 issues P V; 4 to 11 and 12 to 19
// turn scores into weights, the two groups taking tiles in turn, so that one computes while the other waits; in a group, two
// warps share 32 lanes of TMEM, 32 columns a thread.
constexpr int kThreads = 640, kSoftmaxWarps = 16, kGroupWarps = 8, kFirstSoftmax = 4;
constexpr int kRows = 64;   // query rows a CTA
constexpr int kTile = 128;  // keys a tile: 64 a CTA's box, and 64 score columns a TMEM lane
constexpr int kMaxK = 8, kMaxV = 4;        // most stages
constexpr int kScores = 4, kWeights = 2;  // buffers of scores, two a group of softmax warps, and of weights, one a group
constexpr int kSmem = 224 * 1024;
constexpr float kGrow = 8.f;  // log2 of the growth of a row's maximum that its outputs bear
// log2 by which weights are larger than their offsets make them: fp16 has nothing below 2^-24, so a far tail, or a flat map
// beside a sharp one, would count in the fp32 sums and not in the product.  One map's reach 2^(kGrow + 7) = 2^15, four maps',
// of at most 1 each, 4 x 2^13.
template <typename T, bool kMix>
constexpr float kLift = std::is_same<T, __half>::value ? (kMix ? 13.f : 7.f) : 0.f;

// A CTA's shared memory.  Paired loads take about 0.9 us from a stage's release to its next tile, in which a pair of
// tensor cores consumes about 2000 cycles' worth: rings of 64 KB and more for keys and values keep them fed.
struct Shape {
  int rpb, chunks;   // 64-column blocks a branch, and a map
  int blocks, runs;  // key columns side by side, in blocks (all maps', or a map's), and how many such runs a tile has
  int wide, kslots;  // blocks a key stage, stages
  int nc, npv, per;  // columns a P V product, products, 64-column blocks of one in a CTA
  int q_bytes, k_stage, v_stage, p_bytes, nvs;
  int off_k, off_v, off_p, smem, tmem_cols;
};

// outputs: values and weights have room too (else scores alone).
inline Shape make_shape(int maps, int group, int R, int D, bool outputs, bool repeated) {
  Shape s;
  s.rpb = R / 64;
  s.chunks = group * s.rpb;
  s.runs = repeated ? maps : 1;  // (maps that repeat a branch read its columns once each)
  s.blocks = repeated ? s.chunks : maps * s.chunks;
  s.nc = D < 256 ? D : 256;
  s.npv = D / s.nc;
  s.per = s.nc / 128;
  s.q_bytes = kRows * maps * group * R * 2;
  s.v_stage = 64 * D;  // 64 keys, half of D columns
  s.p_bytes = kRows * kTile * 2;
  const int rings = kSmem - s.q_bytes - (outputs ? kWeights * s.p_bytes : 0);
  // (several maps: one P V for the keys of all of them, so that keys want the room)
  s.nvs = maps > 1 ? 2 : (rings - 65536) / s.v_stage;
  s.nvs = !outputs ? 0 : s.nvs > kMaxV ? kMaxV : s.nvs < 2 ? 2 : s.nvs;
  for (s.wide = 4;; s.wide /= 2) {  // wide boxes, but four stages where the units are small
    s.k_stage = s.wide * 64 * 128;
    s.kslots = (rings - s.nvs * s.v_stage) / s.k_stage;
    if (s.blocks % s.wide == 0 && (s.kslots >= (maps > 1 ? 4 : 2) || s.wide == 1)) break;
  }
  s.kslots = s.kslots > kMaxK ? kMaxK : s.kslots;
  s.off_k = s.q_bytes;
  s.off_v = s.off_k + s.kslots * s.k_stage;
  s.off_p = s.off_v + s.nvs * s.v_stage;
  const int used = s.off_p + (outputs ? kWeights * s.p_bytes : 0);
  s.smem = used < 120 * 1024 ? 120 * 1024 : used;  // one CTA an SM: TMEM
  s.tmem_cols = D / 2 + kScores * 64 > 256 ? 512 : 256;
  if (D / 2 + kScores * 64 > 512) s.tmem_cols = 0;
  return s;
}

struct ChunkParams {
  Cache c;
  Plan plan;
  Shape shape;
  int R, D, maps, group;
  int branch0[kMaxMaps];
  int brow, qrow;      // positions a box of keys or values, rows a box of queries
  int pairs;           // CTA pairs that run side by side
  int phase;           // several maps: 1 sums, 2 outputs; one map: 0
  const float *scales, *weights;
  void* y;
  int64_t y_row;       // elements from row to row
  float* part;         // [pieces][2 CTAs][D / 16] blocks of 32 rows by 32 columns
  float* part_ml;      // [pieces][2][128]: one map's maximum (log2) and sum
  float* stats;        // [pieces][2][maps][128]: phase 1's
  int* status;
};

// ------------------------------------------------------------------------------------------------ plan
constexpr int kPlanThreads = 256, kPlanWarps = kPlanThreads / 32, kLengths = 10, kEnds = 6;
constexpr int kAtOnce = 1024;  // sequences

// One CTA; a warp a sequence, but for the sums over sequences.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const Cache c, const Plan plan, int few_most, int pairs) {
  __shared__ int2 kept[kAtOnce];    // the first sequences' new tokens (of chunks), and tokens that they had
  __shared__ int2 before[kAtOnce];  // tiles and pieces of a sequence, then of those before it
  __shared__ unsigned long long units[kPlanWarps];
  __shared__ long long sums[2][kPlanWarps];
  __shared__ int counts[kLengths], made[2], several, best;
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  auto load = [&](int b) {
    const Sequence s = sequence(c, b);
    return make_int2(s.n > few_most ? s.n : 0, (int)s.held);
  };
  constexpr int nk_shift = 7;  // of kTile
  for (int b = threadIdx.x; b < c.B && b < kAtOnce; b += kPlanThreads) kept[b] = load(b);
  for (int b = threadIdx.x; b < c.B; b += kPlanThreads) plan.odd[b] = 0;
  if (threadIdx.x < kLengths) counts[threadIdx.x] = 0;
  if (threadIdx.x == 0) made[0] = made[1] = several = 0;
  __syncthreads();
  auto get = [&](int b) { return b < kAtOnce ? kept[b] : load(b); };
  auto tiles_of = [](int2 s) { return (s.x + 127) >> 7; };
  auto keys_of = [&](int2 s, int i) {  // key tiles of query tile i
    const int64_t e = (int64_t)s.y + min(s.x, (i + 1) * 128);
    return (int)(((e < c.capacity ? e : c.capacity) + (1 << nk_shift) - 1) >> nk_shift);
  };
  unsigned long long all = 0;
  for (int b = warp; b < c.B; b += kPlanWarps) {
    const int2 s = get(b);
    for (int i = lane; i < tiles_of(s); i += 32) all += keys_of(s, i);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  if (lane == 0) units[warp] = all;
  __syncthreads();
  all = 0;
#pragma unroll
  for (int w = 0; w < kPlanWarps; ++w) all += units[w];
  // The pieces' length: of a few that suit one or two rounds of the CTA pairs, the one that is done first, counting a
  // piece's start and end as kEnds key tiles.  Lane f + 10 k counts the pieces of the f-th in every third tile.
  const int f = lane % kLengths, third = lane / kLengths;
  int length;
  {
    const int extra = 16 >> (f % 5 - 1 < 0 ? 0 : f % 5 - 1);  // none, a 16th, an 8th, a 4th, half more
    const int64_t round = (int64_t)pairs * (f < 5 ? 1 : 2), base = ((int64_t)all + round - 1) / round;
    const int64_t len = base + (f % 5 ? (base + extra - 1) / extra : 0);
    length = (int)(len < 1 ? 1 : len);
  }
  int n = 0;
  for (int b = warp; b < c.B; b += kPlanWarps) {
    const int2 s = get(b);
    if (third < 3)
      for (int i = third; i < tiles_of(s); i += 3) n += ((unsigned)keys_of(s, i) + length - 1) / (unsigned)length;
  }
  if (n) atomicAdd(&counts[f], n);
  __syncthreads();
  if (warp == 0) {
    const int64_t cost = (int64_t)((counts[f] + pairs - 1) / pairs) * (length + kEnds);
    int64_t least = cost;
#pragma unroll
    for (int o = 16; o; o >>= 1) least = min(least, (int64_t)__shfl_xor_sync(0xffffffffu, (long long)least, o));
    const int from = __ffs(__ballot_sync(0xffffffffu, cost == least)) - 1;
    if (lane == from) best = length;
  }
  __syncthreads();
  // tiles and pieces in order
  constexpr long long kMost = 1 << 30;  // (of starts that do not rise: no plan has room for as many)
  long long tiles_before = 0, pieces_before = 0;
  for (int base = 0; base < c.B; base += kAtOnce) {
    const int at_once = min(c.B - base, kAtOnce);
    for (int k = warp; k < at_once; k += kPlanWarps) {
      const int2 s = get(base + k);
      const int tiles = tiles_of(s);
      int count = 0;
      for (int i = lane; i < tiles; i += 32) count += (unsigned)(keys_of(s, i) + best - 1) / (unsigned)best;
      count = __reduce_add_sync(0xffffffffu, count);
      if (lane == 0) before[k] = make_int2(tiles, count);
    }
    __syncthreads();
    {  // four sequences a thread
      constexpr int kEach = kAtOnce / kPlanThreads;
      int2 own[kEach];
      long long t = 0, m = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int k = threadIdx.x * kEach + i;
        own[i] = k < at_once ? before[k] : make_int2(0, 0);
        t += own[i].x;
        m += own[i].y;
      }
      long long ts = t, ms = m;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, ts, o), v = __shfl_up_sync(0xffffffffu, ms, o);
        if (lane >= o) {
          ts += u;
          ms += v;
        }
      }
      if (lane == 31) {
        sums[0][warp] = ts;
        sums[1][warp] = ms;
      }
      __syncthreads();
      t = tiles_before + ts - t;
      m = pieces_before + ms - m;
#pragma unroll
      for (int w = 0; w < kPlanWarps; ++w) {
        if (w < warp) {
          t += sums[0][w];
          m += sums[1][w];
        }
        tiles_before += sums[0][w];
        pieces_before += sums[1][w];
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int k = threadIdx.x * kEach + i;
        if (k < at_once) before[k] = make_int2((int)min(t, kMost), (int)min(m, kMost));
        t += own[i].x;
        m += own[i].y;
      }
    }
    __syncthreads();
    for (int k = warp; k < at_once; k += kPlanWarps) {
      const int b = base + k;
      const int2 s = get(b);
      const int tiles = tiles_of(s), tile0 = before[k].x;
      if (tiles == 0) continue;
      int piece0 = before[k].y;
      const Sequence whole = sequence(c, b);
      for (int i0 = 0; i0 < tiles; i0 += 32) {
        const int i = i0 + lane, keys = i < tiles ? keys_of(s, i) : 0, own = (unsigned)(keys + best - 1) / (unsigned)best;
        int at = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, at, o);
          if (lane >= o) at += u;
        }
        const int more = __shfl_sync(0xffffffffu, at, 31), first = piece0 + at - own;
        // (starts that do not rise bring more tokens than there are rows: what the plan has no room for is the other kernel's)
        const bool fits = i < tiles && tile0 + i < plan.tiles_most && first + own <= plan.pieces_most;
        if (fits) plan.tile_piece[tile0 + i] = first;
        if (i < tiles && !fits) plan.odd[b] = 1;
        if (fits) {
          atomicMax(&made[0], tile0 + i + 1);
          atomicMax(&made[1], first + own);
          if (own > 1) several = 1;
        }
        const int4 tokens = make_int4((int)whole.first, (int)whole.held, 0, 0);
        if (__all_sync(0xffffffffu, own <= 1)) {  // a piece a tile: a lane each
          if (fits && own) {
            plan.pieces[3 * first] = make_int4(b, i, 0, keys);
            plan.pieces[3 * first + 1] = make_int4(first, 1, whole.n, whole.fits);
            plan.pieces[3 * first + 2] = tokens;
          }
        } else {
          // (a tile's pieces side by side: the warp writes one tile after another, a piece a lane)
          for (int j = 0; j < min(32, tiles - i0); ++j) {
            const int from = __shfl_sync(0xffffffffu, first, j), many = __shfl_sync(0xffffffffu, fits ? own : 0, j);
            const int last = __shfl_sync(0xffffffffu, keys, j);
            for (int m = lane; m < many; m += 32) {
              plan.pieces[3 * (from + m)] = make_int4(b, i0 + j, m * best, min(best, last - m * best));
              plan.pieces[3 * (from + m) + 1] = make_int4(from, many, whole.n, whole.fits);
              plan.pieces[3 * (from + m) + 2] = tokens;
            }
          }
        }
        piece0 = (int)min((long long)piece0 + more, kMost);
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    plan.tile_piece[made[0]] = made[1];
    *reinterpret_cast<int4*>(plan.head) = make_int4(made[1], made[0], several, 0);
  }
}

// ------------------------------------------------------------------------------------------------ attention
DA_DEV bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// A stage or buffer of a ring, and the parity of its barrier.
struct Turn {
  int i;
  uint32_t phase;
  DA_DEV void next(int n) {
    if (++i == n) {
      i = 0;
      phase ^= 1;
    }
  }
};

template <typename T, bool kMix>
__global__ void __launch_bounds__(kThreads, 1) chunk_kernel(const __grid_constant__ CUtensorMap tq,
                                                            const __grid_constant__ CUtensorMap tk,
                                                            const __grid_constant__ CUtensorMap tv,
                                                            const __grid_constant__ ChunkParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];  // (with the static part, all of an SM's 227 KB: none for padding)
  __shared__ uint64_t q_full, o_full;
  __shared__ uint64_t k_full[kMaxK], k_empty[kMaxK], v_full[kMaxV], v_empty[kMaxV];
  __shared__ uint64_t s_full[kScores], s_empty[kScores], p_full[kWeights], p_empty[kWeights];
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag, bad_flag;
  __shared__ float top[2][2][128];  // what the four threads of a row in a group tell each other
  __shared__ float row_ref[kRows];             // one map: each row's offset, handed from tile to tile

  const Shape& L = p.shape;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank() & 1u;
  const int piece = blockIdx.x / 2;  // (the plan has room for every CTA pair's piece)
  if (piece >= p.pairs) {  // behind the first round there is no launch to overlap with, but pieces that a plan of the most has
    grid_dependency_wait();
    if (piece >= p.plan.head[0]) return;
  }
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
    for (int i = 0; i < kScores; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 2 * kGroupWarps);  // each warp of a group, of both CTAs
    }
    for (int i = 0; i < kWeights; ++i) {
      mbar_init(&p_full[i], 2 * kGroupWarps);
      mbar_init(&p_empty[i], 1);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc<2>(&tmem_base, L.tmem_cols);
    tmem_relinquish<2>();
  }
  if (threadIdx.x == 0) {
    prefetch_tmap(&tq);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  grid_dependency_wait();  // the plan and the appended tokens are visible from here on
  grid_launch_dependents();
  const int4 here = p.plan.pieces[3 * piece], tile = p.plan.pieces[3 * piece + 1], seq = p.plan.pieces[3 * piece + 2];
  const bool on = piece < p.plan.head[0];
  const int t0 = here.y * 128;  // first token of the tile in its sequence
  const int n = tile.z, held = seq.y;
  const int64_t reach = (int64_t)held + min(n, t0 + 128);
  const int64_t end = reach < p.c.capacity ? reach : p.c.capacity;  // positions that some row sees
  const int nj = here.w, maps = kMix ? p.maps : 1;
  const bool outputs = !kMix || p.phase == 2;
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
  // (the pieces that run side by side start at different tiles of their ranges: any order gives the same rows)
  int first = on ? piece % nj : 0;
  auto tile_after = [&](int j) { return j + 1 == nj ? 0 : j + 1; };

  if (!on) {
  } else if (warp == 0) {
    // ---------------------------------------------------------------- keys (both CTAs)
    // (pages of fewer than 64 positions: a lane a box, its slot looked up a tile ahead; one lane for all of them, a look-up
    // after another, took 93 us instead of 59 for 512 tokens behind 32768 in pages of 16)
    const int across = p.brow == 64 ? 1 : L.wide, r0 = lane / across * p.brow, e = lane % across;
    const int to = (e * 64 + r0) * 128;
    auto lookup = [&](int kt) { return slot_of((int64_t)(here.z + kt) * kTile + (int)rank * 64 + r0); };
    int slot = r0 < 64 ? lookup(first) : 0;
    if (rank == 0 && lane == 0) mbar_arrive_expect_tx(&q_full, 2 * L.q_bytes / kRows * p.qrow);
    const uint32_t qf = mapa_shared(smem_u32(&q_full), 0), kf = mapa_shared(smem_u32(&k_full[0]), 0);
    {  // a lane a block of queries (fewer packed rows than a CTA's 64: the other rows hold anything, and are no sequence's)
      const int row = seq.x + t0 + 64 * (int)rank;  // (rows past the last token are zeros)
      const int s = lane / L.chunks, in = lane % L.chunks;
      if (s < maps)
        tma_load_4d_pair(&tq, qf, smem + lane * (kRows * 128), 0, row, p.branch0[s] + in / L.rpb, in % L.rpb);
    }
    Turn st{0, 0};
    bool ok = true;
    int used = 0;
    for (int j = 0, kt = first; r0 < 64 && ok && j < nj; ++j) {
      const int at = slot;
      kt = tile_after(kt);
      if (j + 1 < nj) slot = lookup(kt);
      for (int s = 0; ok && s < L.runs; ++s)
        for (int c = 0; c < L.blocks; c += L.wide, st.next(L.kslots), ++used) {
          if (!(ok = mbar_wait(&k_empty[st.i], st.phase ^ 1u, ab, 71))) break;
          if (rank == 0 && lane == 0) mbar_arrive_expect_tx(&k_full[st.i], 2 * L.k_stage);
          tma_load_3d_pair(&tk, kf + st.i * 8, smem + L.off_k + st.i * L.k_stage + to, 0, at, p.branch0[s] * L.rpb + c + e);
        }
    }
    __syncwarp();
    if (rank == 0 && lane == 0) {  // none of the loads may be in flight at teardown
      mbar_wait_drain(&q_full, 0);
      for (int i = 0; i < min(used, L.kslots); ++i) {
        if (st.i-- == 0) {
          st.i = L.kslots - 1;
          st.phase ^= 1;
        }
        mbar_wait_drain(&k_full[st.i], st.phase);
      }
    }
  } else if (warp == 2) {
    // ---------------------------------------------------------------- values (both CTAs)
    Turn st{0, 0};
    int used = 0;
    if (outputs) {
      const uint32_t vf = mapa_shared(smem_u32(&v_full[0]), 0);
      // One box: this CTA's column blocks of each of the value groups; or a lane a box of a page and a block.
      const int across = p.brow == 64 ? 1 : L.npv * L.per, r0 = lane / across * p.brow, i = lane % across / L.per, e = lane % across % L.per;
      auto lookup = [&](int kt, int c) { return slot_of((int64_t)(here.z + kt) * kTile + c * 64 + r0); };
      const int to = ((i * L.per + e) * 64 + r0) * 128;
      bool ok = true;
      int slot = r0 < 64 ? lookup(first, 0) : 0;
      for (int j = 0, kt = first; r0 < 64 && ok && j < nj; ++j)
        for (int c = 0; c < 2; ++c, st.next(L.nvs), ++used) {
          const int at = slot;
          if (c) kt = tile_after(kt);
          if (c == 0 || j + 1 < nj) slot = lookup(kt, c ^ 1);
          if (!(ok = mbar_wait(&v_empty[st.i], st.phase ^ 1u, ab, 72))) break;
          if (rank == 0 && lane == 0) mbar_arrive_expect_tx(&v_full[st.i], 2 * L.v_stage);
          tma_load_4d_pair(&tv, vf + st.i * 8, smem + L.off_v + st.i * L.v_stage + to, 0, at, (int)rank * L.per + e, i);
        }
    }
    __syncwarp();
    if (outputs) named_bar_sync(2, 32 * (kSoftmaxWarps + 1));  // bad_flag is final
    if (rank == 0 && lane == 0)
      for (int i = 0; i < min(used, L.nvs); ++i) {
        if (st.i-- == 0) {
          st.i = L.nvs - 1;
          st.phase ^= 1;
        }
        mbar_wait_drain(&v_full[st.i], st.phase);
      }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- scores (the pair's leader)
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = idesc_f16(128, kTile, std::is_same<T, __nv_bfloat16>::value, false, false);
      const uint64_t qd = sdesc_sw128(smem_u32(smem), 16, 1024);
      const uint32_t hi = (uint32_t)(qd >> 32), q_lo = (uint32_t)qd, k_lo = (uint32_t)sdesc_sw128(smem_u32(smem + L.off_k), 16, 1024);
      const uint32_t d0 = tmem + (uint32_t)(p.D / 2);
      const int chunks = L.chunks, wide = L.wide, slots = L.kslots;
      const uint32_t step = (uint32_t)L.k_stage >> 4;
      bool ok = mbar_wait(&q_full, 0, ab, 73);
      tc_fence_after();
      Turn st{0, 0};
      int unit = 0, in = 0;  // block of the stage
      for (int j = 0; ok && j < nj; ++j) {
        uint32_t a = q_lo;
        for (int s = 0; s < maps; ++s, ++unit) {
          // a group's units take its own two buffers in turn (one that the groups shared would complete phases that a group
          // never waits for, and a wait for the phase after those would end at once)
          const int group = (outputs ? j : unit) & 1, turn = outputs ? (j >> 1) * maps + s : unit >> 1;
          const int buffer = 2 * group + (turn & 1);
          const uint32_t d = d0 + (uint32_t)(buffer * 64), parity = ((turn >> 1) & 1u) ^ 1u;
          if (in == 0) ok = mbar_wait2(&s_empty[buffer], parity, &k_full[st.i], st.phase, ab, 74);
          else ok = mbar_wait(&s_empty[buffer], parity, ab, 74);
          if (!ok) break;
          tc_fence_after();
          for (int c = 0; c < chunks; ++c, a += kRows * 128 / 16) {
            if (c && in == 0) {
              if (!(ok = mbar_wait(&k_full[st.i], st.phase, ab, 75))) break;
              tc_fence_after();
            }
            const uint32_t b = k_lo + (uint32_t)st.i * step + (uint32_t)in * (kRows * 128 / 16);
#pragma unroll
            for (int k = 0; k < 4; ++k)  // +32 B per K step of 16 = +2 in the encoded address
              mma_f16_lo<2>(d, a + 2 * k, b + 2 * k, hi, hi, idesc, (c | k) ? 1u : 0u);
            if (++in == wide) {
              mma_commit_pair(smem_u32(&k_empty[st.i]));
              st.next(slots);
              in = 0;
            }
          }
          if (!ok) break;
          mma_commit_pair(smem_u32(&s_full[buffer]));
        }
      }
      if (!outputs) {
        mma_commit_pair(smem_u32(&o_full));
        mbar_wait_drain(&o_full, 0);  // every score product has completed
      }
    }
  } else if (warp == 3) {
    // ---------------------------------------------------------------- P V (the pair's leader)
    if (rank == 0 && outputs && elect_one()) {
      const uint32_t idesc = idesc_f16(128, L.nc, std::is_same<T, __nv_bfloat16>::value, false, true);  // B = V, MN-major
      const uint64_t pd = sdesc_sw128(smem_u32(smem + L.off_p), 16, 1024);
      // MN-major V: rows are keys (K), 128 B = 64 value columns (N); LBO = distance between 64-column boxes, SBO = 8 key rows
      const uint64_t vd = sdesc_sw128(smem_u32(smem + L.off_v), 64 * 128, 1024);
      const uint32_t p_hi = (uint32_t)(pd >> 32), v_hi = (uint32_t)(vd >> 32);
      const uint32_t group = (uint32_t)(L.per * (64 * 128) >> 4), step = (uint32_t)L.v_stage >> 4;
      const uint32_t d1 = tmem + (uint32_t)(L.nc / 2);
      const bool two = L.npv == 2;
      const int slots = L.nvs;
      Turn st{0, 0}, pb{0, 0};
      bool ok = true;
      for (int j = 0; ok && j < nj; ++j, pb.next(kWeights)) {
        if (!(ok = mbar_wait(&p_full[pb.i], pb.phase, ab, 76))) break;
        tc_fence_after();
        uint32_t a = (uint32_t)pd + (uint32_t)(pb.i * (L.p_bytes >> 4));
        for (int c = 0; c < 2; ++c, a += kRows * 128 / 16, st.next(slots)) {
          if (!(ok = mbar_wait(&v_full[st.i], st.phase, ab, 77))) break;
          tc_fence_after();
          const uint32_t b = (uint32_t)vd + (uint32_t)st.i * step;
          {
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // K step of 16 keys: A +32 B (+2), B +16 rows x 128 B (+128)
              mma_f16_lo<2>(tmem, a + 2 * k, b + 128 * k, p_hi, v_hi, idesc, (j | c | k) ? 1u : 0u);
              if (two) mma_f16_lo<2>(d1, a + 2 * k, b + group + 128 * k, p_hi, v_hi, idesc, (j | c | k) ? 1u : 0u);
            }
            mma_commit_pair(smem_u32(&v_empty[st.i]));
          }
        }
        if (!ok) break;
        mma_commit_pair(smem_u32(&p_empty[pb.i]));
      }
      mma_commit_pair(smem_u32(&o_full));
      mbar_wait_drain(&o_full, 0);  // every P V product (and so every score product) has completed
    }
  } else if (warp >= kFirstSoftmax) {
    // ---------------------------------------------------------------- weights, epilogue
    const int quad = warp & 3, group = (warp - kFirstSoftmax) / kGroupWarps;  // lanes of TMEM; whose turn
    const int part = ((warp - kFirstSoftmax) >> 2) & 1;                      // which 32 of a lane's 64 columns
    const int l = quad * 32 + lane;
    const int r = l & 63, half = l >> 6;  // row of the CTA; which 64 keys of a tile
    const int trow = 64 * (int)rank + r;  // row of the tile
    const int t = t0 + trow;              // token of the sequence
    const int64_t sees = min((int64_t)held + t + 1, end);
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t scores = tmem + lanes + (uint32_t)(p.D / 2 + group * 128 + part * 32);
    float* scratch = reinterpret_cast<float*>(smem + L.off_k);  // [2][4][128]: the keys' ring, when they are done with
    const uint32_t s_leader = mapa_shared(smem_u32(&s_empty[0]), 0), p_leader = mapa_shared(smem_u32(&p_full[0]), 0);
    const float kLog2e = 1.4426950408889634f;
    const float gsc = rsqrtf((float)p.group) * kLog2e;
    bool ok = true;
    Turn sb{0, 0};

    // The group's next scores, 32 a thread; the buffer is given back.
    auto take = [&](float (&v)[32]) {
      if (ok) ok = mbar_wait(&s_full[2 * group + sb.i], sb.phase, ab, 78);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        tmem_ld32(scores + (uint32_t)(sb.i * 64), v);
        tmem_wait_ld();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(s_leader + (2 * group + sb.i) * 8);
      sb.next(2);
    };
    // Visible keys among the thread's 32 of tile kt.
    auto visible = [&](int kt) -> int {
      return (int)clamp64(sees - ((int64_t)(here.z + kt) * kTile + half * 64 + part * 32), 0, 32);
    };
    // A tile's weights into buffer `group`, as the tiles take turns; p_phase is of its barrier.
    uint32_t p_phase = 1;
    const uint32_t box = smem_u32(smem + L.off_p + group * L.p_bytes) + half * (kRows * 128);
    auto give = [&](const float (&e)[32]) {
      if (ok) ok = mbar_wait(&p_empty[group], p_phase, ab, 79);
      ok = __all_sync(0xffffffffu, ok);
      p_phase ^= 1;
      if (ok) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          st_shared_v4(box + sw128_offset(r, part * 4 + i), pack2<T>(e[8 * i], e[8 * i + 1]), pack2<T>(e[8 * i + 2], e[8 * i + 3]),
                       pack2<T>(e[8 * i + 4], e[8 * i + 5]), pack2<T>(e[8 * i + 6], e[8 * i + 7]));
        fence_proxy_async();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(p_leader + group * 8);
    };
    auto hide = [](float (&v)[32], int lim) {
      if (!__all_sync(0xffffffffu, lim == 32))
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = i < lim ? v[i] : -INFINITY;
    };
    auto largest = [](const float (&v)[32]) {
      float a = v[0], b = v[1], c = v[2], d = v[3];
#pragma unroll
      for (int i = 4; i < 32; i += 4) {
        a = fmaxf(a, v[i]);
        b = fmaxf(b, v[i + 1]);
        c = fmaxf(c, v[i + 2]);
        d = fmaxf(d, v[i + 3]);
      }
      return fmaxf(fmaxf(a, b), fmaxf(c, d));
    };

    float factor = 1.f;                // of the outputs in TMEM
    float ref = -INFINITY, sum = 0.f;  // one map: offset of the weights (log2), this thread's sum
    if constexpr (kMix) {
      float scale[kMaxMaps];
#pragma unroll
      for (int s = 0; s < kMaxMaps; ++s) scale[s] = s < maps ? p.scales[s] * gsc : 0.f;
      if (p.phase == 1) {
        // ---- each map's maximum (of the scaled scores) and sum of its weights against it
        float mx[kMaxMaps], sm[kMaxMaps];
#pragma unroll
        for (int s = 0; s < kMaxMaps; ++s) {
          mx[s] = -INFINITY;
          sm[s] = 0.f;
        }
        int unit = 0;
        for (int j = 0, kt = first; j < nj; ++j, kt = tile_after(kt)) {
          const int lim = visible(kt);
#pragma unroll
          for (int s = 0; s < kMaxMaps; ++s) {
            if (s >= maps) break;
            if ((unit++ & 1) == group) {
              float v[32];
              take(v);
              if (ok) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] *= scale[s];
                hide(v, lim);
                const float next = fmaxf(mx[s], largest(v)), at = next == -INFINITY ? 0.f : next;
                float a = 0.f, b = 0.f;
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                  a += ex2(v[i] - at);
                  b += ex2(v[i + 1] - at);
                }
                sm[s] = fmaf(sm[s], mx[s] == -INFINITY ? 1.f : ex2(mx[s] - at), a + b);  // (the sum is 0 then, or NaN)
                mx[s] = next;
              }
            }
          }
        }
        named_bar_sync(1, 32 * kSoftmaxWarps);  // (every score product is over)
#pragma unroll
        for (int s = 0; s < kMaxMaps; ++s) {
          if (s >= maps) break;
          scratch[(group * 2 + part) * 128 + l] = mx[s];
          scratch[512 + (group * 2 + part) * 128 + l] = ok ? sm[s] : NAN;
          named_bar_sync(1, 32 * kSoftmaxWarps);
          if (group == 0 && part == 0 && half == 0) {  // the eight threads of a row: groups, parts and halves
            float m = -INFINITY, a = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, scratch[(i >> 1) * 128 + (i & 1) * 64 + r]);
            const float at = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float mi = scratch[(i >> 1) * 128 + (i & 1) * 64 + r];
              a += scratch[512 + (i >> 1) * 128 + (i & 1) * 64 + r] * (mi == -INFINITY ? 1.f : ex2(mi - at));
            }
            float* dst = p.stats + ((size_t)piece * 2 * maps + s) * 128 + trow;
            dst[0] = m;
            dst[(size_t)maps * 128] = a;
          }
          named_bar_sync(1, 32 * kSoftmaxWarps);
        }
      } else {
        // ---- the pieces' sums of this row; offsets so that the mixture's largest weight is near 1 (2^13 in fp16)
        // (the row's eight threads share them out: a map and every other piece each)
        float off[kMaxMaps], al[kMaxMaps], shift = -INFINITY;
        {
          float* meet = &top[0][0][0];  // [4][2][64]
          const int s = group * 2 + part;
          float m = -INFINITY, a = 0.f;
          if (s < maps) {
            const float* src = p.stats + ((size_t)tile.x * 2 * maps + s) * 128 + trow;
            const size_t next = (size_t)2 * maps * 128;
#pragma unroll 4
            for (int i = half; i < tile.y; i += 2) {
              const float mi = src[i * next], ai = src[i * next + (size_t)maps * 128];
              const float to = fmaxf(m, mi), at = to == -INFINITY ? 0.f : to;
              a = a * (m == -INFINITY ? 1.f : ex2(m - at)) + ai * (mi == -INFINITY ? 1.f : ex2(mi - at));
              m = to;
            }
          }
          meet[(s * 2 + half) * 64 + r] = m;
          named_bar_sync(1, 32 * kSoftmaxWarps);
          const float to = fmaxf(meet[s * 128 + r], meet[s * 128 + 64 + r]), at = to == -INFINITY ? 0.f : to;
          a *= m == -INFINITY ? 1.f : ex2(m - at);
          named_bar_sync(1, 32 * kSoftmaxWarps);
          meet[(s * 2 + half) * 64 + r] = a;
          named_bar_sync(1, 32 * kSoftmaxWarps);
          a = meet[s * 128 + r] + meet[s * 128 + 64 + r];
          named_bar_sync(1, 32 * kSoftmaxWarps);
          meet[(s * 2 + half) * 64 + r] = half ? log2f(a) : to;
          named_bar_sync(1, 32 * kSoftmaxWarps);
#pragma unroll
          for (int i = 0; i < kMaxMaps; ++i) {
            off[i] = al[i] = 0.f;
            if (i >= maps) continue;
            const float log_sum = meet[i * 128 + 64 + r];
            al[i] = p.weights ? p.weights[i] : 1.f;
            off[i] = meet[i * 128 + r] + log_sum;
            shift = fmaxf(shift, log2f(fabsf(al[i])) - log_sum);
          }
        }
        shift = fminf(fmaxf(shift, -100.f), 100.f) - kLift<T, true>;
        factor = ex2(shift);
#pragma unroll
        for (int s = 0; s < kMaxMaps; ++s) off[s] += shift;
        for (int j = 0, kt = first; j < nj; ++j, kt = tile_after(kt)) {
          if ((j & 1) != group) continue;
          const int lim = visible(kt);
          float pm[32];
#pragma unroll
          for (int s = 0; s < kMaxMaps; ++s) {
            if (s >= maps) break;
            float v[32];
            take(v);
            if (!ok) continue;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float e = ex2(fmaf(v[i], scale[s], -off[s]));
              pm[i] = s == 0 ? al[0] * e : fmaf(al[s], e, pm[i]);
            }
          }
          // (a temperature may have any sign: a hidden key's weight is set, not made by a score of minus infinity)
          if (!__all_sync(0xffffffffu, lim == 32))
#pragma unroll
            for (int i = 0; i < 32; ++i) pm[i] = i < lim ? pm[i] : 0.f;
          give(pm);
        }
      }
    } else {
      // ---- one map: weights against a maximum that follows the row.  The offset of tile j + 1 starts from tile j's, which the
      // other group leaves in row_ref.
      const float scale = p.scales[0] * gsc;
      for (int j = 0, kt = first; j < nj; ++j, kt = tile_after(kt)) {
        if ((j & 1) != group) continue;
        float v[32], big = -INFINITY;
        take(v);
        if (ok) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] *= scale;
          hide(v, visible(kt));
          big = largest(v);
        }
        float (&mine)[2][128] = top[group];
        mine[part][l] = big;
        if (j) named_bar_sync(3 + group, 32 * kSoftmaxWarps);  // tile j - 1's offsets are there (and the maxima)
        else named_bar_sync(5, 32 * kGroupWarps);
        big = fmaxf(fmaxf(mine[0][l], mine[1][l]), fmaxf(mine[0][l ^ 64], mine[1][l ^ 64]));
        const float last = j ? row_ref[r] : -INFINITY;
        if (last != ref) {  // the other group's tile raised it
          if (ref != -INFINITY) sum *= ex2(ref - last);
          ref = last;
        }
        const bool grown = big > ref + kGrow || (ref == -INFINITY && big > ref);
        const float next = grown ? big : ref;
        const bool rescale = grown && ref != -INFINITY;
        const bool any = named_bar_or(5 + group, 32 * kGroupWarps, rescale);  // (row_ref is read: it may be written)
        if (half == 0 && part == 0) row_ref[r] = next;
        if (j + 1 < nj) named_bar_arrive(4 - group, 32 * kSoftmaxWarps);
        if (any) {  // the outputs so far, once the products into them are done: tile j - 1's
          const float c = rescale ? ex2(ref - next) : 1.f;
          sum *= c;
          // (its buffer's products before those, tile j - 3's, may be under way still, and a wait for the later ones would end
          // at once then; those of the group's own tile j - 2 come after them and cannot be two phases on)
          const uint32_t done = group ? p_phase ^ 1u : p_phase;
          if (ok && j >= 2) ok = mbar_wait(&p_empty[group], p_phase, ab, 80);
          if (ok) ok = mbar_wait(&p_empty[group ^ 1], done, ab, 80);
          ok = __all_sync(0xffffffffu, ok);
          if (ok) {
            tc_fence_after();
            for (int col = part * (p.D / 4); col < (part + 1) * (p.D / 4); col += 32) {
              float o[32];
              tmem_ld32(tmem + lanes + (uint32_t)col, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= c;
              tmem_st32(tmem + lanes + (uint32_t)col, o);
            }
            tmem_wait_st();
            tc_fence_before();
          }
        }
        ref = next;
        const float at = ref == -INFINITY ? 0.f : ref - kLift<T, false>;
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          v[i] = ex2(v[i] - at);
          v[i + 1] = ex2(v[i + 1] - at);
          a += v[i];
          b += v[i + 1];
        }
        sum += a + b;
        give(v);
      }
    }

    // ---- epilogue
    if (outputs) {
      named_bar_sync(2, 32 * (kSoftmaxWarps + 1));
      const bool wrong = !tile.w || *reinterpret_cast<volatile int*>(&bad_flag);
      if (wrong && warp == kFirstSoftmax && lane == 0) atomicOr(p.status, DA_DEV_BAD_PAGE);
      if (!kMix) {  // (the group that had the tile before the last one may have an older offset)
        const float last = row_ref[r];
        if (ref != -INFINITY && ref != last) sum *= ex2(ref - last);
        ref = last;
        scratch[(group * 2 + part) * 128 + l] = sum;
        named_bar_sync(1, 32 * kSoftmaxWarps);
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += scratch[i * 128 + r] + scratch[i * 128 + 64 + r];
        named_bar_sync(1, 32 * kSoftmaxWarps);
      }
      if (ok) ok = mbar_wait(&o_full, 0, ab, 81);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      const bool single = tile.y == 1;
      if (!kMix && single) factor = 1.f / sum;
      if (wrong || !ok) factor = NAN;
      if (!kMix && !single && group == 0 && part == 0 && half == 0 && t < n) {
        p.part_ml[(size_t)piece * 256 + trow] = ref;
        p.part_ml[(size_t)piece * 256 + 128 + trow] = wrong || !ok ? NAN : sum;
      }
      float odd = 0.f;  // becomes NaN with any output that is no number
      if (ok) {
        // 32 rows by 32 columns at a time go through shared memory (the rings, done with), each to a place of its own: a
        // piece's part as one bulk copy into a block of 4 KB (4500 cycles for a CTA's 128 KB when all write, against 7000
        // by stores), a finished row's columns so that they are stored side by side.
        const int base = trow - lane;       // tile row of lane 0 (a warp's lanes are consecutive rows)
        for (int tc = (group * 2 + part) * 32; tc < p.D / 2; tc += 128) {
          const int col = tc / (L.nc / 2) * L.nc + half * (L.nc / 2) + tc % (L.nc / 2);
          float o[32];
          tmem_ld32(tmem + lanes + (uint32_t)tc, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            odd = fmaf(o[e], 0.f, odd);
            o[e] *= factor;
          }
          const int blk = tc / 32 * 4 + quad;
          const uint32_t stage = smem_u32(smem + L.off_k) + (uint32_t)blk * 4096;
          if (!single) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              st_shared_v4(stage + sw128_offset(lane, e), __float_as_uint(o[4 * e]), __float_as_uint(o[4 * e + 1]),
                           __float_as_uint(o[4 * e + 2]), __float_as_uint(o[4 * e + 3]));
            fence_proxy_async();
            __syncwarp();
            if (lane == 0)
              bulk_store(p.part + (((size_t)piece * 2 + rank) * (p.D / 16) + blk) * 1024, smem + L.off_k + blk * 4096, 4096);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              st_shared_v4(stage + lane * 64 + ((e ^ ((lane >> 1) & 3)) << 4), pack2<T>(o[8 * e], o[8 * e + 1]),
                           pack2<T>(o[8 * e + 2], o[8 * e + 3]), pack2<T>(o[8 * e + 4], o[8 * e + 5]),
                           pack2<T>(o[8 * e + 6], o[8 * e + 7]));
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int row = e * 8 + lane / 4;
              const uint4 w = ld_shared_v4(stage + row * 64 + (((lane & 3) ^ ((row >> 1) & 3)) << 4));
              if (t0 + base + row < n)
                *reinterpret_cast<uint4*>(static_cast<T*>(p.y) + ((int64_t)seq.x + t0 + base + row) * p.y_row + col + (lane & 3) * 8) = w;
            }
          }
        }
      }
      if (!single && lane == 0) {
        tma_store_commit();
        tma_store_wait_all();
      }
      const bool spoiled = named_bar_or(1, 32 * kSoftmaxWarps, t < n && !wrong && ok && odd != 0.f);
      if (spoiled && warp == kFirstSoftmax && lane == 0) atomicOr(p.plan.odd + here.x, 1);
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) tmem_dealloc<2>(tmem, L.tmem_cols);
}

// Adds the pieces of a tile that has several: a warp takes 128 columns of a row.
template <typename T>
DA_DEV void join_tile(const ChunkParams& p, const bool weighted, int index) {
  const int first = p.plan.tile_piece[index], pieces = p.plan.tile_piece[index + 1] - first;
  if (pieces < 2) return;
  const int4 here = p.plan.pieces[3 * first], tile = p.plan.pieces[3 * first + 1], seq = p.plan.pieces[3 * first + 2];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, parts = p.D / 128;
  const int trow = blockIdx.y * (8 / parts) + warp / parts, t = here.y * 128 + trow, col = (warp % parts) * 128 + lane * 4;
  if (t >= tile.z) return;
  const float* ml = p.part_ml + (size_t)first * 256 + trow;
  float top = -INFINITY, sum = 0.f;
  if (weighted) {
    for (int i = lane; i < pieces; i += 32) top = fmaxf(top, ml[(size_t)i * 256]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -INFINITY) top = 0.f;
  }
  // the block of 32 rows by 32 columns, as the chunk kernel's TMEM has them, and the place in its row
  const int nc = p.shape.nc, half = col % nc / (nc / 2), tc = col / nc * (nc / 2) + col % (nc / 2), r = trow & 63;
  const int blk = tc / 32 * 4 + half * 2 + r / 32;
  const float* src = p.part + (((size_t)first * 2 + trow / 64) * (p.D / 16) + blk) * 1024 + (r % 32) * 32 +
                     ((tc % 32 / 4) ^ (r & 7)) * 4;
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
  T* y = static_cast<T*>(p.y) + ((int64_t)seq.x + t) * p.y_row + col;
  *reinterpret_cast<uint2*>(y) = make_uint2(pack2<T>(o.x * f, o.y * f), pack2<T>(o.z * f, o.w * f));
}

template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const ChunkParams p, const bool weighted) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int4 head = *reinterpret_cast<const int4*>(p.plan.head);
  if (!head.z) return;
  for (int tile = blockIdx.x; tile < head.y; tile += gridDim.x) join_tile<T>(p, weighted, tile);
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
  return 16 + round16(B * 4) + round16((tiles + 1) * 4) + pieces * 48;
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
  p.R = a.R;
  p.D = a.D;
  p.group = a.group;
  p.status = a.status;
  p.pairs = sm_count() / 2;
  const bool mix = a.maps > 1 && !a.per_map;
  p.maps = mix ? a.maps : 1;
  const bool repeated = p.maps > a.H;
  p.shape = make_shape(p.maps, a.group, a.R, a.D, true, repeated);
  const Shape L = p.shape;
  if (L.kslots < 2 || !L.tmem_cols) return DA_ERR_UNSUPPORTED;
  p.brow = a.c.page < 64 ? a.c.page : 64;
  p.qrow = a.c.tokens < kRows ? (int)a.c.tokens : kRows;
  const bool whole = p.brow == 64;
  const CUtensorMapDataType dt = a.dtype == DA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tq, tk, tv;
  auto map_keys = [&](int wide) {  // (column in its block, slot, block)
    const uint64_t dims[3] = {64, (uint64_t)a.c.pages * a.c.page, (uint64_t)a.H * a.R / 64};
    const uint64_t strides[2] = {(uint64_t)a.H * a.R * 2, 128};
    const uint32_t box[3] = {64, (uint32_t)p.brow, (uint32_t)(whole ? wide : 1)};
    return make_tmap_blocks(&tk, a.key_pages, dt, 2, 3, dims, strides, box);
  };
  {  // queries: (column in its block of 64, row, branch, block)
    const uint64_t dims[4] = {64, (uint64_t)a.c.tokens, (uint64_t)a.H, (uint64_t)a.R / 64};
    const uint64_t strides[3] = {(uint64_t)a.q_row * 2, a.H > 1 ? (uint64_t)a.q_branch * 2 : 16, 128};
    const uint32_t box[4] = {64, (uint32_t)p.qrow, 1, 1};
    if (int rc = make_tmap_blocks(&tq, a.q, dt, 2, 4, dims, strides, box)) return rc;
  }
  {  // values: (column in its block, slot, block inside an nc-wide group, group)
    const uint64_t dims[4] = {64, (uint64_t)a.c.pages * a.c.page, (uint64_t)L.nc / 64, (uint64_t)a.D / L.nc};
    const uint64_t strides[3] = {(uint64_t)a.D * 2, 128, (uint64_t)L.nc * 2};
    const uint32_t box[4] = {64, (uint32_t)p.brow, (uint32_t)(whole ? L.per : 1), (uint32_t)(whole ? L.npv : 1)};
    if (int rc = make_tmap_blocks(&tv, a.value_pages, dt, 2, 4, dims, strides, box)) return rc;
  }
  if (int rc = launch_kernel(plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, false, a.c, p.plan, a.few_most,
                             sm_count() / 2))
    return rc;
  const dim3 grid((unsigned)(2 * pieces)), block(kThreads);
  if (int rc = mix ? allow_smem<chunk_kernel<T, true>>(kSmem) : allow_smem<chunk_kernel<T, false>>(kSmem)) return rc;
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
      p.shape = make_shape(p.maps, a.group, a.R, a.D, false, repeated);
      if (int rc = map_keys(p.shape.wide)) return rc;
      if (int rc = launch_kernel(chunk_kernel<T, true>, grid, block, p.shape.smem, st, true, tq, tk, tv, p)) return rc;
      p.phase = 2;
      p.shape = L;
      if (int rc = map_keys(L.wide)) return rc;
      if (int rc = launch_kernel(chunk_kernel<T, true>, grid, block, L.smem, st, true, tq, tk, tv, p)) return rc;
    } else {
      if (int rc = map_keys(L.wide)) return rc;
      if (int rc = launch_kernel(chunk_kernel<T, false>, grid, block, L.smem, st, true, tq, tk, tv, p)) return rc;
    }
    const int64_t rows = 16 * a.D / 128, side = 8 * (int64_t)sm_count() / rows + 1;  // (as many CTAs as run side by side)
    if (int rc = launch_kernel(join_kernel<T>, dim3((unsigned)(tiles < side ? tiles : side), (unsigned)rows), dim3(256), 0, st,
                               false, p, !mix))
      return rc;
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
  p.odd = reinterpret_cast<int*>(at);
  at += round16(B * 4);
  p.tile_piece = reinterpret_cast<int*>(at);
  at += round16((tiles + 1) * 4);
  p.pieces = reinterpret_cast<int4*>(at);
  p.tiles_most = (int)tiles;
  p.pieces_most = (int)pieces;
  return p;
}

int chunk_attention(const ChunkArgs& a, cudaStream_t st) {
  return a.dtype == DA_BF16 ? run<__nv_bfloat16>(a, st) : run<__half>(a, st);
}

}  // namespace paged
}  // namespace da
