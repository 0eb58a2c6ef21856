// Outer routed attention of a few new tokens a sequence over a paged cache (decoding, drafts):
//
//   Y_t = sum_s alpha_s softmax_{j <= p_t}(gamma_s <q_{s,t}, k_{s,j}>) V_j,   p_t = lengths[b] + t.
//
// Such a call reads each sequence's keys and values once and computes little: bytes bound it.  The (map, token) pairs
// of up to 16 / maps tokens of a sequence are the 16 rows of one matrix product: row (s, t) holds q's branches of map
// s and zeros in the other branches' columns, so all maps' scores come from one pass over the H R columns of a key
// tile, and all rows share the value tile.  Each row keeps its own running maximum, sum and output; the maps are
// mixed once, at the end, which needs no second pass over the keys for their sums.  (Where 8 rows hold a sequence's new
// tokens the other 8 take what the rounding of the weights left.)
//
// Work: the (sequence, 16 rows) jobs' tiles of 32 keys form one flat list, which the CTAs share evenly, whatever the
// sequences' lengths (up to 32 sequences: pieces of their own, one a CTA, where those are no longer; struct Cut).  A job
// that lies in one CTA is finished there; the pieces of one that does not leave their unnormalised rows in the
// workspace, and combine_kernel joins them in order.  Which CTA has which piece follows from the lengths alone, so both
// kernels work it out from the device's own data and the host needs no lengths.
//
// A tile: one warp brings the keys and values of 32 positions by TMA (one box each where a page has 32 positions), as
// many tiles ahead as shared memory holds.  Four warps take 8 keys each over all H R columns, keep the rows' maxima and
// sums, and hand the weights over through shared memory to four warps that take D / 4 columns each of the output, so
// that a tile's scores overlap the outputs of the one before.  (Eight warps doing both in turn: 192 us at 64 sequences of up to
// 8192, against 107.)  The products are 16 x 8 x 16 instructions: 16 rows fill them, and 128-row ones
// would spend 8 times the work on rows that do not exist.  Weights go in as two 16-bit parts, for an error of the output's own
// rounding (1.7e-3 in bf16 against 64 bits; one part 2.3e-3); in fp16 also of 2^-32 of the row's largest weight a key, half its
// smallest step (kLift).
//
// Measured (bf16, 512 value columns, joining included): 64 sequences of 4096 to 8192, 256 key columns, 609 MB, 104 us, 5.8
// TB/s, where a copy's rate would take 93 us; one sequence of 131072, 512 key columns, 268 MB, 57 us, 4.7 TB/s: two launches,
// the first tiles' way from memory and the join count there.  One token of a sequence of 512 takes 10.6 us, and five drafted
// tokens of eight sequences of up to 2008 (two maps) 21 us: latency of those steps and of a CTA's few dependent tiles.
// With 256 and 128 value columns, two CTAs an SM, 96 registers a thread and 194 to 226 bytes of spills, the 64 sequences take 98 and
// 95 us, 4.1 and 3.2 TB/s.
#include <math.h>

#include "host_util.h"
#include "paged_chunk.h"

namespace da {
namespace paged {

constexpr int kKeys = 32;      // positions a tile
constexpr int kScoreWarps = 4, kValueWarps = 4;  // and one warp that brings the tiles
constexpr int kThreads = 32 * (kScoreWarps + kValueWarps + 1);
constexpr int kMaxStages = 8;
constexpr int kPPitch = 40;    // 16-bit weights a row
constexpr float kGrow = 8.f;   // log2 of the growth of a row's maximum that its output bears
// log2 by which weights are larger than 2^(score - offset): fp16 has nothing below 2^-24, so a far tail of small weights would
// count in the fp32 sum and not in the product.  Up to 2^(kGrow + 7) = 2^15 they still fit.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f;

struct FewParams {
  Cache c;
  const void* q;
  int64_t q_branch, q_row;  // strides in elements
  const float *scales, *weights;
  void* y;
  float* part;  // [2 * CTAs][16][D] rows, then [2 * CTAs][2][16] maxima (log2) and sums
  int* status;
  int H, R, D, maps, group, lanes;  // lanes: maps rounded up to a power of two
  int job_rows;                     // 16, or 8: job_rows / lanes tokens a job
  int few_most;                     // sequences with more new tokens are another kernel's
  int few_rows, slice;              // combine_kernel's rows a sequence, columns a CTA: D, 64 or 16
  int stages, stage_bytes, key_bytes, brow;
  int ctas;
  int per_map, zero_rest;
  Plan chunks;                      // of the other kernel, if it ran
  int chunked;
};

// Tiles of one job, and of all jobs, of sequence s.
DA_DEV int job_tiles(const Cache& c, const Sequence& s) { return (int)((positions(c, s) + kKeys - 1) / kKeys); }
DA_DEV int64_t sequence_tiles(const FewParams& p, const Sequence& s, int b) {
  if (s.n == 0 || (s.n > p.few_most && !(p.chunked && left_odd(p.chunks, b)))) return 0;
  const int tokens = p.job_rows / p.lanes;
  return (int64_t)((s.n + tokens - 1) / tokens) * job_tiles(p.c, s);
}

// Tiles a CTA of `ctas`.
DA_DEV int64_t share_of(int64_t total, int ctas) {
  if (total < 0x7fff0000) return ((uint32_t)total + (uint32_t)ctas - 1) / (uint32_t)ctas;
  return (total + ctas - 1) / ctas;
}

// How up to 32 sequences' jobs are cut up, worked out by a warp (all lanes alike, but for a lane's own sequence).  Either into
// pieces of their own, one a CTA, of `share` tiles at most -- a CTA then loads one job's queries and leaves one piece -- or,
// where that takes longer pieces than even shares (their share and one tile more), into even shares of the flat list.
struct Cut {
  Sequence s;               // the lane's own
  int64_t tiles, ahead;     // of the lane's sequence, and of those before it
  int64_t total, share;
  int pieces, pieces_ahead;  // of a job of the lane's sequence (0: even shares), of the sequences before it
};

DA_DEV Cut cut(const FewParams& p) {
  const int lane = threadIdx.x % 32;
  Cut c;
  c.s = lane < p.c.B ? sequence(p.c, lane) : Sequence{0, 0, 0, true};
  c.tiles = lane < p.c.B ? sequence_tiles(p, c.s, lane) : 0;
  int64_t inc = c.tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  c.ahead = inc - c.tiles;
  c.total = __shfl_sync(0xffffffffu, inc, 31);
  c.share = share_of(c.total, p.ctas);
  c.pieces = c.pieces_ahead = 0;
  if (c.total == 0) return c;  // (all sequences are the chunk kernel's: no share to divide by)
  const int job = c.tiles ? job_tiles(p.c, c.s) : 1;
  const int64_t jobs = c.total < 0x7fffffff ? (uint32_t)c.tiles / (uint32_t)job : c.tiles / job;
  if (!__all_sync(0xffffffffu, jobs <= p.ctas)) return c;
  const int64_t least = c.share;
#pragma unroll 1
  for (int64_t share = least; share <= least + 1; ++share) {
    const int k = share < 0x7fffffff ? (int)(((uint32_t)job + (uint32_t)share - 1) / (uint32_t)share) : 1;
    int n = (int)jobs * k;  // (k is at most ctas + 1, as share is at least total / ctas)
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += u;
    }
    if (__shfl_sync(0xffffffffu, n, 31) <= p.ctas) {
      c.share = share;
      c.pieces = k;
      c.pieces_ahead = n - (int)jobs * k;
      break;
    }
  }
  return c;
}

// Sum over `threads` threads' values (all of them call it; every one gets it).  `buf` holds 32 entries.
template <int threads>
DA_DEV int64_t block_sum(int64_t v, int64_t* buf) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = v;
  __syncthreads();
  int64_t t = 0;
#pragma unroll
  for (int i = 0; i < threads / 32; ++i) t += buf[i];
  return t;
}

// D += A B for a 16 x 16 (row) and a 16 x 8 (column) matrix.
template <typename T>
DA_DEV void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

DA_DEV void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
DA_DEV void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// The pieces of one CTA, in order.  Every thread of the CTA walks them alike.
struct Walk {
  int b;
  int64_t off, left;  // tile of sequence b's list, tiles still to do
  Sequence s;         // sequence b, if known
  bool known;
};

struct Piece {
  Sequence s;
  int b, job, t0, t1;  // tiles [t0, t1) of the job's
  int tiles;           // of the whole job
};

DA_DEV bool next_piece(const FewParams& p, Walk& w, Piece& x) {
  while (w.left > 0 && w.b < p.c.B) {
    if (!w.known) w.s = sequence(p.c, w.b);
    w.known = true;
    x.s = w.s;
    const int64_t all = sequence_tiles(p, x.s, w.b);
    if (w.off < all) {
      x.b = w.b;
      x.tiles = job_tiles(p.c, x.s);
      x.job = w.off < 0x7fffffff ? (int)((uint32_t)w.off / (uint32_t)x.tiles) : (int)(w.off / x.tiles);
      x.t0 = (int)(w.off - (int64_t)x.job * x.tiles);
      x.t1 = (int)(x.t0 + w.left < x.tiles ? x.t0 + w.left : x.tiles);
      w.left -= x.t1 - x.t0;
      w.off += x.t1 - x.t0;
      return true;
    }
    ++w.b;
    w.off = 0;
    w.known = false;
  }
  return false;
}

// Positions that some row of the job sees.
DA_DEV int64_t job_end(const Cache& c, const Sequence& s, int job, int tokens) {
  const int last = min(s.n, (job + 1) * tokens);
  const int64_t e = s.held + last;
  return e < c.capacity ? e : c.capacity;
}

// kHalf: 8 rows a job.  A weight is multiplied in two parts, rounded to T and what that left: as two products, or, with 8 rows,
// in the other 8 rows of one.
// kSteps: column steps of 16 that the queries' registers hold (H R at most 16 kSteps); kNT: value columns in tiles of 8 a
// warp (D = 32 kNT); kCtas: CTAs an SM.
template <typename T, int kSteps, int kNT, int kCtas, bool kHalf>
__global__ void __launch_bounds__(kThreads, kCtas) few_kernel(const __grid_constant__ CUtensorMap tk,
                                                             const __grid_constant__ CUtensorMap tv, const FewParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], p_full[2], p_empty[2];
  __shared__ int bad[kMaxStages];  // the tile's pages are not all in the cache
  __shared__ __align__(16) uint16_t weight[2][2][16 * kPPitch];  // rounded to T, and what that left, rounded too
  __shared__ __align__(16) float warp_max[2][16][kScoreWarps];
  __shared__ float rescale[2][16], row_max[16], row_sum[kScoreWarps][16];
  __shared__ int64_t buf[32], start_off;
  __shared__ Sequence start_seq;
  __shared__ int start_b, abort_flag, piece_bad;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kValueWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&p_full[i], kScoreWarps);
      mbar_init(&p_empty[i], kValueWarps);
    }
    fence_mbar_init();
  }
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- this CTA's share of the flat list of tiles
  const int64_t used = p.zero_rest ? clamp64(p.c.starts[p.c.B], 0, p.c.tokens) : p.c.tokens;
  const int64_t before = p.zero_rest ? clamp64(p.c.starts[0], 0, used) : 0;
  int64_t total, share, begin;
  Walk walk{0, 0, 0, {0, 0, 0, true}, true};
  if (p.c.B <= 32) {  // every warp for itself, a sequence a lane
    const Cut c = cut(p);
    total = c.total;
    share = c.share;
    begin = (int64_t)blockIdx.x * share;
    int64_t off = begin - c.ahead, left = share < total - begin ? share : total - begin;
    bool here = off >= 0 && off < c.tiles;
    if (__any_sync(0xffffffffu, c.pieces)) {
      const int tiles = c.tiles ? job_tiles(p.c, c.s) : 1, piece = (int)blockIdx.x - c.pieces_ahead;
      const int length = (tiles + c.pieces - 1) / c.pieces, job = piece / c.pieces, part = piece - job * c.pieces;
      off = (int64_t)job * tiles + part * length;
      left = min(length, tiles - part * length);
      here = piece >= 0 && off < c.tiles;
      begin = __any_sync(0xffffffffu, here) ? 0 : total;
    }
    const int b = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    if (b >= 0) {
      walk.b = b;
      walk.off = __shfl_sync(0xffffffffu, off, b);
      walk.left = __shfl_sync(0xffffffffu, left, b);
      walk.s.first = __shfl_sync(0xffffffffu, c.s.first, b);
      walk.s.held = __shfl_sync(0xffffffffu, c.s.held, b);
      walk.s.n = __shfl_sync(0xffffffffu, c.s.n, b);
      walk.s.fits = __shfl_sync(0xffffffffu, (int)c.s.fits, b) != 0;
    }
    __syncthreads();  // (the barriers are initialised)
  } else {
    int64_t mine = 0;
    Sequence own{0, 0, 0, true};
    for (int b = tid; b < p.c.B; b += kThreads) mine += sequence_tiles(p, sequence(p.c, b), b);
    total = block_sum<kThreads>(mine, buf);
    share = share_of(total, p.ctas);
    begin = (int64_t)blockIdx.x * share;
    int64_t done = 0;  // tiles of the sequences before this round's
    for (int base = 0; begin < total; base += kThreads) {
      const int b = base + tid;
      int64_t v = 0;
      if (b < p.c.B) {
        own = sequence(p.c, b);
        v = sequence_tiles(p, own, b);
      }
      int64_t inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      __syncthreads();
      if (lane == 31) buf[warp] = inc;
      __syncthreads();
      int64_t at = done + inc - v, all = 0;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) {
        if (i < warp) at += buf[i];
        all += buf[i];
      }
      if (begin >= at && begin < at + v) {
        start_b = b;
        start_off = begin - at;
        start_seq = own;
      }
      done += all;
      if (begin < done) break;  // (found at the latest with the last sequence)
    }
    __syncthreads();
    if (begin < total) walk = {start_b, start_off, share < total - begin ? share : total - begin, start_seq, true};
  }
  if (before || used < p.c.tokens) {  // rows of no sequence
    const int64_t words = (int64_t)(p.per_map ? p.maps : 1) * p.D / 8, gap = (used - before) * words;
    uint4* y = static_cast<uint4*>(p.y);
    for (int64_t i = (int64_t)blockIdx.x * kThreads + tid; i < p.c.tokens * words - gap; i += (int64_t)gridDim.x * kThreads)
      y[i < before * words ? i : i + gap] = make_uint4(0, 0, 0, 0);
  }
  if (begin >= total) return;
  Abort ab{&abort_flag, p.status};
  const int tokens = p.job_rows / p.lanes;
  Piece x;
  int st = 0;         // stage of the next tile
  uint32_t phase = 0;  // of its barriers
  auto next_stage = [&]() {
    if (++st == p.stages) {
      st = 0;
      phase ^= 1;
    }
  };
  const int key_box = p.brow * 2 * p.H * p.R, value_box = p.brow * 2 * p.D, block = p.brow * 128;

  if (warp == kScoreWarps + kValueWarps) {
    // ---------------------------------------------------------------- brings the tiles
    if (lane == 0) {
      prefetch_tmap(&tk);
      prefetch_tmap(&tv);
    }
    bool ok = true;
    int brought = 0;
    const int boxes = kKeys / p.brow;
    while (ok && next_piece(p, walk, x)) {
      const int64_t end = job_end(p.c, x.s, x.job, tokens);
      const int t1 = min(x.t1, (int)((end + kKeys - 1) / kKeys));
      const int* row = p.c.table + x.b * p.c.table_stride;
      int cached = -1, entry = 0;  // this lane's entry of the 32 pages from `cached` on
      for (int t = x.t0; t < t1; ++t, ++brought, next_stage()) {
        if (lane == 0) ok = mbar_wait(&empty[st], phase ^ 1u, ab, 61);
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        if (!ok) break;
        // pages of the boxes (a box lies in one page); boxes past `end` are not fetched
        const int64_t pos = (int64_t)t * kKeys;
        const int first = (int)(pos >> p.c.page_shift);
        if (cached < 0 || first >= cached + 31) {
          cached = first;
          const int64_t i = (int64_t)first + lane;
          entry = i * p.c.page < p.c.capacity ? row[i] : -1;
        }
        int good = 0, wrong = 0, slot[2] = {-1, -1};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int64_t at = pos + u * p.brow;
          if (u >= boxes || at >= end) continue;
          const int page = __shfl_sync(0xffffffffu, entry, (int)(at >> p.c.page_shift) - cached);
          if (page < 0 || page >= p.c.pages) {
            wrong = 1;
          } else {
            slot[u] = (page << p.c.page_shift) + (int)(at & (p.c.page - 1));
            ++good;
          }
        }
        if (lane == 0) {
          bad[st] = wrong;
          mbar_arrive_expect_tx(&full[st], good * (key_box + value_box));
          uint8_t* base = smem + st * p.stage_bytes;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (slot[u] < 0) continue;
            tma_load_3d(&tk, &full[st], base + u * key_box, 0, slot[u], 0);
            tma_load_3d(&tv, &full[st], base + p.key_bytes + u * value_box, 0, slot[u], 0);
          }
        }
        __syncwarp();
      }
    }
    // the last tiles' loads land before the CTA's shared memory is given back
    if (lane == 0)
      for (int i = 0; i < min(brought, p.stages); ++i) {
        if (st-- == 0) {
          st = p.stages - 1;
          phase ^= 1;
        }
        mbar_wait_drain(&full[st], phase);
      }
    return;
  }

  const int g = lane / 4, pair = (lane % 4) * 2;
  const int map_shift = 31 - __clz(tokens), token_of = tokens - 1;
  // row r: map r >> map_shift (at least `maps`, so none, for the upper rows of kHalf), token r & token_of
  const int s0 = g >> map_shift, s1 = (g + 8) >> map_shift, k0 = g & token_of, k1 = (g + 8) & token_of;
  uint32_t tile_phase = 0;  // of p_full and p_empty, buffer `pb`
  int pb = 0;
  // (After a wait that gave up every warp still walks all pieces, its waits failing at once: the barriers meet.)

  if (warp < kScoreWarps) {
    // (queries of 512 columns take 128 registers: given by the output warps.  232 + 104, or 192 + 144, are two 168s, what
    // every warp starts with)
    if constexpr (kSteps == 32 && kNT < 16) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    if constexpr (kSteps == 32 && kNT == 16) asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // ------------------------------------------------------------------ scores and weights of 8 positions a warp
    const int steps = p.H * p.R / 16;
    const float kLog2e = 1.4426950408889634f;
    const float scale0 = s0 < p.maps ? p.scales[s0] * rsqrtf((float)p.group) * kLog2e : 0.f;
    const float scale1 = s1 < p.maps ? p.scales[s1] * rsqrtf((float)p.group) * kLog2e : 0.f;
    const uint32_t queries = smem_u32(smem + p.stages * p.stage_bytes);
    const int key = warp * 8 + (lane & 7), kr = p.brow == 32 ? key : key & 15;
    const uint32_t key_off = (p.brow == 32 ? 0 : (key >> 4) * key_box) + kr * 128 + (((lane >> 3) ^ (kr & 7)) << 4);
    while (next_piece(p, walk, x)) {
      const int64_t end = job_end(p.c, x.s, x.job, tokens);
      const int t1 = min(x.t1, (int)((end + kKeys - 1) / kKeys));
      const int64_t q0 = x.s.first + (int64_t)x.job * tokens;  // packed row of the job's first token
      const int live = min(tokens, x.s.n - x.job * tokens);
      const bool on0 = s0 < p.maps && k0 < live, on1 = s1 < p.maps && k1 < live;
      const int64_t sees0 = on0 ? min(x.s.held + x.job * tokens + k0 + 1, end) : 0;
      const int64_t sees1 = on1 ? min(x.s.held + x.job * tokens + k1 + 1, end) : 0;
      // the job's rows, each with its map's branches and zeros elsewhere, by way of shared memory
      const int row_chunks = p.H * p.R / 8;
      for (int i = tid; i < 16 * row_chunks; i += 32 * kScoreWarps) {
        const int row = i / row_chunks, c = i - row * row_chunks, h = c * 8 / p.R, s = row >> map_shift, k = row & token_of;
        const int h0 = p.H >= p.maps ? s * p.group : s * p.H / p.maps;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (s < p.maps && k < live && h >= h0 && h < h0 + p.group)
          w = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + h * p.q_branch + (q0 + k) * p.q_row + (c * 8 - h * p.R));
        st_shared_v4(queries + (c >> 3) * 2048 + sw128_offset(row, c & 7), w.x, w.y, w.z, w.w);
      }
      named_bar_sync(1, 32 * kScoreWarps);
      uint32_t qf[kSteps][4];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (i < steps) ldmatrix4(qf[i], queries + (i >> 2) * 2048 + sw128_offset(lane & 15, (i & 3) * 2 + (lane >> 4)));
        else qf[i][0] = qf[i][1] = qf[i][2] = qf[i][3] = 0;
      }
      float ref0 = -INFINITY, ref1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // rows g and g + 8: offsets, this thread's sums
      bool wrong = !x.s.fits, ok = true;
      for (int t = x.t0; t < t1; ++t, next_stage()) {
        ok &= mbar_wait(&full[st], phase, ab, 62);
        __syncwarp();
        wrong |= bad[st] != 0;
        const uint32_t kb = smem_u32(smem + st * p.stage_bytes) + key_off;
        float sc[4][4];  // four sums, so that no product waits for the one before it
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
#pragma unroll
        for (int i = 0; i < kSteps / 2; ++i) {
          if (2 * i < steps) {
            uint32_t b[4];
            ldmatrix4(b, (kb + (i >> 1) * block) ^ ((i & 1) << 6));
            mma16816<T>(sc[(2 * i) & 3], qf[2 * i], b[0], b[1]);
            mma16816<T>(sc[(2 * i + 1) & 3], qf[2 * i + 1], b[2], b[3]);
          }
        }
        const int64_t at = (int64_t)t * kKeys + warp * 8 + pair;
        const float v00 = at < sees0 ? (sc[0][0] + sc[1][0] + (sc[2][0] + sc[3][0])) * scale0 : -INFINITY;
        const float v01 = at + 1 < sees0 ? (sc[0][1] + sc[1][1] + (sc[2][1] + sc[3][1])) * scale0 : -INFINITY;
        const float v10 = at < sees1 ? (sc[0][2] + sc[1][2] + (sc[2][2] + sc[3][2])) * scale1 : -INFINITY;
        const float v11 = at + 1 < sees1 ? (sc[0][3] + sc[1][3] + (sc[2][3] + sc[3][3])) * scale1 : -INFINITY;
        float top0 = fmaxf(v00, v01), top1 = fmaxf(v10, v11);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, o));
          top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, o));
        }
        if ((lane & 3) == 0) {
          warp_max[pb][g][warp] = top0;
          warp_max[pb][g + 8][warp] = top1;
        }
        named_bar_sync(1, 32 * kScoreWarps);
        const float4 m0 = *reinterpret_cast<const float4*>(warp_max[pb][g]), m1 = *reinterpret_cast<const float4*>(warp_max[pb][g + 8]);
        top0 = fmaxf(fmaxf(m0.x, m0.y), fmaxf(m0.z, m0.w));
        top1 = fmaxf(fmaxf(m1.x, m1.y), fmaxf(m1.z, m1.w));
        float c0 = 1.f, c1 = 1.f;
        if (top0 > ref0 + kGrow || (ref0 == -INFINITY && top0 > ref0)) {
          c0 = ref0 == -INFINITY ? 1.f : ex2(ref0 - top0);
          ref0 = top0;
        }
        if (top1 > ref1 + kGrow || (ref1 == -INFINITY && top1 > ref1)) {
          c1 = ref1 == -INFINITY ? 1.f : ex2(ref1 - top1);
          ref1 = top1;
        }
        const float off0 = ref0 == -INFINITY ? 0.f : ref0 - kLift<T>, off1 = ref1 == -INFINITY ? 0.f : ref1 - kLift<T>;
        const float p00 = ex2(v00 - off0), p01 = ex2(v01 - off0), p10 = ex2(v10 - off1), p11 = ex2(v11 - off1);
        l0 = fmaf(l0, c0, p00 + p01);
        l1 = fmaf(l1, c1, p10 + p11);
        ok &= mbar_wait(&p_empty[pb], tile_phase ^ 1u, ab, 63);
        __syncwarp();
        const uint32_t w0 = pack2<T>(p00, p01), w1 = pack2<T>(p10, p11);
        const float2 r0 = unpack2<T>(w0), r1 = unpack2<T>(w1);
        const int own = g * kPPitch + warp * 8 + pair;
        *reinterpret_cast<uint32_t*>(&weight[pb][0][own]) = w0;
        *reinterpret_cast<uint32_t*>(&weight[pb][kHalf ? 0 : 1][own + (kHalf ? 8 * kPPitch : 0)]) = pack2<T>(p00 - r0.x, p01 - r0.y);
        if constexpr (!kHalf) {
          *reinterpret_cast<uint32_t*>(&weight[pb][0][own + 8 * kPPitch]) = w1;
          *reinterpret_cast<uint32_t*>(&weight[pb][1][own + 8 * kPPitch]) = pack2<T>(p10 - r1.x, p11 - r1.y);
        }
        if (warp == 0 && (lane & 3) == 0) {
          rescale[pb][g] = c0;
          rescale[pb][g + 8] = kHalf ? c0 : c1;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[pb]);
        pb ^= 1;
        tile_phase ^= pb == 0;
      }
      // ---- the piece's maxima and sums
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, o);
        l1 += __shfl_xor_sync(0xffffffffu, l1, o);
      }
      if (!ok) l0 = l1 = NAN;
      if ((lane & 3) == 0) {
        row_sum[warp][g] = l0;
        row_sum[warp][g + 8] = l1;
        if (warp == 0) {
          row_max[g] = ref0;
          row_max[g + 8] = ref1;
        }
      }
      if (tid == 0) {
        piece_bad = wrong;
        if (wrong) atomicOr(p.status, DA_DEV_BAD_PAGE);
      }
      named_bar_sync(2, 32 * (kScoreWarps + kValueWarps));
      named_bar_sync(2, 32 * (kScoreWarps + kValueWarps));  // they are read
    }
    return;
  }

  // ------------------------------------------------------------------ outputs of D / 4 columns a warp
  if constexpr (kSteps == 32 && kNT < 16) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
  if constexpr (kSteps == 32 && kNT == 16) asm volatile("setmaxnreg.dec.sync.aligned.u32 144;");
  const int w4 = warp - kScoreWarps, col0 = w4 * (kNT * 8);
  const int kr = lane & 15;  // position of a half tile (a box of 16, or half of one of 32)
  const uint32_t value_off = (col0 >> 6) * block + kr * 128 + (((((col0 & 63) >> 3) | (lane >> 4)) ^ (kr & 7)) << 4);
  const uint32_t half_off = p.brow == 32 ? 16 * 128 : value_box;
  bool first_piece = true;
  while (next_piece(p, walk, x)) {
    const int64_t end = job_end(p.c, x.s, x.job, tokens);
    const int t1 = min(x.t1, (int)((end + kKeys - 1) / kKeys));
    const int64_t q0 = x.s.first + (int64_t)x.job * tokens;
    const int live = min(tokens, x.s.n - x.job * tokens);
    float acc[kNT][4];
#pragma unroll
    for (int i = 0; i < kNT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
    bool ok = true;
    for (int t = x.t0; t < t1; ++t, next_stage()) {
      ok &= mbar_wait(&full[st], phase, ab, 64);
      const uint32_t vb = smem_u32(smem + st * p.stage_bytes) + p.key_bytes;
      const int64_t pos = (int64_t)t * kKeys;
      bool odd = false;
      // Values of positions that no row sees hold anything: 0 times them must stay 0.  A later token's value that is no
      // number stays out of the earlier tokens' rows, which 0 times it would spoil.
      const bool ragged = pos + kKeys > end, mixed = live > 1 && pos + kKeys > x.s.held + (int64_t)x.job * tokens + 1;
      if (ragged || mixed) {
        __syncwarp();
        constexpr uint32_t kExp = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
        for (int i = tid - 32 * kScoreWarps; i < kKeys * kNT * 4; i += 32 * kValueWarps) {
          const int key = i / (kNT * 4), chunk = i % (kNT * 4);
          const int box = p.brow == 32 ? 0 : key >> 4, in = p.brow == 32 ? key : key & 15;
          const uint32_t at = vb + box * value_box + (chunk >> 3) * block + sw128_offset(in, chunk & 7);
          if (pos + key >= end) {
            st_shared_v4(at, 0, 0, 0, 0);
          } else if (mixed) {
            const uint4 w = ld_shared_v4(at);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= (ws[e] & kExp) == kExp || ((ws[e] >> 16) & kExp) == kExp;
          }
        }
        fence_proxy_async();
        odd = named_bar_or(3, 32 * kValueWarps, odd);
      }
      ok &= mbar_wait(&p_full[pb], tile_phase, ab, 65);
      __syncwarp();
      const float c0 = rescale[pb][g], c1 = rescale[pb][g + 8];
      if (__any_sync(0xffffffffu, c0 != 1.f || c1 != 1.f)) {
#pragma unroll
        for (int i = 0; i < kNT; ++i) {
          acc[i][0] *= c0;
          acc[i][1] *= c0;
          acc[i][2] *= c1;
          acc[i][3] *= c1;
        }
      }
      if (odd) {
#pragma unroll 1
        for (int key = 0; key < kKeys; ++key) {
          const int own = g * kPPitch + key;
          auto part = [&](int i, int at) { return unpack2<T>(weight[pb][i][at]).x; };
          const float w0 = kHalf ? part(0, own) + part(0, own + 8 * kPPitch) : part(0, own) + part(1, own);
          const float w1 = kHalf ? 0.f : part(0, own + 8 * kPPitch) + part(1, own + 8 * kPPitch);
          const int box = p.brow == 32 ? 0 : key >> 4, in = p.brow == 32 ? key : key & 15;
#pragma unroll
          for (int i = 0; i < kNT; ++i) {
            const int col = col0 + i * 8;
            uint32_t u;
            asm volatile("ld.shared.b32 %0, [%1];"
                         : "=r"(u) : "r"(vb + box * value_box + (col >> 6) * block + sw128_offset(in, (col & 63) >> 3) + pair * 2));
            const float2 v = unpack2<T>(u);
            acc[i][0] += w0 == 0.f ? 0.f : w0 * v.x;
            acc[i][1] += w0 == 0.f ? 0.f : w0 * v.y;
            acc[i][2] += w1 == 0.f ? 0.f : w1 * v.x;
            acc[i][3] += w1 == 0.f ? 0.f : w1 * v.y;
          }
        }
      } else {
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
          uint32_t a[4], rest[4];
          const uint32_t from = smem_u32(weight[pb][0]) + ((lane & 15) * kPPitch + k2 * 16 + (lane >> 4) * 8) * 2;
          ldmatrix4(a, from);
          if constexpr (!kHalf) ldmatrix4(rest, from + 16 * kPPitch * 2);
          const uint32_t at = vb + value_off + k2 * half_off;
#pragma unroll
          for (int n2 = 0; n2 < kNT / 2; ++n2) {
            uint32_t b[4];
            ldmatrix4_trans(b, (at + (n2 >> 2) * block) ^ ((n2 & 3) << 5));
            mma16816<T>(acc[2 * n2], a, b[0], b[1]);
            mma16816<T>(acc[2 * n2 + 1], a, b[2], b[3]);
            if constexpr (!kHalf) {
              mma16816<T>(acc[2 * n2], rest, b[0], b[1]);
              mma16816<T>(acc[2 * n2 + 1], rest, b[2], b[3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&p_empty[pb]);
        mbar_arrive(&empty[st]);
      }
      pb ^= 1;
      tile_phase ^= pb == 0;
    }

    // ---- the job's output, or this piece of it
    if constexpr (kHalf) {
#pragma unroll
      for (int i = 0; i < kNT; ++i) {
        acc[i][0] += acc[i][2];
        acc[i][1] += acc[i][3];
      }
    }
    named_bar_sync(2, 32 * (kScoreWarps + kValueWarps));
    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
    for (int i = 0; i < kScoreWarps; ++i) {
      sum0 += row_sum[i][g];
      sum1 += row_sum[i][g + 8];
    }
    if (piece_bad || !ok) sum0 = sum1 = NAN;
    if (x.t1 - x.t0 == x.tiles) {
      const float w0 = s0 < p.maps ? (p.weights ? p.weights[s0] : 1.f) / sum0 : 0.f;
      const float w1 = s1 < p.maps ? (p.weights ? p.weights[s1] : 1.f) / sum1 : 0.f;
      T* y = static_cast<T*>(p.y);
#pragma unroll
      for (int i = 0; i < kNT; ++i) {
        const int col = col0 + i * 8 + pair;
        float a0 = s0 < p.maps ? acc[i][0] * w0 : 0.f, a1 = s0 < p.maps ? acc[i][1] * w0 : 0.f;
        float b0 = s1 < p.maps ? acc[i][2] * w1 : 0.f, b1 = s1 < p.maps ? acc[i][3] * w1 : 0.f;
        if (p.per_map) {
          if (s0 < p.maps && k0 < live)
            *reinterpret_cast<uint32_t*>(y + ((q0 + k0) * p.maps + s0) * p.D + col) = pack2<T>(a0, a1);
          if (s1 < p.maps && k1 < live)
            *reinterpret_cast<uint32_t*>(y + ((q0 + k1) * p.maps + s1) * p.D + col) = pack2<T>(b0, b1);
          continue;
        }
        // maps of a token: rows 8 apart (a thread's own), then 4 (lanes 16 apart), then 2
        if (!kHalf && p.lanes == 1 && k1 < live) *reinterpret_cast<uint32_t*>(y + (q0 + k1) * p.D + col) = pack2<T>(b0, b1);
        if (!kHalf && p.lanes > 1) {
          a0 += b0;
          a1 += b1;
        }
        if (p.lanes > (kHalf ? 1 : 2)) {
          a0 += __shfl_xor_sync(0xffffffffu, a0, 16);
          a1 += __shfl_xor_sync(0xffffffffu, a1, 16);
        }
        if (kHalf && p.lanes == 4) {
          a0 += __shfl_xor_sync(0xffffffffu, a0, 8);
          a1 += __shfl_xor_sync(0xffffffffu, a1, 8);
        }
        if (s0 == 0 && k0 < live) *reinterpret_cast<uint32_t*>(y + (q0 + k0) * p.D + col) = pack2<T>(a0, a1);
      }
    } else {
      const int slot = 2 * blockIdx.x + (first_piece ? 0 : 1);
      float* rows = p.part + (size_t)slot * 16 * p.D;
      const bool on0 = s0 < p.maps && k0 < live, on1 = s1 < p.maps && k1 < live;
#pragma unroll
      for (int i = 0; i < kNT; ++i) {
        const int col = col0 + i * 8 + pair;
        if (on0) *reinterpret_cast<float2*>(rows + g * p.D + col) = make_float2(acc[i][0], acc[i][1]);
        if (on1) *reinterpret_cast<float2*>(rows + (g + 8) * p.D + col) = make_float2(acc[i][2], acc[i][3]);
      }
      float* ml = p.part + (size_t)2 * p.ctas * 16 * p.D + (size_t)slot * 32;
      if (w4 == 0 && (lane & 3) == 0) {
        ml[g] = row_max[g];
        ml[g + 8] = row_max[g + 8];
        ml[16 + g] = sum0;
        ml[24 + g] = sum1;
      }
    }
    first_piece = false;
    named_bar_sync(2, 32 * (kScoreWarps + kValueWarps));  // row_max and row_sum are free again
  }
}

constexpr int kMaxPieces = 512;
struct Joining {
  float w[4][kMaxPieces], l[4][kMaxPieces];  // each map's weights and sums of the pieces
  float4 o[256];                             // the columns' sums of each warp's, or each turn's, pieces
};

// One packed row's p.slice columns from its pieces c0, c0 + 1, ...: the first in slot `slot0`, the later ones, which open
// their CTAs, in slots 2 c.  A thread takes four columns of every 1024 / p.slice-th piece.
template <typename T>
DA_DEV void join(const FewParams& p, int64_t row, int t, int c0, int pieces, int slot0, Joining& j) {
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, tokens = p.job_rows / p.lanes, across = p.slice / 4;
  const float* ml = p.part + (size_t)2 * p.ctas * 16 * p.D;
  // each map's weights of the pieces: 2^(m_c - M) / sum, times alpha
  if (warp < p.maps) {
    const int r = warp * tokens + t;
    float top = -INFINITY, sum = 0.f;
#pragma unroll 4
    for (int i = lane; i < pieces; i += 32) {
      const float* at = ml + (size_t)(i ? 2 * (c0 + i) : slot0) * 32 + r;
      const float m = at[0], l = at[16];
      j.w[warp][i] = m;
      j.l[warp][i] = l;
      top = fmaxf(top, m);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    for (int i = lane; i < pieces; i += 32) {
      const float m = j.w[warp][i], e = m == -INFINITY ? 0.f : ex2(m - top);
      sum += j.l[warp][i] * e;  // (a NaN sum, of a piece with a bad page, stays)
      j.w[warp][i] = e;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float f = (p.weights ? p.weights[warp] : 1.f) / sum;
    for (int i = lane; i < pieces; i += 32) j.w[warp][i] *= f;
  }
  __syncthreads();
  const int c4 = tid % across, col = blockIdx.y * p.slice + c4 * 4, part = tid / across, parts = 256 / across;
  T* y = static_cast<T*>(p.y);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int m = 0; m < p.maps; ++m) {
#pragma unroll 4
    for (int i = part; i < pieces; i += parts) {
      const float w = j.w[m][i];
      const float4 v = *reinterpret_cast<const float4*>(
          p.part + ((size_t)(i ? 2 * (c0 + i) : slot0) * 16 + m * tokens + t) * p.D + col);
      if (w == 0.f) continue;  // (a piece that the row does not see)
      o.x = fmaf(w, v.x, o.x);
      o.y = fmaf(w, v.y, o.y);
      o.z = fmaf(w, v.z, o.z);
      o.w = fmaf(w, v.w, o.w);
    }
    if (!p.per_map && m + 1 < p.maps) continue;
    for (int k = across; k < 32; k <<= 1) {  // (the lanes of a warp that have the same columns)
      o.x += __shfl_xor_sync(0xffffffffu, o.x, k);
      o.y += __shfl_xor_sync(0xffffffffu, o.y, k);
      o.z += __shfl_xor_sync(0xffffffffu, o.z, k);
      o.w += __shfl_xor_sync(0xffffffffu, o.w, k);
    }
    if (across >= 32) j.o[tid] = o;
    else if (lane < across) j.o[warp * across + lane] = o;
    __syncthreads();
    if (tid < across) {
      for (int i = 1; i < min(8, parts); ++i) {
        const float4 v = j.o[i * across + tid];
        o.x += v.x;
        o.y += v.y;
        o.z += v.z;
        o.w += v.w;
      }
      const int64_t at = p.per_map ? (row * p.maps + m) * p.D + col : row * p.D + col;
      *reinterpret_cast<uint2*>(y + at) = make_uint2(pack2<T>(o.x, o.y), pack2<T>(o.z, o.w));
    }
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    __syncthreads();
  }
}

// Joins the pieces of the jobs that lie in several CTAs: one CTA a packed token and p.slice columns.
template <typename T>
__global__ void __launch_bounds__(256) combine_kernel(const FewParams p) {
  __shared__ int64_t buf[32];
  __shared__ Joining j;
  const int tid = threadIdx.x, b = blockIdx.x / p.few_rows;
  // (The pieces' kernel lets this one start after it has itself waited for the kernels before it, so what those wrote --
  // the step's lengths and the chunks' plan -- may be read before the wait for the pieces.)
  const Sequence s = sequence(p.c, b);
  const bool mine = (int)(blockIdx.x % p.few_rows) < s.n && sequence_tiles(p, s, b) > 0;
  int64_t total = 0, ahead = 0;
  int job_pieces = 0, first_piece = 0;
  if (mine && p.c.B <= 32) {
    const Cut c = cut(p);
    total = c.total;
    ahead = __shfl_sync(0xffffffffu, c.ahead, b);
    job_pieces = __shfl_sync(0xffffffffu, c.pieces, b);
    first_piece = __shfl_sync(0xffffffffu, c.pieces_ahead, b);
  } else if (mine) {
    for (int i = tid; i < p.c.B; i += 256) {
      const int64_t v = sequence_tiles(p, sequence(p.c, i), i);
      total += v;
      if (i < b) ahead += v;
    }
    total = block_sum<256>(total, buf);
    ahead = block_sum<256>(ahead, buf);
  }
  grid_dependency_wait();
  grid_launch_dependents();
  if (!mine) return;
  const int64_t share = share_of(total, p.ctas);
  const int tokens = p.job_rows / p.lanes, tiles = job_tiles(p.c, s);
  for (int i = blockIdx.x % p.few_rows; i < s.n; i += p.few_rows) {
    if (job_pieces) {
      const int c = first_piece + i / tokens * job_pieces;
      if (job_pieces > 1) join<T>(p, s.first + i, i % tokens, c, job_pieces, 2 * c, j);
      continue;
    }
    const int64_t f0 = ahead + (int64_t)(i / tokens) * tiles, f1 = f0 + tiles;
    const int c0 = (int)(f0 / share), c1 = (int)((f1 - 1) / share);
    if (c0 < c1)  // (else finished where it was computed)
      join<T>(p, s.first + i, i % tokens, c0, c1 - c0 + 1, 2 * c0 + (f0 > c0 * share ? 1 : 0), j);
  }
}

}  // namespace paged
}  // namespace da

namespace {

using namespace da;

struct FewPlan {
  int stages, stage_bytes, key_bytes, smem, ctas, few_rows, job_rows;
};

// Two CTAs an SM where queries and outputs leave registers for them (H R and D up to 256): one computes while the other
// waits.  Shared memory holds as many tiles as fit.
int ctas_per_sm(int wide, int D) { return wide <= 256 && D <= 256 ? 2 : 1; }

FewPlan few_plan(int64_t tokens, int64_t B, int64_t capacity, int64_t max_new, int wide, int D, int lanes) {
  FewPlan f;
  f.job_rows = max_new * lanes <= 8 ? 8 : 16;  // a sequence's new tokens in one job, if it can be
  f.key_bytes = paged::kKeys * 2 * wide;
  f.stage_bytes = f.key_bytes + paged::kKeys * 2 * D;
  const int per_sm = ctas_per_sm(wide, D);
  f.stages = (227 * 1024 / per_sm - 1024 - 8 * 1024 - 32 * wide) / f.stage_bytes;  // (a CTA's own 1 KB, fixed buffers, alignment, queries)
  if (f.stages > paged::kMaxStages) f.stages = paged::kMaxStages;
  f.smem = f.stages * f.stage_bytes + 32 * wide + 1024;
  const int64_t rows = f.job_rows / lanes, jobs = tokens / rows + B < tokens ? tokens / rows + B : tokens;
  const int64_t tiles = (capacity + paged::kKeys - 1) / paged::kKeys;
  const int64_t most = (int64_t)sm_count() * per_sm, need = jobs * (tiles > 0 ? tiles : 1);
  f.ctas = (int)(need < most ? need : most);
  if (f.ctas < 1) f.ctas = 1;
  if (f.ctas > paged::kMaxPieces) f.ctas = paged::kMaxPieces;
  f.few_rows = (int)(max_new < 64 ? max_new : 64);
  return f;
}

int64_t few_workspace(const FewPlan& f, int D) {
  return f.ctas > 1 ? (int64_t)2 * f.ctas * (16 * D + 32) * (int64_t)sizeof(float) : 0;
}

int lanes_of(int maps) { return maps == 1 ? 1 : maps == 2 ? 2 : 4; }

bool attn_shape(int H, int R, int D, int maps) {
  if (H < 1 || R < 64 || R % 64 || maps < 1 || maps > 4 || (H % maps && maps % H)) return false;
  if (H > 512 || R > 512 || (H > maps ? H : maps) * R > 512) return false;
  return D == 128 || D == 256 || D == 512;
}

template <typename T, int kSteps, int kNT, int kCtas, bool kHalf>
int launch_few(const paged::FewParams& p, const FewPlan& f, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st) {
  if (int rc = allow_smem<paged::few_kernel<T, kSteps, kNT, kCtas, kHalf>>(219 * 1024)) return rc;
  if (int rc = launch_kernel(paged::few_kernel<T, kSteps, kNT, kCtas, kHalf>, dim3((unsigned)f.ctas), dim3(paged::kThreads), f.smem, st,
                             false, tk, tv, p))
    return rc;
  if (f.ctas == 1) return DA_OK;
  return launch_kernel(paged::combine_kernel<T>, dim3((unsigned)(p.c.B * p.few_rows), (unsigned)(p.D / p.slice)), dim3(256), 0, st,
                       false, p);
}

template <typename T, bool kHalf>
int launch_few(const paged::FewParams& p, const FewPlan& f, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st) {
  const int wide = p.H * p.R;
  if (wide <= 256)
    return p.D == 512   ? launch_few<T, 16, 16, 1, kHalf>(p, f, tk, tv, st)
           : p.D == 256 ? launch_few<T, 16, 8, 2, kHalf>(p, f, tk, tv, st)
                        : launch_few<T, 16, 4, 2, kHalf>(p, f, tk, tv, st);
  return p.D == 512   ? launch_few<T, 32, 16, 1, kHalf>(p, f, tk, tv, st)
         : p.D == 256 ? launch_few<T, 32, 8, 1, kHalf>(p, f, tk, tv, st)
                      : launch_few<T, 32, 4, 1, kHalf>(p, f, tk, tv, st);
}

template <typename T>
int launch_few(const paged::FewParams& p, const FewPlan& f, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st) {
  return p.job_rows == 8 ? launch_few<T, true>(p, f, tk, tv, st) : launch_few<T, false>(p, f, tk, tv, st);
}

}  // namespace

namespace {

// A sequence whose new tokens are one job here, 16 (map, token) rows, reads its cache once; more of them go to the chunk
// kernel, whose tiles have 128 tokens.  Eight sequences of 4096 tokens (one map of 256 columns, D 512): 8 new ones each
// 34 us here, 30 there, 32 new ones 108 and 32; one sequence of 32768, 64 new ones: 185 and 40; but one of 2048 tokens 1 new
// one: 10 here, 21 there.
int few_most(int lanes) { return 16 / lanes; }
bool has_chunks(int64_t max_new, int lanes) { return max_new > few_most(lanes); }

}  // namespace

extern "C" int64_t da_paged_attn_workspace_size(int64_t tokens, int64_t B, int64_t table_cols, int page, int64_t max_new,
                                                int H, int R, int D, int maps, int per_map) {
  if (!attn_shape(H, R, D, maps) || tokens < 0 || B < 0 || table_cols < 0 || page < 1) return -1;
  if (tokens == 0 || B == 0) return 0;
  if (max_new < 1 || max_new > tokens) max_new = tokens;
  const int lanes = lanes_of(maps);
  const int64_t chunks = has_chunks(max_new, lanes) ? paged::chunk_workspace(tokens, B, few_most(lanes), D, maps, per_map) : 0;
  return chunks + few_workspace(few_plan(tokens, B, table_cols * page, max_new, H * R, D, lanes), D);
}

extern "C" int da_paged_attn(const void* q, int64_t q_branch_stride, int64_t q_row_stride, int64_t tokens,
                             const void* key_pages, const void* value_pages, int dtype, int64_t pages, int page, int H,
                             int R, int D, int maps, const int* table, int64_t table_stride, int64_t table_cols,
                             const int* lengths, const int* starts, int64_t B, int64_t max_new, const float* scales,
                             const float* weights, int per_map, int zero_rest, void* y, void* workspace,
                             int64_t workspace_bytes, int* status, void* stream) {
  if (!q || !key_pages || !value_pages || !table || !lengths || !starts || !scales || !y || !status) return DA_ERR_NULL;
  if (dtype != DA_BF16 && dtype != DA_F16) return DA_ERR_DTYPE;
  if (!attn_shape(H, R, D, maps)) return DA_ERR_UNSUPPORTED;
  if (maps > 1 && !per_map && !weights) return DA_ERR_NULL;
  paged::FewParams p;
  if (int rc = paged::make_cache(&p.c, table, table_stride, table_cols, lengths, starts, B, tokens, pages, page)) return rc;
  for (const void* a : {q, key_pages, value_pages, (const void*)y})
    if (reinterpret_cast<uintptr_t>(a) % 16) return DA_ERR_ALIGN;
  if (q_row_stride % 8 || (H > 1 && q_branch_stride % 8)) return DA_ERR_ALIGN;
  if (tokens == 0) return DA_OK;
  if (B == 0 || B > 0x7fffffff / 64 || table_cols < 1) return DA_ERR_SHAPE;
  if (max_new < 1 || max_new > tokens) max_new = tokens;
  if (int rc = bind_device(key_pages)) return rc;
  const int lanes = lanes_of(maps);
  const bool chunked = has_chunks(max_new, lanes);
  const FewPlan f = few_plan(tokens, B, p.c.capacity, max_new, H * R, D, lanes);
  const int64_t chunk_bytes = chunked ? paged::chunk_workspace(tokens, B, few_most(lanes), D, maps, per_map) : 0;
  const int64_t need = chunk_bytes + few_workspace(f, D);
  if (workspace_bytes < need || (need && !workspace)) return DA_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return DA_ERR_ALIGN;
  p.q = q;
  p.q_branch = q_branch_stride;
  p.q_row = q_row_stride;
  p.scales = scales;
  p.weights = per_map ? nullptr : weights;
  p.y = y;
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + chunk_bytes);
  p.status = status;
  p.H = H;
  p.R = R;
  p.D = D;
  p.maps = maps;
  p.group = H >= maps ? H / maps : 1;
  p.lanes = lanes;
  p.job_rows = f.job_rows;
  p.few_most = chunked ? few_most(lanes) : 0x7fffffff;
  p.chunked = chunked;
  if (chunked) p.chunks = paged::chunk_plan(workspace, tokens, B, p.few_most);
  p.few_rows = f.few_rows < p.few_most ? f.few_rows : p.few_most;
  // The join, D 512: whole rows where sequences are many and so have few pieces each (128 sequences of 250 to 500, 4 tokens:
  // the call takes 34 us, 50 by 64 columns), narrower slices where few rows have many (one of 32000: 37 and 21 us).
  const int64_t rows = (int64_t)p.c.B * p.few_rows;
  p.slice = B >= 32 ? D : rows * (D / 64) >= sm_count() ? 64 : 16;
  p.stages = f.stages;
  p.stage_bytes = f.stage_bytes;
  p.key_bytes = f.key_bytes;
  p.brow = page < paged::kKeys ? page : paged::kKeys;
  p.ctas = f.ctas;
  p.per_map = per_map;
  p.zero_rest = zero_rest;
  const CUtensorMapDataType dt = dtype == DA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tk, tv;
  for (int i = 0; i < 2; ++i) {  // (column in its block of 64, slot, block)
    const uint64_t width = i ? D : H * R;
    const uint64_t dims[3] = {64, (uint64_t)pages * page, width / 64};
    const uint64_t strides[2] = {width * 2, 128};
    const uint32_t box[3] = {64, (uint32_t)p.brow, (uint32_t)(width / 64)};
    if (int rc = make_tmap_blocks(i ? &tv : &tk, i ? value_pages : key_pages, dt, 2, 3, dims, strides, box)) return rc;
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (chunked) {
    const paged::ChunkArgs a{p.c, q, q_branch_stride, q_row_stride, key_pages, value_pages, dtype, H, R, D, maps, p.group,
                             scales, weights, per_map, y, p.few_most, workspace, status};
    if (int rc = paged::chunk_attention(a, st)) return rc;
  }
  return dtype == DA_BF16 ? launch_few<__nv_bfloat16>(p, f, tk, tv, st) : launch_few<__half>(p, f, tk, tv, st);
}
