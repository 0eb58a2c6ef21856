// Tile plan of the outer routed attention's forward kernels: 128 query rows a CTA pair, keys and values through stage
// rings, scores and outputs folded in TMEM.
#pragma once

#include "attn_common.h"

namespace da {
namespace attn {

constexpr int kRows = 64;       // query rows per CTA
constexpr int kMaxK = 8, kMaxV = 4, kMaxSB = 4, kMaxPB = 2;

// Tile plan.  The paired MMA reaches full rate only with N = 256 (its issue
// cost is ~46 cycles regardless of N), so a single map scores 256 keys per
// tile; mixed maps use 128-key tiles processed map by map through rotating
// TMEM score buffers.  Keys and values stream as 64-wide chunks through
// independent stage rings; everything is sized to fit 225 KB of shared
// memory and 512 TMEM columns.
struct Layout {
  int kw, nk, kchunks, rpb;
  int kbb, kslots;  // key chunks per TMA box (one issue), ring slots of kbb chunks
  int nc, npv, per;
  int q_bytes, k_stage, v_stage, p_bytes;
  int nks, nvs, nsb, npb;
  int off_q, off_k, off_v, off_p, off_red, smem;
  int tmem_s, s_cols, tmem_cols;
};

// coarse: many query tiles per SM (throughput-bound), so key boxes of up to 32 KB; otherwise every
// pair has only a few key tiles and 16 KB boxes let the first products start sooner.
// avail: bytes of shared memory to plan with.
__host__ __device__ inline Layout make_layout(int maps, int group, int R, int D, bool mix, bool coarse = true,
                                              int avail = 225 * 1024) {
  Layout L;
  L.kw = maps * group * R;
  L.rpb = R / 64;
  L.kchunks = group * L.rpb;
  L.nc = D < 256 ? D : 256;
  L.npv = D / L.nc;
  L.per = (L.nc / 2) / 64;
  L.q_bytes = kRows * L.kw * 2;
  L.v_stage = 64 * D;  // 64 keys x D/2 columns (bf16) per CTA
  // the 4 KB reduction buffer aliases P buffer 0: it is used only while no P.V product reads P
  const int red = 0;
  L.nk = 0;
  for (int nk = mix ? 128 : 256; nk >= 128 && L.nk == 0; nk -= 128) {
    const int k_stage = (nk / 2) * 128, p_bytes = kRows * nk * 2;
    const int rest = avail - L.q_bytes - 2 * p_bytes - 2 * L.v_stage - red;
    if (rest >= (nk == 256 ? 4 : 2) * k_stage) {  // 256-key tiles only with two 32 KB key boxes
      L.nk = nk;
      L.k_stage = k_stage;
      L.p_bytes = p_bytes;
      L.npb = 2;
      L.nvs = 2;
      L.nks = rest / k_stage > kMaxK ? kMaxK : rest / k_stage;
    }
  }
  if (L.nk == 0) {  // last resort: single-buffered probabilities
    L.nk = 128;
    L.k_stage = 64 * 128;
    L.p_bytes = kRows * 128 * 2;
    L.npb = 1;
    L.nvs = 2;
    const int rest = avail - L.q_bytes - L.p_bytes - 2 * L.v_stage - red;
    L.nks = rest / L.k_stage > kMaxK ? kMaxK : rest / L.k_stage;
  }
  // The value ring feeds P.V, which waits for a whole softmax tile: stages
  // moved from the key ring (while it still holds a full score tile of keys)
  // let the values of the next tile land during that softmax.
  {
    const int ring = avail - L.q_bytes - L.npb * L.p_bytes - red;  // bytes of both rings
    while (L.nvs < kMaxV) {
      const int nks = (ring - (L.nvs + 1) * L.v_stage) / L.k_stage;
      if (nks < L.kchunks * (mix ? maps : 1) || nks < 2) break;  // keep a key tile of every map
      ++L.nvs;
      L.nks = nks > kMaxK ? kMaxK : nks;
    }
  }
  // A stage costs about the same whatever its size, so key chunks of the same rows are fetched
  // several column blocks per box (up to 32 KB) while the ring keeps two boxes, one per producer.
  L.kbb = 1;
  for (int b = 4; b >= 2; b /= 2)
    if (L.rpb % b == 0 && L.nks / b >= 2 && b * L.k_stage <= (coarse ? 32768 : 16384)) {
      L.kbb = b;
      break;
    }
  L.kslots = L.nks / L.kbb;
  L.nks = L.kslots * L.kbb;
  L.s_cols = L.nk / 2;
  L.tmem_s = D / 2;
  const int nsb = (512 - D / 2) / L.s_cols;
  L.nsb = nsb > kMaxSB ? kMaxSB : nsb;
  L.off_q = 0;
  L.off_k = L.off_q + L.q_bytes;
  L.off_v = L.off_k + L.nks * L.k_stage;
  L.off_p = L.off_v + L.nvs * L.v_stage;
  L.off_red = L.off_p;  // aliases P buffer 0 (p_bytes >= 16 KB > 4 KB)
  const int used = L.off_p + L.npb * L.p_bytes;
  L.smem = used < 120 * 1024 ? 120 * 1024 : used;  // one CTA per SM
  const int cols = D / 2 + L.nsb * L.s_cols;
  L.tmem_cols = cols <= 32 ? 32 : cols <= 64 ? 64 : cols <= 128 ? 128 : cols <= 256 ? 256 : 512;
  return L;
}

}  // namespace attn
}  // namespace da
