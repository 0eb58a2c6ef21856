// What the two attention kernels over a paged cache share: which sequences each takes, and the plan of the chunks.
#pragma once

#include "paged.cuh"

namespace da {
namespace paged {

// The chunk kernel's plan, made on the device from the step's lengths: `head` is {pieces, tiles, whether a tile has several pieces, 0}; tile k, of 128 new
// tokens, has the pieces tile_piece[k] .. tile_piece[k + 1]; piece i is {sequence, tile of the sequence, first key tile, key
// tiles}, {first piece of its tile, pieces of its tile, the sequence's new tokens, whether the table holds it} and {its
// first packed row, tokens that it had, 0, 0}.  odd[b] says that live rows of sequence b came out NaN.
struct Plan {
  int* head;
  int* odd;
  int* tile_piece;
  int4* pieces;
  int tiles_most, pieces_most;
};

struct ChunkArgs {
  Cache c;
  const void* q;
  int64_t q_branch, q_row;
  const void *key_pages, *value_pages;
  int dtype, H, R, D, maps, group;
  const float *scales, *weights;
  int per_map;
  void* y;
  int few_most;  // sequences with at most that many new tokens are the other kernel's
  void* workspace;
  int* status;
};

// Bytes of the workspace for steps of `tokens` rows and B sequences (a multiple of 16).
int64_t chunk_workspace(int64_t tokens, int64_t B, int few_most, int D, int maps, bool per_map);
Plan chunk_plan(void* workspace, int64_t tokens, int64_t B, int few_most);
int chunk_attention(const ChunkArgs& a, cudaStream_t st);

// Whether the chunk kernel left NaN in live rows of sequence b, the other kernel's to compute again: a masked value that is no
// number spoils the rows of a matrix product, which weigh it with 0.
DA_DEV bool left_odd(const Plan& p, int b) { return p.odd[b] != 0; }

}  // namespace paged
}  // namespace da
