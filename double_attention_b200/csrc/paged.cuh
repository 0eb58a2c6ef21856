// What the operators over a paged cache share: the cache and the step's sequences as the kernels see them, and the
// search of a packed token's sequence.
//
// A cache's keys lie in pages [pages, page, H, R] and its values in pages [pages, page, D]; sequence b's position j is
// slot j % page of page table[b, j / page].  A step brings starts[b + 1] - starts[b] new tokens of sequence b, packed one
// sequence after another, to the lengths[b] tokens that it has.  All of these are device data: a number that leaves the
// table or the cache is never followed; it sets DA_DEV_BAD_PAGE in the status word.
#pragma once

#include "../../include/da_b200.h"
#include "common.cuh"

namespace da {
namespace paged {

struct Cache {
  const int* table;    // [B, table_cols], rows table_stride apart
  const int* lengths;  // [B]
  const int* starts;   // [B + 1]
  int64_t table_stride;
  int64_t capacity;    // table_cols * page: positions that the table has
  int64_t tokens;      // packed rows (of which starts[B] are in use)
  int B, pages, page, page_shift;
};

// Sequence b of a step: its first packed row, its new tokens, and the tokens that it had (as far as the table goes;
// `fits` tells whether that holds all of them).
struct Sequence {
  int64_t first;
  int64_t held;
  int n;
  bool fits;
};

// Checks what the host can see of a step and fills in `c`; returns a DA_ERR_* status.
inline int make_cache(Cache* c, const int* table, int64_t table_stride, int64_t table_cols, const int* lengths,
                      const int* starts, int64_t B, int64_t tokens, int64_t pages, int page) {
  constexpr int64_t kMost = 0x7fffffff;
  if (B < 0 || B >= kMost || tokens < 0 || tokens > kMost || table_cols < 0 || table_stride < table_cols) return DA_ERR_SHAPE;
  if (page < 16 || page > 65536 || (page & (page - 1))) return DA_ERR_SHAPE;
  if (pages < 1 || pages > kMost / page || table_cols > kMost / page) return DA_ERR_SHAPE;  // slots and positions in 31 bits
  c->table = table;
  c->lengths = lengths;
  c->starts = starts;
  c->table_stride = table_stride;
  c->capacity = table_cols * page;
  c->tokens = tokens;
  c->B = (int)B;
  c->pages = (int)pages;
  c->page = page;
  c->page_shift = 0;
  while ((1 << c->page_shift) < page) ++c->page_shift;
  return DA_OK;
}

DA_DEV int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : v > hi ? hi : v; }

DA_DEV Sequence sequence(const Cache& c, int b) {
  Sequence s;
  s.first = clamp64(c.starts[b], 0, c.tokens);
  s.n = (int)(clamp64(c.starts[b + 1], s.first, c.tokens) - s.first);
  const int64_t held = c.lengths[b];
  s.fits = held >= 0 && held + s.n <= c.capacity;
  s.held = clamp64(held, 0, c.capacity);
  return s;
}

// Positions of sequence s after the step, as far as the table goes.
DA_DEV int64_t positions(const Cache& c, const Sequence& s) {
  const int64_t p = s.held + s.n;
  return p < c.capacity ? p : c.capacity;
}

// The sequence that packed row `row` belongs to (the last b with starts[b] <= row), B for a row behind the last one.
// Called by whole warps; 32 entries a step.
DA_DEV int find_sequence(const Cache& c, int64_t row) {
  const int lane = threadIdx.x % 32;
  int lo = 0, hi = c.B;  // the number of ends starts[1..B] at or before row lies in [lo, hi]
  while (hi > lo) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + (lane + 1) * step;  // end i at or before row: at least i of them
    const bool before = i <= hi && clamp64(c.starts[i], 0, c.tokens) <= row;
    const int k = __popc(__ballot_sync(0xffffffffu, before));
    const int next_hi = lo + (k + 1) * step - 1;
    lo += k * step;
    hi = next_hi < hi ? next_hi : hi;
  }
  return lo;
}

}  // namespace paged
}  // namespace da
