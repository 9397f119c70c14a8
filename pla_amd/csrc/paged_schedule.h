// How the attention over a paged cache is dealt out.  Host and device use the same functions: the host's side is arithmetic
// for tests and logs.
//
// The unit of work is a tile of keys, 32 for each wavefront of a workgroup that works together, 32 where wavefronts work alone, for
// one (request, key-value head, block of query rows).  All units of a call stand in one line - requests, within them heads, within them
// row blocks, within them tiles - and every worker (workgroup) takes an equal stretch of it, which wavefronts that work alone share
// out in the same way.  So a batch of very different lengths keeps the whole chip busy to the end, and one long request is split as
// finely as there are workers, with no number of splits to choose and no length read back by the host.  A run of tiles that a
// stretch cuts is summed up in pieces: every piece leaves its rows' maxima, sums and unnormalised outputs in the workspace, in slot
// 2 w + 1 of worker w if it is the first of its run (at most one a worker: the last run it begins), in slot 2 w otherwise (at most
// one: the run its stretch begins in).
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define PLA_HD __host__ __device__ inline
#else
#define PLA_HD inline
#endif

namespace pla {

// Division by a number known ahead: with 2^(b - 1) < d <= 2^b the factor ceil(2^(31 + b) / d) has 32 bits and is off by less than
// one part in 2^31, so the quotient of a number below 2^31 is exact.
struct PagedDivisor { uint32_t factor; int shift; };
inline PagedDivisor paged_divisor(int d) {
  int bits = 0;
  while ((1ll << bits) < d) ++bits;
  return {(uint32_t)(((1ull << (31 + bits)) + d - 1) / d), bits + 31};
}
PLA_HD int paged_quotient(const PagedDivisor& d, int n) { return (int)((uint64_t)(uint32_t)n * d.factor >> d.shift); }

struct PagedShape {
  int heads, group;                       // key-value heads, query heads of each
  PagedDivisor by_group;
  int row_bits, tile_bits;                // query rows of a block and keys of a tile are 2 to these
  int units, extra;                       // that a worker has at least, but for the last; that a run takes on top of its tiles
  int max_query, tokens;                  // longest window, rows of q
  int64_t positions;                      // that a row of the block table has pages for
};

struct PagedRequest {
  int64_t begin;                          // first token row
  int window, length;                     // token rows, cached tokens with them
  int keys;                               // positions below `length` that have a page
  int blocks, tiles;                      // of rows (0: the request is passed over) and of keys (at least one: rows that see
                                          // nothing are written too)
};

PLA_HD PagedRequest paged_request(const PagedShape& s, int64_t begin, int64_t end, int64_t length) {
  PagedRequest r{};
  if (begin < 0 || end <= begin || end > s.tokens || end - begin > s.max_query) return r;
  r.begin = begin;
  r.window = (int)(end - begin);
  r.length = (int)(length < 0 ? 0 : length > INT32_MAX ? INT32_MAX : length);
  r.keys = (int)(r.length < s.positions ? r.length : s.positions);
  r.blocks = (r.window * s.group + (1 << s.row_bits) - 1) >> s.row_bits;
  r.tiles = (r.keys > 0 ? ((r.keys - 1) >> s.tile_bits) + 1 : 1) + s.extra;
  return r;
}
PLA_HD int paged_weight(const PagedShape& s, const PagedRequest& r) { return r.tiles * r.blocks * s.heads; }     // fits: the host checks

// Keys that the token row `row / group` of a request sees (they are the first ones).
PLA_HD int paged_limit(const PagedShape& s, const PagedRequest& r, int row) {
  const int64_t limit = (int64_t)r.length - r.window + paged_quotient(s.by_group, row) + 1;
  return (int)(limit < 0 ? 0 : limit < r.keys ? limit : r.keys);
}

// Where the keys of half a step lie, in elements from the cache's start: place `place` of block `entry` of the table; -1: nowhere.
PLA_HD int64_t paged_place(int entry, int place, int blocks, int64_t block_stride, int64_t token_stride) {
  return entry >= 0 && entry < blocks ? entry * block_stride + place * token_stride : -1;
}

// The line of `total` units and its workers: every worker has a unit, and the first `rest` of them have one more than the others.
struct PagedLine {
  int64_t total, each;
  int workers, rest;
};
PLA_HD int64_t paged_divide(int64_t a, int64_t b) {        // of numbers that are not negative; short where they are
  return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}
PLA_HD PagedLine paged_line(const PagedShape& s, int grid, int64_t total) {
  PagedLine l{total, 0, 0, 0};
  if (total <= 0) return l;
  l.workers = total < (int64_t)grid * s.units ? ((int)total + s.units - 1) / s.units : grid;
  l.each = paged_divide(total, l.workers);
  l.rest = (int)(total - l.each * l.workers);
  return l;
}
PLA_HD int64_t paged_stretch(const PagedLine& l, int worker) { return l.each * worker + (worker < l.rest ? worker : l.rest); }
PLA_HD int paged_worker_of(const PagedLine& l, int64_t unit) {
  const int64_t longer = (l.each + 1) * l.rest;
  return (int)(unit < longer ? paged_divide(unit, l.each + 1) : l.rest + paged_divide(unit - longer, l.each));
}

// Where in a request's part of the line its unit `offset` lies.
struct PagedStart { int head, block, tile; };
PLA_HD PagedStart paged_start(const PagedRequest& r, int offset) {
  const int run = (uint32_t)offset / (uint32_t)r.tiles, head = (uint32_t)run / (uint32_t)r.blocks;
  return {head, run - head * r.blocks, offset - run * r.tiles};
}

struct PagedSegment {
  int head, block, tile, tiles;           // tiles [tile, tile + tiles) of a run
  int slot;                               // of the workspace, -1: the run is whole
  int pieces;                             // of the run (1: it is whole) where this is its first, else 0
};

// The segment that starts at `at` in the request `r`, unit `unit` of the line; `end`: of the stretch.
PLA_HD PagedSegment paged_segment(const PagedLine& l, const PagedRequest& r, const PagedStart& at, int64_t unit, int64_t end, int worker) {
  PagedSegment s{at.head, at.block, at.tile, 0, 0, 0};
  const int64_t left = end - unit;
  s.tiles = r.tiles - s.tile < left ? r.tiles - s.tile : (int)left;
  const bool whole = s.tiles == r.tiles;
  s.slot = whole ? -1 : 2 * worker + (s.tile == 0 ? 1 : 0);
  s.pieces = s.tile != 0 ? 0 : whole ? 1 : paged_worker_of(l, unit + r.tiles - 1) - worker + 1;
  return s;
}

}  // namespace pla
