// How the attention over a paged cache is dealt out.  Host and device use the same functions: the host's side is arithmetic
// for tests and logs.
//
// The unit of work is a tile of TILE keys for one (request, key-value head, block of query rows).  All units of a call stand
// in one line - requests, within them heads, within them row blocks, within them tiles - and every worker (workgroup) takes
// an equal stretch of it.  So a batch of very different lengths keeps the whole chip busy to the end, and one long request is
// split as finely as there are workers, with no number of splits to choose and no length read back by the host.  A run of
// tiles that a stretch cuts is summed up in pieces: every piece leaves its rows' maxima, sums and unnormalised outputs in the
// workspace, in slot 2 w + 1 of worker w if it is the first of its run (at most one a worker: the last run it begins), in
// slot 2 w otherwise (at most one: the run its stretch begins in).
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define PLA_HD __host__ __device__ inline
#else
#define PLA_HD inline
#endif

namespace pla {

constexpr int PAGED_TILE = 128;           // keys a workgroup takes at a time, 32 a wavefront

struct PagedShape {
  int heads, group;                       // key-value heads, query heads of each
  int rows;                               // query rows of a block
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
  r.blocks = (r.window * s.group + s.rows - 1) / s.rows;
  r.tiles = r.keys > 0 ? (r.keys - 1) / PAGED_TILE + 1 : 1;
  return r;
}
PLA_HD int64_t paged_weight(const PagedShape& s, const PagedRequest& r) { return (int64_t)r.tiles * r.blocks * s.heads; }

// Keys that the token row `row / group` of a request sees (they are the first ones).
PLA_HD int paged_limit(const PagedShape& s, const PagedRequest& r, int row) {
  const int64_t limit = (int64_t)r.length - r.window + row / s.group + 1;
  return (int)(limit < 0 ? 0 : limit < r.keys ? limit : r.keys);
}

// Every worker has a unit, and from eight on their number divides by the XCDs.
PLA_HD int paged_workers(int grid, int64_t total) {
  const int n = total < grid ? (int)total : grid;
  return n >= 8 ? n & ~7 : n;
}
PLA_HD int64_t paged_stretch(int worker, int workers, int64_t total) { return worker * total / workers; }
PLA_HD int paged_worker_of(int64_t unit, int workers, int64_t total) {
  return (int)(((unit + 1) * workers + total - 1) / total - 1);
}

struct PagedSegment {
  int head, block, tile, tiles;           // tiles [tile, tile + tiles) of a run
  int slot;                               // of the workspace, -1: the run is whole
  int pieces;                             // of the run, where this is its first piece
};

// The segment that starts `offset` units into the request `r`, which is unit `unit` of the line; `end`: of the stretch.
PLA_HD PagedSegment paged_segment(const PagedRequest& r, int64_t offset, int64_t unit, int64_t end, int worker, int workers,
                                  int64_t total) {
  PagedSegment s;
  const int64_t run = offset / r.tiles;
  s.tile = (int)(offset - run * r.tiles);
  s.head = (int)(run / r.blocks);
  s.block = (int)(run - (int64_t)s.head * r.blocks);
  const int64_t left = end - unit;
  s.tiles = r.tiles - s.tile < left ? r.tiles - s.tile : (int)left;
  const bool first = s.tile == 0;
  s.slot = first && s.tiles == r.tiles ? -1 : 2 * worker + (first ? 1 : 0);
  s.pieces = first ? paged_worker_of(unit + r.tiles - 1, workers, total) - worker + 1 : 0;
  return s;
}

}  // namespace pla
