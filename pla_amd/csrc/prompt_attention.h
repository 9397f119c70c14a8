// What the attention over prompts and shared prefixes takes, and how its keys are dealt out.  Host and device use the same functions.
#pragma once

#include "common.h"
#include "paged_schedule.h"

namespace pla {

constexpr int PROMPT_KEYS = 64;           // of a tile
constexpr int PROMPT_ROWS = 128;          // of a block: query heads of a key-value head, token by token

// A row block of a sequence and a piece of its keys, as a workgroup takes them.
struct PromptItem {
  int n, row0, rows;                      // sequence; first row of the block, rows of the block that are there (0: no item)
  int window, keys;                       // tokens and keys of the sequence
  int pieces, piece, first;               // of the block's keys at most, this one, item of the first
  int64_t begin, key_begin;               // first token row, first key (dense)
};

struct PromptAttention {
  const uint16_t* q; int64_t q_token, q_head;
  const uint16_t* k; int64_t k_token, k_head;
  const uint16_t* v; int64_t v_token, v_head;
  const void* offsets; int offsets_wide;          // NULL: all token rows over one prefix of `lengths`[0] keys
  const void* key_offsets; int key_offsets_wide;  // dense keys
  const void* lengths; int lengths_wide;          // paged keys
  int64_t kv_block; int blocks, block_size; PagedDivisor page_of;
  const int32_t* table; int64_t table_row; int table_rows;
  const void* mapping; int mapping_wide;
  const uint16_t* gate; int64_t gate_token, gate_head;
  uint16_t* out; int64_t out_token, out_head;
  int batch, tokens, heads, group; PagedDivisor by_group;
  int64_t positions;                              // dense: rows of k; paged: positions of a row of the table
  float scale_log2; uint32_t flip;                // of the magnitude of the scale; sign bits of a pair of query values
  int items, least;                               // pieces that a head's keys are cut into (0: not at all), tiles of one at least
  int slots, slot_rows;                           // of the workspace, for each head; rows of one
  PromptItem* plan;                               // of all slots, where a call over sequences is split
  float* partial; float2* tops;                   // a slot an item and head: outputs, references and sums of its rows
  float* rows; float2* row_tops;                  // a prefix: the same of each row [token][query head], joined
};

// How keys are dealt out.  A call of many row blocks has a workgroup for each, the longest of a sequence first.  Where there are fewer, a
// block's keys are cut into pieces, so that the blocks of a long sequence do not go on when all others are done: as many as make the whole
// batch, were all blocks of a sequence as long as its last one, about `items` pieces of equal size, none under `least` tiles.  Pieces of
// different blocks begin at the same keys, so that the caches hold them for all.  The batch's lengths stand on the device, so it is there
// that the size is worked out; the host knows that blocks and pieces together are no more than blocks + items, nor than the blocks and,
// for each, every `least` tiles of the keys behind its first.
PLA_HD int prompt_tiles(int keys) { return (int)(((int64_t)keys + PROMPT_KEYS - 1) / PROMPT_KEYS); }
PLA_HD int prompt_piece(int items, int64_t total, int least) {
  if (items <= 0) return INT32_MAX;
  const int64_t even = paged_divide(total + items - 1, items);
  return (int)(even < least ? least : even < INT32_MAX ? even : INT32_MAX);
}
PLA_HD int prompt_pieces(int tiles, int most) { return tiles <= most ? 1 : (tiles - 1) / most + 1; }
// A block of `tiles` tiles in at most `most` pieces: `pieces` workgroups (one for nothing) have `tiles` each, the last one what is left.
struct PromptShare { int tiles, pieces; };
PLA_HD PromptShare prompt_share(int tiles, int most, int least) {
  const int even = (tiles + most - 1) / most, each = most == 1 || even >= least ? even : least;
  return {each, tiles <= each ? 1 : (tiles + each - 1) / each};
}

// Parts of a row's sums are brought from their maximum `m` to a common one, `top` >= m (equal infinities are no step).  The factor may
// come out zero: then a finite part has nothing left (a value of 1e38 times the smallest number would not be nothing), an infinite one
// stays, as the formula's weights are never zero.
__device__ __forceinline__ float step_factor(float m, float top) { return m == top ? 1.f : __builtin_amdgcn_exp2f(m - top); }
__device__ __forceinline__ float brought(float x, float f) { return f > 0.f || x - x == 0.f ? x * f : x; }
__device__ __forceinline__ float add_brought(float sum, float x, float f) { return f > 0.f || x - x == 0.f ? fmaf(x, f, sum) : sum + x; }

constexpr int PROMPT_PLAN = 2048;         // sequences of a call that is split at most
constexpr PLA_HD int prompt_residency(int D) { return D == 256 ? 1 : D == 64 ? 3 : 2; }       // workgroups a CU
struct PromptLaunch {
  int64_t blocks, items, pieces;                  // row blocks at most, workgroups a head, pieces (0: not split) to cut a head's keys into
  int least, slot_rows, join_rows;
  bool split, plan;                               // whether keys are cut into pieces, whether the items are listed
  int64_t tops_at, plan_at, rows_at, row_tops_at, bytes;   // workspace
};
PromptLaunch prompt_launch(int batch, int64_t tokens, int HQ, int HKV, int D, int64_t keys, bool prefix);
int check_prompt(int batch, int64_t tokens, int HQ, int HKV, int D);
// Checks what is left of the arguments and launches.
int launch_prompt(PromptAttention p, const PromptLaunch& l, bool paged, int D, float scale, int act, void* workspace, int64_t workspace_bytes, hipStream_t s);

}  // namespace pla
