// What the attention over prompts and shared prefixes takes, and how its keys are dealt out.  Host and device use the same functions.
#pragma once

#include "common.h"
#include "paged_schedule.h"

namespace pla {

constexpr int PROMPT_KEYS = 64;           // of a tile

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
  int splits;
  float* partial; float2* tops;                   // pieces: [split][token][query head]
};

// Key tiles of a row block that sees `keys` keys: `pieces` workgroups have `tiles` each, the last one what is left.
struct PromptShare { int tiles, pieces; };
PLA_HD PromptShare prompt_share(int keys, int splits) {
  const int tiles = (int)(((int64_t)keys + PROMPT_KEYS - 1) / PROMPT_KEYS);
  const int even = (tiles + splits - 1) / splits, each = splits == 1 || even >= 4 ? even : 4;
  return {each, tiles <= each ? 1 : (tiles + each - 1) / each};
}

struct PromptLaunch { int rows; int64_t blocks; int splits; };          // rows of a block, blocks at most, pieces of a block's keys at most
PromptLaunch prompt_launch(int batch, int64_t tokens, int HQ, int HKV, int D, int64_t keys);
int check_prompt(int batch, int64_t tokens, int HQ, int HKV, int D);
// Workspace of the pieces: where their references and sums start behind the outputs, and all of it (`always`: where there is one piece too).
int64_t prompt_tops_at(const PromptLaunch& l, int64_t tokens, int HQ, int D);
int64_t prompt_bytes(const PromptLaunch& l, int64_t tokens, int HQ, int D, bool always);
// Checks what is left of the arguments and launches.
int launch_prompt(PromptAttention p, const PromptLaunch& l, bool paged, int HQ, int D, float scale, int act, void* workspace, int64_t workspace_bytes,
                  hipStream_t s);

}  // namespace pla
