// Causal attention of prompts over their own keys, or over a paged cache that holds earlier ones too:
//
//   o = sum_p softmax_p(scale q.k_p) v_p  [* sigmoid(gate)]      over the keys p < keys - window + j + 1
//
// for token j of a window of `window` tokens at the end of `keys` keys; and of all token rows over one prefix, whose outputs the attention
// over their own keys goes on with.  The query heads of a key-value head and the tokens of the window are the rows of one product, in
// blocks of 128, 32 a wavefront, so a tile of 64 keys and values is fetched once for them.
//
//   S^T = K Q^T    keys are the rows: lane (query, half) gets the scores of its query at keys 8 i + 4 half .. + 3 of 32,
//   O^T = V^T P^T  which is the operand that the second product wants, if its contraction runs over the keys in that order; the values
//                  come out of LDS in it by transposing reads.  No weight crosses a lane, a query's maximum and sum cross one.
//
// Queries and outputs stay in registers (32 x 32 x 16 products), keys and values go to LDS past the registers, the next tile's under this
// one's products.  A row of LDS is put in an order in which both kinds of reads meet no bank twice (none counted; in the plain order of
// granules 33 % of the LDS's cycles were such, and one prompt of 32 768 tokens took 4090 us in place of 3940).  The loads of operands
// are issued four ahead of the products that take them (3990 us against 4096 where the compiler puts them right before; one prompt of 4000
// and one of 9000 tokens with heads of 256 channels 847 against 923).
//
// Two workgroups a CU (heads of 64: three; 256: one, whose registers and tiles fill it), so that one's products run under the other's
// exponentials: 64 queries a wavefront, which halves the reads of LDS but leaves room for one workgroup, take 5080 us.  Products and
// exponentials of one wavefront in a software pipeline, values a tile behind, gain nothing on top (3960).
//
// Bound by the matrix cores and, at their rate, by the power that they may draw: one prompt of 32 768 tokens (16 + 2 heads of 128) runs
// at 1.1 PFLOP/s with the clock at 1.8 GHz, a product of two 16 384 x 16 384 matrices of the library at 1.37.  Half of a heads-of-64 tile's
// time are exponentials, sums and roundings.
//
// The maximum is not followed as long as it grows by less than 2^8: the weights, in 32 bits until they are rounded, hold what it may be behind,
// and the outputs need no factor then.  Weights are rounded once, to the queries' type, to meet the values (off by half a step of it, as
// the outputs are by their own rounding; two parts would cost half as many products again).  fp16 weights are scaled by 2^7, so that the
// smallest that count are not subnormal and the largest, 2^15, is finite.
//
// Infinite and NaN values: a weight of zero times one is NaN, where the formula has no product (a key that the row does not see) or an
// infinite one (a weight that is zero only in 32 bits).  The loop does not look for them.  Where an output comes out infinite or NaN the
// workgroup runs once more, with such values taken out of the product and brought in row by row.  Finite values whose sum is not come that
// way too (bf16 reaches 3.4e38, as FP32 does): the weights are scaled by 2^-28 there, which changes no other result but those below 2^-98,
// of which digits are lost.  So does the join.  Of a prefix all rows of q are taken, and an infinite or NaN row of no request has its
// workgroup run twice as well (64 such rows beside 64 chats over a prefix of 8000 keys 90 us, finite ones 59, none 49).

#include "decode_common.h"
#include "prefill_common.h"
#include <type_traits>

#include "prompt_attention.h"

namespace pla {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
template <typename act_t> __device__ __forceinline__ f32x16_t mfma32(bf16x8_t a, bf16x8_t b, f32x16_t c);
template <> __device__ __forceinline__ f32x16_t mfma32<bf16_t>(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16_t mfma32<f16_t>(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ int64_t prompt_index(const void* base, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(base)[i] : (int64_t) static_cast<const int32_t*>(base)[i];
}
__device__ __forceinline__ int64_t lane_value(int64_t x, int lane) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)x, lane) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32);
}

// Tokens and keys of sequence n; no tokens where its offsets are not within the tensors.
template <bool PAGED>
__device__ __forceinline__ void prompt_sequence(const PromptAttention& p, int n, int64_t& begin, int& window, int64_t& key_begin, int& keys) {
  begin = prompt_index(p.offsets, p.offsets_wide, n);
  const int64_t end = prompt_index(p.offsets, p.offsets_wide, n + 1);
  bool good = begin >= 0 && end > begin && end <= p.tokens;
  int64_t length;
  if constexpr (PAGED) {
    key_begin = 0;
    length = prompt_index(p.lengths, p.lengths_wide, n);
    length = length < 0 ? 0 : length < INT32_MAX ? length : INT32_MAX;
  } else {
    key_begin = prompt_index(p.key_offsets, p.key_offsets_wide, n);
    const int64_t key_end = prompt_index(p.key_offsets, p.key_offsets_wide, n + 1);
    good = good && key_begin >= 0 && key_end >= key_begin && key_end <= p.positions;
    length = good ? key_end - key_begin : 0;
  }
  window = good ? (int)(end - begin) : 0;
  keys = (int)length;
}

__device__ __forceinline__ int prompt_blocks(const PromptAttention& p, int window) { return (int)(((int64_t)window * p.group + PROMPT_ROWS - 1) / PROMPT_ROWS); }

// Row block `index` of a call without a list of them.  Blocks of a sequence stand last one first: it has the most keys, and the shortest end the
// call.
template <bool PAGED>
__device__ __forceinline__ bool prompt_block(const PromptAttention& p, int index, PromptItem& b) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < p.batch; base += 64) {
    int64_t begin = 0, key_begin = 0;
    int window = 0, keys = 0;
    if (base + lane < p.batch) prompt_sequence<PAGED>(p, base + lane, begin, window, key_begin, keys);
    // (sequences that share rows may come to more blocks than there are workgroups)
    const int mine = prompt_blocks(p, window);
    int below = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int x = __shfl_up(below, d);
      if (lane >= d) below = min(below + x, 1 << 30);
    }
    const int all = __builtin_amdgcn_readlane(below, 63);
    if (index >= all) {
      index -= all;
      continue;
    }
    const int at = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(below > index)) - 1);
    b.n = base + at;
    b.window = __builtin_amdgcn_readlane(window, at);
    b.keys = __builtin_amdgcn_readlane(keys, at);
    b.begin = lane_value(begin, at);
    b.key_begin = lane_value(key_begin, at);
    b.row0 = (__builtin_amdgcn_readlane(below, at) - 1 - index) * PROMPT_ROWS;
    b.rows = min(PROMPT_ROWS, b.window * p.group - b.row0);
    b.pieces = 1;
    b.piece = b.first = 0;
    return true;
  }
  return false;
}

// Through the scalar cache: nothing writes the plan any more.
__device__ __forceinline__ PromptItem planned_item(const PromptAttention& p, int index) {
  typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
  const scalar_ptr x = (scalar_ptr) reinterpret_cast<const int32_t*>(p.plan + index);
  auto wide = [&](int i) { return (int64_t)((uint64_t)(uint32_t)x[i] | (uint64_t)(uint32_t)x[i + 1] << 32); };
  return PromptItem{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7], wide(8), wide(10)};
}

// Item `index` of a call over one prefix, whose blocks are alike; BY_BLOCK: its row block `index`.
template <bool BY_BLOCK>
__device__ __forceinline__ bool prefix_item(const PromptAttention& p, int index, PromptItem& b) {
  const int64_t length = prompt_index(p.lengths, p.lengths_wide, 0);
  const int keys = (int)(length < 0 ? 0 : length < p.positions ? length : p.positions), blocks = prompt_blocks(p, p.tokens), tiles = prompt_tiles(keys);
  const int pieces = prompt_pieces(tiles, prompt_piece(p.items, (int64_t)blocks * tiles, p.least));
  const int rank = BY_BLOCK ? index : index / pieces;
  if (rank >= blocks) return false;
  const int row0 = rank * PROMPT_ROWS;
  b = PromptItem{0, row0, min(PROMPT_ROWS, p.tokens * p.group - row0), p.tokens, keys, pieces, BY_BLOCK ? 0 : index - rank * pieces, rank * pieces, 0, 0};
  return true;
}

// Keys that row `row` of a sequence sees (they are the first ones).  Keys without a page count as ones that nobody sees.
__device__ __forceinline__ int prompt_limit(const PromptAttention& p, const PromptItem& b, int row) {
  const int64_t limit = p.offsets ? (int64_t)b.keys - b.window + paged_quotient(p.by_group, row) + 1 : b.keys;
  const int64_t most = b.keys < p.positions ? b.keys : p.positions;
  return (int)(limit < 0 ? 0 : limit < most ? limit : most);
}

// The list of a call's items, block by block, the last one of a sequence first.  One workgroup; the host has seen to it that there are
// no more than PROMPT_PLAN sequences.
template <bool PAGED>
__global__ __launch_bounds__(1024) void prompt_plan_kernel(const PromptAttention p) {
  __shared__ int first[PROMPT_PLAN + 1], pieces_of[PROMPT_PLAN];
  __shared__ int64_t sums[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // of `x` over all threads before this one; `all`: over all
  auto scan = [&](int64_t x, int64_t& all) {
    int64_t below = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t y = __shfl_up(below, d);
      if (lane >= d) below += y;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = below;
    __syncthreads();
    int64_t before = 0;
    all = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) before += sums[w];
      all += sums[w];
    }
    return before + below - x;
  };
  constexpr int EACH = PROMPT_PLAN / 1024;
  int64_t begin, key_begin, total = 0;
  int window[EACH], tiles[EACH], keys;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    window[i] = tiles[i] = 0;
    if (EACH * tid + i < p.batch) {
      prompt_sequence<PAGED>(p, EACH * tid + i, begin, window[i], key_begin, keys);
      tiles[i] = prompt_tiles((int)(keys < p.positions ? keys : p.positions));
    }
    total += (int64_t)prompt_blocks(p, window[i]) * tiles[i];
  }
  int64_t all, items = 0;
  scan(total, all);
  const int most = prompt_piece(p.items, all, p.least);
  int pieces[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    pieces[i] = prompt_pieces(tiles[i], most);
    items += (int64_t)prompt_blocks(p, window[i]) * pieces[i];
  }
  int64_t at = scan(items, all);
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    // (sequences that share rows may come to more items than there is room for)
    first[EACH * tid + i] = (int)(at < p.slots ? at : p.slots);
    pieces_of[EACH * tid + i] = pieces[i];
    at += (int64_t)prompt_blocks(p, window[i]) * pieces[i];
  }
  if (tid == 0) first[PROMPT_PLAN] = (int)(all < p.slots ? all : p.slots);
  __syncthreads();
  const int count = first[PROMPT_PLAN];
  for (int i = tid; i < p.slots; i += 1024) {
    PromptItem b{};
    if (i < count) {
      int low = 0, high = PROMPT_PLAN - 1;        // the last sequence that starts at or before i
      while (low < high) {
        const int mid = (low + high + 1) >> 1;
        if (first[mid] <= i) low = mid;
        else high = mid - 1;
      }
      b.n = low;
      prompt_sequence<PAGED>(p, low, b.begin, b.window, b.key_begin, b.keys);
      b.pieces = pieces_of[low];
      const int rank = (i - first[low]) / b.pieces;
      b.piece = i - first[low] - rank * b.pieces;
      b.first = i - b.piece;
      b.row0 = (prompt_blocks(p, b.window) - 1 - rank) * PROMPT_ROWS;
      b.rows = min(PROMPT_ROWS, b.window * p.group - b.row0);
      if (b.first + b.pieces > p.slots) b.rows = 0;
    }
    p.plan[i] = b;
  }
}

template <typename act_t> constexpr float PROMPT_SHIFT = 0.f;
template <> constexpr float PROMPT_SHIFT<f16_t> = 7.f;
constexpr float PROMPT_SLACK = 8.f;
template <typename act_t> constexpr float PROMPT_ROOM = 0.f;        // of a second run's weights: 2^20 of the largest values are finite
template <> constexpr float PROMPT_ROOM<bf16_t> = 28.f;

__device__ __forceinline__ float halves_max(float x) {
  const LanePair a = swap_halves(x);
  return fmaxf(a.lo, a.hi);
}
__device__ __forceinline__ float halves_sum(float x) {
  const LanePair a = swap_halves(x);
  return a.lo + a.hi;
}

typedef const __attribute__((address_space(3))) unsigned char* lds_bytes;
__device__ __forceinline__ bf16x8_t lds_operand(uint32_t at) {
  return __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>((lds_bytes)(uintptr_t)at));
}
__device__ __forceinline__ i16x4_t lds_transposed(uint32_t at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(lds_bytes)(uintptr_t)at);
}

template <typename act_t> __device__ __forceinline__ uint32_t all_exponent(uint32_t pair) {      // 0xffff in each half that is infinite or NaN
  const uint32_t mask = __is_same(act_t, bf16_t) ? 0x7f80u : 0x7c00u;
  return ((pair & mask) == mask ? 0xffffu : 0u) | ((pair >> 16 & mask) == mask ? 0xffff0000u : 0u);
}

template <typename act_t, int D, bool PAGED>
__global__ __launch_bounds__(256, prompt_residency(D)) void prompt_attention_kernel(const PromptAttention p) {
  constexpr int KEYS = PROMPT_KEYS, STEPS = D / 16, TILES = D / 32, PITCH = 2 * D, TILE = KEYS * PITCH;
  constexpr int LANES = PITCH / 16, ROWS_A_COPY = 64 / LANES, COPIES = 16 / ROWS_A_COPY;           // of 16 keys or values, by a wavefront
  __shared__ __align__(1024) unsigned char tiles[2][2][TILE];         // keys and values
  __shared__ uint32_t there[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int index = blockIdx.x / p.heads, head = blockIdx.x - index * p.heads;
  PromptItem b;
  if (p.plan) b = planned_item(p, index);
  else if (!(PAGED && !p.offsets ? prefix_item<false>(p, index, b) : prompt_block<PAGED>(p, index, b))) return;
  if (b.rows == 0) return;
  const int tiles_seen = prompt_tiles(prompt_limit(p, b, b.row0 + b.rows - 1));
  const PromptShare share = prompt_share(tiles_seen, b.pieces, p.least);
  if (b.piece >= share.pieces) return;
  const int first_tile = b.piece * share.tiles, last_tile = min(first_tile + share.tiles, tiles_seen);
  const int copy_row = lane / LANES, granule = lane % LANES;
  auto key_swizzle = [](int r) { return D == 64 ? (r >> 1 & 3) | (r >> 4 & 1) << 2 : (r & 7) | (r >> 4 & 1) << 3; };
  auto value_swizzle = [](int r) { return D == 64 ? 4 * (r >> 1 & 1) : 4 * (r & 3); };
  // Copies: wavefront w has keys and values 16 w .. + 15 of a tile.
  uint32_t k_off[COPIES], v_off[COPIES];
#pragma unroll
  for (int c = 0; c < COPIES; ++c) {
    const int r = ROWS_A_COPY * c + copy_row;
    k_off[c] = (uint32_t)(r * p.k_token * 2) + 16 * (granule ^ key_swizzle(16 * wave + r));
    v_off[c] = (uint32_t)(r * p.v_token * 2) + 16 * (granule ^ value_swizzle(r));
  }
  const uint32_t lds = lds_address(&tiles[0][0][0]);
  // Operands: K rows are keys, lane (col, half) reads granule 2 s + half of key 32 t + col; values four keys and sixteen channels a
  // group of 16 lanes.
  const uint32_t k_at = lds + col * PITCH + 16 * (half ^ key_swizzle(col));
  const int v_row = 4 * half + ((lane & 15) >> 2);
  const uint32_t v_at = lds + TILE + v_row * PITCH + 16 * ((2 * (lane >> 4 & 1) + ((lane & 3) >> 1)) ^ value_swizzle(v_row)) + 8 * (lane & 1);

  // This wavefront's rows; those past the end repeat the last one.
  const int row = b.row0 + min(32 * wave + col, b.rows - 1), limit = prompt_limit(p, b, row);
  const int j = paged_quotient(p.by_group, row), query_head = head * p.group + row - j * p.group;
  const int64_t token = b.begin + j;
  const bool real = 32 * wave + col < b.rows, mine = 32 * wave < b.rows;
  bf16x8_t q[STEPS];
  {
    const uint16_t* src = p.q + token * p.q_token + query_head * p.q_head + 8 * half;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      u32x4_t x = *reinterpret_cast<const u32x4_t*>(src + 16 * s);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] ^= p.flip;
      q[s] = __builtin_bit_cast(bf16x8_t, x);
    }
  }
  const int least = __builtin_amdgcn_readfirstlane(prompt_limit(p, b, b.row0 + min(32 * wave, b.rows - 1)));
  const int most = __builtin_amdgcn_readfirstlane(prompt_limit(p, b, b.row0 + min(32 * wave + 31, b.rows - 1)));
  bool has_row = true;
  const int32_t* pages = nullptr;
  if constexpr (PAGED) {
    const int64_t table_row = p.mapping ? prompt_index(p.mapping, p.mapping_wide, b.n) : b.n;
    has_row = table_row >= 0 && table_row < p.table_rows;
    pages = uniform_pointer(p.table + (has_row ? table_row : 0) * p.table_row);
  }
  const int keys = min((int64_t)b.keys, p.positions);
  auto group_of = [&](int tile) { return min(tile * KEYS + 16 * wave, max(keys - 1, 0) & ~15); };
  auto page_entry = [&](int tile) {
    if (!PAGED || !has_row || keys == 0) return -1;
    return *(const __attribute__((address_space(4))) int32_t*)(pages + paged_quotient(p.page_of, group_of(tile)));
  };
  // A tile's keys and values; those behind the sequence repeat its last one.
  const uint16_t* k_base = p.k + head * p.k_head + (PAGED ? 0 : b.key_begin * p.k_token);
  const uint16_t* v_base = p.v + head * p.v_head + (PAGED ? 0 : b.key_begin * p.v_token);
  auto copy_tile = [&](int tile, int buffer, int entry) {
    const uint32_t to = lds + buffer * 2 * TILE + wave * 16 * PITCH;
    const int key0 = group_of(tile);
    int last = keys - 1 - key0;
    uint64_t k_at = (uint64_t)(uint32_t)key0 * (uint32_t)p.k_token, v_at = (uint64_t)(uint32_t)key0 * (uint32_t)p.v_token;
    if constexpr (PAGED) {
      const bool ok = entry >= 0 && entry < p.blocks;
      const int place = key0 - paged_quotient(p.page_of, key0) * p.block_size;
      k_at = ok ? entry * p.kv_block + (uint64_t)(uint32_t)place * (uint32_t)p.k_token : 0;
      v_at = k_at;
      last = ok ? last : 15;
      if (lane == 0) reinterpret_cast<unsigned char*>(&there[buffer])[wave] = ok;
    }
    const char *k_from = uniform_pointer(reinterpret_cast<const char*>(k_base + k_at)), *v_from = uniform_pointer(reinterpret_cast<const char*>(v_base + v_at));
    if (last >= 15) {
#pragma unroll
      for (int c = 0; c < COPIES; ++c) dma16(k_from, k_off[c], to + 1024 * c);
#pragma unroll
      for (int c = 0; c < COPIES; ++c) dma16(v_from, v_off[c], to + TILE + 1024 * c);
    } else {
#pragma unroll
      for (int c = 0; c < COPIES; ++c) {
        const int back = max(ROWS_A_COPY * c + copy_row - last, 0);
        dma16(k_from, k_off[c] - (uint32_t)(back * p.k_token * 2), to + 1024 * c);
        dma16(v_from, v_off[c] - (uint32_t)(back * p.v_token * 2), to + TILE + 1024 * c);
      }
    }
  };
  f32x16_t o[TILES];
  float top, sum;

  auto pass = [&](auto careful) {
    constexpr bool CAREFUL = decltype(careful)::value;
    top = -INFINITY;
    sum = 0.f;
#pragma unroll
    for (int c = 0; c < TILES; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[c][i] = 0.f;
    auto sees = [&](int key0, uint32_t flags, int h, int i) {
      const int key = 32 * h + 8 * (i / 4) + 4 * half + (i & 3);
      return (key0 + key < limit) & ((flags >> (8 * (2 * h + i / 8)) & 1) != 0);
    };
    constexpr int HALVES = KEYS / 32;
    constexpr uint32_t ALL = 0x01010101u;
    f32x16_t s[HALVES];
    auto scores = [&](int buffer) {
      const uint32_t kb = k_at + buffer * 2 * TILE;
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[h][i] = 0.f;
#pragma unroll
      for (int c = 0; c < STEPS; ++c)
#pragma unroll
        for (int h = 0; h < HALVES; ++h) s[h] = mfma32<act_t>(lds_operand((kb ^ (32u * c)) + h * 32 * PITCH), q[c], s[h]);
      if constexpr (!CAREFUL) {
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int i = 0; i < STEPS * HALVES - 4; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
      }
    };
    auto product = [&](int buffer, int key0, uint32_t flags, const bf16x8_t (&weight)[2 * HALVES]) {
      const uint32_t vb = v_at + buffer * 2 * TILE;
#pragma unroll
      for (int x = 0; x < 2 * HALVES; ++x)
#pragma unroll
        for (int c = 0; c < TILES; ++c) {
          const uint32_t at = (vb ^ (64u * c)) + 16 * x * PITCH;
          const i16x4_t v0 = lds_transposed(at), v1 = lds_transposed(at + 8 * PITCH);
          typedef short i16x8_t __attribute__((ext_vector_type(8)));
          bf16x8_t v = __builtin_bit_cast(bf16x8_t, i16x8_t{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
          if constexpr (CAREFUL) {
            // Infinite and NaN values leave the product.  Where one is, products of marks with marks of the keys that a row sees say
            // which rows get it: marks of positive infinities, marks of negative ones, NaN as both.
            u32x4_t w = __builtin_bit_cast(u32x4_t, v), plus, minus;
            uint32_t any = 0;
            const uint32_t one = __is_same(act_t, bf16_t) ? 0x3f803f80u : 0x3c003c00u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t bad = all_exponent<act_t>(w[i]), mantissa = __is_same(act_t, bf16_t) ? 0x007fu : 0x03ffu;
              const uint32_t nan = bad & (((w[i] & mantissa) ? 0xffffu : 0u) | ((w[i] >> 16 & mantissa) ? 0xffff0000u : 0u));
              const uint32_t negative = ((w[i] & 0x8000u) ? 0xffffu : 0u) | ((w[i] & 0x80000000u) ? 0xffff0000u : 0u);
              plus[i] = one & bad & (nan | ~negative);
              minus[i] = one & bad & (nan | negative);
              any |= bad;
              w[i] &= ~bad;
            }
            v = __builtin_bit_cast(bf16x8_t, w);
            if (__ballot(any != 0) != 0) {
              u32x4_t marks;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                marks[i] = one & ((sees(key0, flags, x / 2, 8 * (x & 1) + 2 * i) ? 0xffffu : 0u) | (sees(key0, flags, x / 2, 8 * (x & 1) + 2 * i + 1) ? 0xffff0000u : 0u));
              f32x16_t up, down;
#pragma unroll
              for (int i = 0; i < 16; ++i) up[i] = down[i] = 0.f;
              up = mfma32<act_t>(__builtin_bit_cast(bf16x8_t, plus), __builtin_bit_cast(bf16x8_t, marks), up);
              down = mfma32<act_t>(__builtin_bit_cast(bf16x8_t, minus), __builtin_bit_cast(bf16x8_t, marks), down);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[c][i] += (up[i] > 0.f ? INFINITY : 0.f) + (down[i] > 0.f ? -INFINITY : 0.f);
            }
          }
          o[c] = mfma32<act_t>(v, weight[x], o[c]);
        }
    };
    // Scores to weights, with the sum; returns the factor of what was summed before.
    auto raise = [&](int key0, uint32_t flags) {
      if (key0 + KEYS > least || flags != ALL) {
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[h][i] = sees(key0, flags, h, i) ? s[h][i] : -INFINITY;
      }
      float high = fmaxf(s[0][0], s[HALVES - 1][0]);
#pragma unroll
      for (int i = 1; i < 16; ++i) high = fmaxf(fmaxf(s[0][i], s[HALVES - 1][i]), high);
      high = halves_max(high) * p.scale_log2;
      const float now = high > top + PROMPT_SLACK ? high : top, f = step_factor(top, now);
      top = now;
      return f;
    };
    auto weigh = [&](float f, bf16x8_t (&weight)[2 * HALVES]) {
      const float zero = (top == -INFINITY ? 0.f : top) - PROMPT_SHIFT<act_t>;
      float part[2] = {sum * f, 0.f};
#pragma unroll
      for (int x = 0; x < 2 * HALVES; ++x) {
        u32x4_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float low = __builtin_amdgcn_exp2f(fmaf(s[x / 2][8 * (x & 1) + 2 * i], p.scale_log2, -zero));
          float high = __builtin_amdgcn_exp2f(fmaf(s[x / 2][8 * (x & 1) + 2 * i + 1], p.scale_log2, -zero));
          if constexpr (CAREFUL && PROMPT_ROOM<act_t> != 0.f) {
            low *= __builtin_ldexpf(1.f, -(int)PROMPT_ROOM<act_t>);
            high *= __builtin_ldexpf(1.f, -(int)PROMPT_ROOM<act_t>);
          }
          part[0] += low;
          part[1] += high;
          w[i] = pack2<act_t>(low, high);
        }
        weight[x] = __builtin_bit_cast(bf16x8_t, w);
      }
      sum = part[0] + part[1];
    };
    int entry = page_entry(first_tile);
    if (first_tile < last_tile) copy_tile(first_tile, 0, entry);
    entry = page_entry(first_tile + 1);
    for (int tile = first_tile; tile < last_tile; ++tile) {
      const int buffer = (tile - first_tile) & 1, key0 = tile * KEYS;
      wait_vmcnt<0>();
      lds_barrier();
      if (tile + 1 < last_tile) {
        copy_tile(tile + 1, buffer ^ 1, entry);
        entry = page_entry(tile + 2);
      }
      if (!mine || key0 >= most) continue;
      uint32_t flags = ALL;
      if constexpr (PAGED) flags = __builtin_amdgcn_readfirstlane(there[buffer]);
      scores(buffer);
      const float f = raise(key0, flags);
      if (__ballot(f != 1.f) != 0) {
#pragma unroll
        for (int c = 0; c < TILES; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[c][i] = CAREFUL ? brought(o[c][i], f) : o[c][i] * f;         // (zero times an infinity: there is another run)
      }
      bf16x8_t weight[2 * HALVES];
      weigh(f, weight);
      product(buffer, key0, flags, weight);
      if constexpr (!CAREFUL && D == 256) {       // (827 -> 815 us; smaller heads, of which a CU has more wavefronts, gain nothing)
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 1);
#pragma unroll
        for (int i = 0; i < 2 * HALVES * TILES - 4; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 4, 1);
      }
    }
    top -= PROMPT_SHIFT<act_t> - (CAREFUL ? PROMPT_ROOM<act_t> : 0.f);
  };
  pass(std::false_type{});
  // A NaN may be one of the formula's, or an infinite or NaN value whose weight is zero: once more, with such values apart.
  float check = 0.f;
#pragma unroll
  for (int c = 0; c < TILES; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) check += o[c][i] * 0.f;
  if (__syncthreads_or(check != check)) pass(std::true_type{});
  if (!mine) return;
  const float total = halves_sum(sum);
  if (share.pieces > 1 || !p.offsets) {
    const int64_t at = share.pieces == 1 ? token * (p.heads * p.group) + query_head
                                         : ((int64_t)(b.first + b.piece) * p.heads + head) * p.slot_rows + 32 * wave + col;
    float* to = (share.pieces == 1 ? p.rows : p.partial) + at * D;
    if (real) {
#pragma unroll
      for (int c = 0; c < TILES; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(to + 32 * c + 8 * i + 4 * half) = float4{o[c][4 * i], o[c][4 * i + 1], o[c][4 * i + 2], o[c][4 * i + 3]};
      if (half == 0) (share.pieces == 1 ? p.row_tops : p.tops)[at] = float2{top, total};
    }
  } else {
    const float norm = total == 0.f ? 0.f : 1.0f / total;         // no key: zeros
#pragma unroll
    for (int c = 0; c < TILES; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        // lane half 0 gets channels 16 x .. + 7 of the 32, half 1 the next eight
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float low = o[c][8 * x + i], high = o[c][8 * x + 4 + i];
          const auto w = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, low), __builtin_bit_cast(uint32_t, high), false, false);
          const uint32_t first = w[0], second = w[1];
          y[i] = __builtin_bit_cast(float, first) * norm;
          y[4 + i] = __builtin_bit_cast(float, second) * norm;
        }
        if (!real) continue;
        const int channel = 32 * c + 16 * x + 8 * half;
        if (p.gate) {
          const u32x4_t g4 = *reinterpret_cast<const u32x4_t*>(p.gate + token * p.gate_token + query_head * p.gate_head + channel);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[2 * i] *= 1.0f / (1.0f + __expf(-lo16<act_t>(g4[i])));
            y[2 * i + 1] *= 1.0f / (1.0f + __expf(-hi16<act_t>(g4[i])));
          }
        }
        *reinterpret_cast<uint4*>(p.out + token * p.out_token + query_head * p.out_head + channel) =
            make_uint4(pack2<act_t>(y[0], y[1]), pack2<act_t>(y[2], y[3]), pack2<act_t>(y[4], y[5]), pack2<act_t>(y[6], y[7]));
      }
  }
}

// Pieces of a row block to its output, or (a prefix) to one piece for each row: a wavefront a row at a time, a lane D / 64 channels.
// Four pieces are in flight (parts of prompts with heads of 64, three or four pieces a block, 142 us; eight, twice the loads, 149).
template <typename act_t, int D>
__global__ __launch_bounds__(256) void prompt_join_kernel(const PromptAttention p) {
  constexpr int LANE = D / 64, AHEAD = 4;
  typedef float lane_t __attribute__((ext_vector_type(LANE)));
  const int index = blockIdx.x / p.heads, head = blockIdx.x - index * p.heads;
  PromptItem b;
  if (p.plan) b = planned_item(p, index);
  else if (!prefix_item<true>(p, index, b)) return;
  if (b.rows == 0 || b.piece != 0 || b.pieces < 2) return;
  const PromptShare share = prompt_share(prompt_tiles(prompt_limit(p, b, b.row0 + b.rows - 1)), b.pieces, p.least);
  if (share.pieces < 2) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int r = blockIdx.y * 4 + wave; r < b.rows; r += 4 * gridDim.y) {
    const int j = paged_quotient(p.by_group, b.row0 + r), query_head = head * p.group + b.row0 + r - j * p.group;
    const int64_t token = b.begin + j, first = ((int64_t)b.first * p.heads + head) * p.slot_rows + r, step = (int64_t)p.heads * p.slot_rows;
    float top, sum;
    lane_t o;
    auto put_together = [&](float room) {
      top = -INFINITY;
      sum = 0.f;
      o = lane_t{};
      for (int i = 0; i < share.pieces; i += AHEAD) {
        float2 y[AHEAD];
        lane_t x[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          const int64_t at = first + min(i + a, share.pieces - 1) * step;
          y[a] = p.tops[at];
          x[a] = *reinterpret_cast<const lane_t*>(p.partial + at * D + LANE * lane);
        }
        float now = top;
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) now = fmaxf(now, y[a].x);          // one piece twice does no harm here
        const float back = step_factor(top, now);
        sum *= back;
#pragma unroll
        for (int c = 0; c < LANE; ++c) o[c] = brought(o[c], back);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          const bool counts = i + a < share.pieces;
          const float f = step_factor(y[a].x, now) * room;
          sum = counts ? fmaf(y[a].y, f, sum) : sum;
#pragma unroll
          for (int c = 0; c < LANE; ++c) o[c] = counts ? add_brought(o[c], x[a][c], f) : o[c];
        }
        top = now;
      }
    };
    put_together(1.f);
    if constexpr (PROMPT_ROOM<act_t> != 0.f) {
      // Finite pieces whose sum is not: once more, scaled as a piece's own sums are.
      float check = 0.f;
#pragma unroll
      for (int c = 0; c < LANE; ++c) check += o[c] * 0.f;
      if (__ballot(check != check) != 0) {
        put_together(__builtin_ldexpf(1.f, -(int)PROMPT_ROOM<act_t>));
        top += PROMPT_ROOM<act_t>;
      }
    }
    if (!p.offsets) {
      const int64_t at = token * (p.heads * p.group) + query_head;
      *reinterpret_cast<lane_t*>(p.rows + at * D + LANE * lane) = o;
      if (lane == 0) p.row_tops[at] = float2{top, sum};
      continue;
    }
    const float norm = sum == 0.f ? 0.f : 1.0f / sum;
    float y[LANE];
#pragma unroll
    for (int c = 0; c < LANE; ++c) {
      y[c] = o[c] * norm;
      if (p.gate) y[c] *= 1.0f / (1.0f + __expf(-to_float(act_t{p.gate[token * p.gate_token + query_head * p.gate_head + LANE * lane + c]})));
    }
    uint16_t* dst = p.out + token * p.out_token + query_head * p.out_head + LANE * lane;
    if constexpr (LANE == 1) *dst = from_float<act_t>(y[0]).bits;
    else if constexpr (LANE == 2) *reinterpret_cast<uint32_t*>(dst) = pack2<act_t>(y[0], y[1]);
    else *reinterpret_cast<uint2*>(dst) = uint2{pack2<act_t>(y[0], y[1]), pack2<act_t>(y[2], y[3])};
  }
}

template <typename act_t, int D, bool PAGED>
static void launch_prompt(const PromptAttention& p, const PromptLaunch& l, hipStream_t s) {
  if (p.plan) prompt_plan_kernel<PAGED><<<1, 1024, 0, s>>>(p);
  prompt_attention_kernel<act_t, D, PAGED><<<dim3((unsigned)(l.items * p.heads)), 256, 0, s>>>(p);
  if (l.split) prompt_join_kernel<act_t, D><<<dim3((unsigned)((p.plan ? l.items : l.blocks) * p.heads), (unsigned)l.join_rows), 256, 0, s>>>(p);
}
template <bool PAGED>
static void launch_prompt(const PromptAttention& p, const PromptLaunch& l, int D, int act, hipStream_t s) {
  if (act == PLA_BF16) {
    if (D == 64) launch_prompt<bf16_t, 64, PAGED>(p, l, s);
    else if (D == 128) launch_prompt<bf16_t, 128, PAGED>(p, l, s);
    else launch_prompt<bf16_t, 256, PAGED>(p, l, s);
  } else {
    if (D == 64) launch_prompt<f16_t, 64, PAGED>(p, l, s);
    else if (D == 128) launch_prompt<f16_t, 128, PAGED>(p, l, s);
    else launch_prompt<f16_t, 256, PAGED>(p, l, s);
  }
}

PromptLaunch prompt_launch(int batch, int64_t tokens, int HQ, int HKV, int D, int64_t keys, bool prefix) {
  PromptLaunch l{};
  const int64_t rows = tokens * (HQ / HKV);
  // a sequence has a block that is not full, and there are no more blocks than rows
  l.blocks = prefix ? (rows + PROMPT_ROWS - 1) / PROMPT_ROWS : rows / PROMPT_ROWS + batch;
  if (l.blocks > rows) l.blocks = rows;
  l.least = prefix ? 4 : 8;
  // Pieces and blocks together fill the chip twice: an unequal end costs less than twice the pieces, which are written and read again.  1500
  // tokens over 60 000 keys 1542 us (three times 1572, four 1574, not split 1650), eighteen parts of prompts with heads of 64 145 (155, 169,
  // 163).  A prefix's blocks are alike and end together: once (100 windows of four over 30 000 keys 96 us, twice 115, half 104), with very few
  // rows, whose pieces are as large as the prefix, half: 64 chats over 8000 keys, 32 + 8 heads of 128, 49.5, once 52.7; heads of 64 44.4 and
  // 43.7, of 256 (16 chats) 56.6 and 51.9.  Above the line: 96 chats, heads of 128, half 62.8, once 63.8; 64, heads of 256, 94.8 and 79.6.
  //
  // Whether keys are cut is decided by what the host knows, all keys of the call or the positions of a row of the table.  With 16 + 2 heads of
  // 128: 100 tokens over 1100 keys 29.8 us (not split 24.8), 1500 30.6 (31.2), 2000 32.8 (39.8), 4000 41 (72); heads of 256 over 1500 41.5
  // (56.7).  It costs where no sequence is long, or its blocks fill the chip by half: nine prompts of 120 tokens 18.2 (8.7), one of 1100
  // 37.6 (24.9), of 3000 85 (61), of 5000 124 (114).  From 513 keys on, rather than 1025: 100 tokens over 900 29.2 (20.8).
  const int64_t room = 256 * prompt_residency(D), groups = l.blocks * HKV;
  const int64_t fill = (!prefix || groups > room / 2 ? 2 * room : groups > room / 32 ? room : room / 2) / HKV - l.blocks;
  l.split = prefix || (groups < 2 * room && batch <= PROMPT_PLAN && keys > 2 * l.least * PROMPT_KEYS);
  l.pieces = !l.split ? 0 : fill > 1 ? fill : 1;
  // Room for them, and workgroups: no block has more pieces than its keys have `least` tiles for, whatever the chip could take.  (A
  // prefix has room for any length.)
  const int64_t allowed = l.blocks * (((keys + PROMPT_KEYS - 1) / PROMPT_KEYS - 1) / l.least);
  l.items = l.blocks + (!prefix && l.pieces > allowed ? allowed : l.pieces);
  // A list of the items: for pieces, and where every workgroup would look through many sequences for its own (prompts of 64 tokens, 16 + 2
  // heads: 128 of them 28.5 us with a list and 25.2 without, 300 54 and 61, 1000 161 and 279), unless it is long itself.
  l.plan = !prefix && (l.split || (batch > 192 && batch <= PROMPT_PLAN && l.blocks <= 8192));
  l.slot_rows = (int)(rows < PROMPT_ROWS ? rows : PROMPT_ROWS);
  // Rows of a block at once: all where few blocks have many pieces (64 chats over 8000 keys 62.6 us, a quarter at once 72).
  l.join_rows = (l.slot_rows + (prefix ? 3 : 15)) / (prefix ? 4 : 16);
  if (l.split || l.plan) {
    int64_t at = l.split ? l.items * HKV * l.slot_rows * D * 4 : 0;
    auto take = [&](int64_t bytes) {
      const int64_t here = at;
      at += (bytes + 255) / 256 * 256;
      return here;
    };
    l.tops_at = take(l.split ? l.items * HKV * l.slot_rows * 8 : 0);
    l.plan_at = take(l.plan ? l.items * (int64_t)sizeof(PromptItem) : 0);
    l.rows_at = take(prefix ? tokens * HQ * D * 4 : 0);
    l.row_tops_at = take(prefix ? tokens * HQ * 8 : 0);
    l.bytes = at;
  }
  return l;
}

int check_prompt(int batch, int64_t tokens, int HQ, int HKV, int D) {
  PLA_REQUIRE(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256, got %d", D);
  PLA_REQUIRE(HKV > 0 && HQ >= HKV && HQ % HKV == 0, "query heads must be a positive multiple of key-value heads");
  PLA_REQUIRE(batch >= 0 && tokens >= 0 && tokens <= (1 << 30) / HQ, "too many rows");
  PLA_REQUIRE((tokens * (HQ / HKV) / PROMPT_ROWS + batch) * HKV < (1 << 23), "too many sequences");
  return 0;
}

int launch_prompt(PromptAttention p, const PromptLaunch& l, bool paged, int D, float scale, int act, void* workspace, int64_t workspace_bytes,
                         hipStream_t s) {
  PLA_REQUIRE(workspace_bytes >= l.bytes && (l.bytes == 0 || workspace), "workspace too small: %lld bytes needed", (long long)l.bytes);
  PLA_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "the workspace must be 16-byte aligned");
  for (const int64_t x : {p.q_token, p.q_head, p.k_token, p.k_head, p.v_token, p.v_head, p.kv_block, p.gate_token, p.gate_head, p.out_token, p.out_head})
    PLA_REQUIRE(x % 8 == 0, "rows must be 16-byte aligned");
  for (const void* x : {(const void*)p.q, (const void*)p.k, (const void*)p.v, (const void*)p.gate, (const void*)p.out})
    PLA_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0, "rows must be 16-byte aligned");
  PLA_REQUIRE(p.k_token >= 0 && p.k_token < (1 << 24) && p.v_token >= 0 && p.v_token < (1 << 24), "token strides of keys and values must be below 2^24");
  // The kernel takes a maximum of scores before it scales them: the sign goes to the queries, and a scale of zero becomes the smallest
  // number, which leaves finite scores equal (to 2^-20) and masked ones at minus infinity.
  p.flip = scale < 0.f ? 0x80008000u : 0u;
  p.scale_log2 = scale == 0.f ? 0x1p-149f : fabsf(scale) * 1.44269504088896341f;
  p.items = (int)l.pieces;
  p.least = l.least;
  p.slots = (int)l.items;
  p.slot_rows = l.slot_rows;
  if (l.split || l.plan) {
    char* ws = static_cast<char*>(workspace);
    p.partial = reinterpret_cast<float*>(ws);
    p.tops = reinterpret_cast<float2*>(ws + l.tops_at);
    p.plan = l.plan ? reinterpret_cast<PromptItem*>(ws + l.plan_at) : nullptr;
    p.rows = reinterpret_cast<float*>(ws + l.rows_at);
    p.row_tops = reinterpret_cast<float2*>(ws + l.row_tops_at);
  }
  if (paged) launch_prompt<true>(p, l, D, act, s);
  else launch_prompt<false>(p, l, D, act, s);
  return check_launch("prompt_attention_kernel");
}

}  // namespace pla

extern "C" int64_t pla_prompt_attention_workspace_bytes(int batch, int64_t tokens, int HQ, int HKV, int head_dim, int64_t keys) {
  using namespace pla;
  if (check_prompt(batch, tokens, HQ, HKV, head_dim) || keys < 0) return -1;
  if (batch == 0 || tokens == 0) return 0;
  return prompt_launch(batch, tokens, HQ, HKV, head_dim, keys, false).bytes;
}

extern "C" int pla_prompt_attention_launch(
    const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
    const void* offsets, int offsets_wide, const void* key_offsets, int key_offsets_wide, const void* gate, int64_t gate_token, int64_t gate_head,
    void* out, int64_t out_token, int64_t out_head, float scale, int batch, int tokens, int64_t keys, int HQ, int HKV, int head_dim, int act_dtype,
    void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace pla;
  if (const int bad = check_prompt(batch, tokens, HQ, HKV, head_dim)) return bad;
  PLA_REQUIRE(act_dtype == PLA_BF16 || act_dtype == PLA_F16, "activations must be bf16 or fp16");
  PLA_REQUIRE(keys >= 0 && keys <= INT32_MAX - 1024, "too many keys");
  if (batch == 0 || tokens == 0) return 0;
  PLA_REQUIRE(q && offsets && out && (keys == 0 || (k && v)), "null tensor pointer");
  PromptAttention p{};
  p.q = (const uint16_t*)q; p.q_token = q_token; p.q_head = q_head;
  p.k = (const uint16_t*)k; p.k_token = k_token; p.k_head = k_head;
  p.v = (const uint16_t*)v; p.v_token = v_token; p.v_head = v_head;
  p.offsets = offsets; p.offsets_wide = offsets_wide;
  p.key_offsets = key_offsets ? key_offsets : offsets; p.key_offsets_wide = key_offsets ? key_offsets_wide : offsets_wide;
  p.gate = (const uint16_t*)gate; p.gate_token = gate_token; p.gate_head = gate_head;
  p.out = (uint16_t*)out; p.out_token = out_token; p.out_head = out_head;
  p.batch = batch; p.tokens = tokens; p.heads = HKV; p.group = HQ / HKV; p.by_group = paged_divisor(HQ / HKV);
  p.positions = keys;
  return launch_prompt(p, prompt_launch(batch, tokens, HQ, HKV, head_dim, keys, false), false, head_dim, scale, act_dtype, workspace, workspace_bytes,
                       static_cast<hipStream_t>(stream));
}

extern "C" int pla_paged_prompt_attention_launch(
    const void* q, int64_t q_token, int64_t q_head, const void* k_cache, const void* v_cache, int64_t kv_block, int64_t kv_token, int64_t kv_head,
    int blocks, int block_size, const int32_t* block_table, int64_t table_row_stride, int table_rows, int table_cols,
    const void* mapping, int mapping_wide, const void* offsets, int offsets_wide, const void* seq_lens, int seq_lens_wide,
    const void* gate, int64_t gate_token, int64_t gate_head, void* out, int64_t out_token, int64_t out_head,
    float scale, int batch, int tokens, int HQ, int HKV, int head_dim, int act_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace pla;
  if (const int bad = check_prompt(batch, tokens, HQ, HKV, head_dim)) return bad;
  PLA_REQUIRE(act_dtype == PLA_BF16 || act_dtype == PLA_F16, "activations must be bf16 or fp16");
  PLA_REQUIRE(block_size > 0 && block_size % 16 == 0, "block_size must be a multiple of 16");
  const int64_t positions = (int64_t)table_cols * block_size;
  PLA_REQUIRE(positions <= (1 << 30), "a row of the block table must hold at most 2^30 positions");
  PLA_REQUIRE(table_rows >= 0 && table_cols >= 0 && table_row_stride >= table_cols, "invalid dimensions");
  if (batch == 0 || tokens == 0) return 0;
  PLA_REQUIRE(mapping || batch <= table_rows, "more requests than rows of the block table");
  PLA_REQUIRE(q && k_cache && v_cache && seq_lens && offsets && out, "null tensor pointer");
  PLA_REQUIRE(block_table || table_rows == 0 || table_cols == 0, "null tensor pointer");
  PLA_REQUIRE(blocks > 0, "the cache must hold a block");
  PromptAttention p{};
  p.q = (const uint16_t*)q; p.q_token = q_token; p.q_head = q_head;
  p.k = (const uint16_t*)k_cache; p.k_token = kv_token; p.k_head = kv_head;
  p.v = (const uint16_t*)v_cache; p.v_token = kv_token; p.v_head = kv_head;
  p.kv_block = kv_block; p.blocks = blocks; p.block_size = block_size; p.page_of = paged_divisor(block_size);
  p.table = block_table; p.table_row = table_row_stride; p.table_rows = table_cols == 0 ? 0 : table_rows;
  p.mapping = mapping; p.mapping_wide = mapping_wide;
  p.offsets = offsets; p.offsets_wide = offsets_wide;
  p.lengths = seq_lens; p.lengths_wide = seq_lens_wide;
  p.gate = (const uint16_t*)gate; p.gate_token = gate_token; p.gate_head = gate_head;
  p.out = (uint16_t*)out; p.out_token = out_token; p.out_head = out_head;
  p.batch = batch; p.tokens = tokens; p.heads = HKV; p.group = HQ / HKV; p.by_group = paged_divisor(HQ / HKV);
  p.positions = positions;
  return launch_prompt(p, prompt_launch(batch, tokens, HQ, HKV, head_dim, positions, false), true, head_dim, scale, act_dtype, workspace, workspace_bytes,
                       static_cast<hipStream_t>(stream));
}
