// Causal attention of prompts over their own keys, or over a paged cache that holds earlier ones too:
//
//   o = sum_p softmax_p(scale q.k_p) v_p  [* sigmoid(gate)]      over the keys p < keys - window + j + 1
//
// for token j of a window of `window` tokens at the end of `keys` keys.  The query heads of a key-value head and the tokens of the
// window are the rows of one product, so keys and values are read once for all of them.

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

// A row block of a sequence, as a workgroup takes it.
struct PromptBlock {
  int n, row0, rows;                      // sequence; first row of the block, rows of the block that are there
  int window, keys;                       // tokens and keys of the sequence
  int64_t begin, key_begin;               // first token row, first key (dense)
};

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

// Row block `index` of the call.  Blocks of a sequence stand last one first: it has the most keys, and the shortest end the call.
template <int ROWS, bool PAGED>
__device__ __forceinline__ bool prompt_block(const PromptAttention& p, int index, PromptBlock& b) {
  const int lane = threadIdx.x & 63;
  if (PAGED && !p.offsets) {              // all token rows over one prefix
    const int64_t length = prompt_index(p.lengths, p.lengths_wide, 0);
    b = PromptBlock{0, index * ROWS, 0, p.tokens, (int)(length < 0 ? 0 : length < p.positions ? length : p.positions), 0, 0};
    b.rows = min(ROWS, b.window * p.group - b.row0);
    return b.rows > 0;
  }
  for (int base = 0; base < p.batch; base += 64) {
    int64_t begin = 0, key_begin = 0;
    int window = 0, keys = 0;
    if (base + lane < p.batch) prompt_sequence<PAGED>(p, base + lane, begin, window, key_begin, keys);
    const int mine = (int)(((int64_t)window * p.group + ROWS - 1) / ROWS);
    int64_t below = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t x = __shfl_up(below, d);
      if (lane >= d) below += x;
    }
    const int64_t all = lane_value(below, 63);
    if (index >= all) {
      index -= (int)all;
      continue;
    }
    const int at = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(below > index)) - 1);
    const int left = (int)lane_value(below, at) - 1 - index;
    b.n = base + at;
    b.window = __builtin_amdgcn_readlane(window, at);
    b.keys = __builtin_amdgcn_readlane(keys, at);
    b.begin = lane_value(begin, at);
    b.key_begin = lane_value(key_begin, at);
    b.row0 = left * ROWS;
    b.rows = min(ROWS, b.window * p.group - b.row0);
    return true;
  }
  return false;
}

// Keys that row `row` of a sequence sees (they are the first ones).  Keys without a page count as ones that nobody sees.
__device__ __forceinline__ int prompt_limit(const PromptAttention& p, const PromptBlock& b, int row) {
  const int64_t limit = p.offsets ? (int64_t)b.keys - b.window + paged_quotient(p.by_group, row) + 1 : b.keys;
  const int64_t most = b.keys < p.positions ? b.keys : p.positions;
  return (int)(limit < 0 ? 0 : limit < most ? limit : most);
}

template <typename act_t> constexpr float PROMPT_SHIFT = 0.f;
template <> constexpr float PROMPT_SHIFT<f16_t> = 7.f;
constexpr float PROMPT_SLACK = 8.f;

// The factor from maximum `m` to maximum `top` >= m; equal infinities are no step.  Never zero: an infinite output stays one.
__device__ __forceinline__ float step_factor(float m, float top) { return m == top ? 1.f : fmaxf(__builtin_amdgcn_exp2f(m - top), 0x1p-126f); }

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

template <typename act_t, int D, int QT, bool PAGED>
__global__ __launch_bounds__(256, QT * D <= 128 ? 2 : 1) void prompt_attention_kernel(const PromptAttention p) {
  constexpr int ROWS = 128 * QT, STEPS = D / 16, TILES = D / 32, PITCH = 2 * D, TILE = PROMPT_KEYS * PITCH;
  constexpr int LANES = PITCH / 16, ROWS_A_COPY = 64 / LANES, COPIES = 16 / ROWS_A_COPY;           // of the 16 keys that a wavefront copies
  __shared__ __align__(1024) unsigned char tiles[2][2][TILE];
  __shared__ uint32_t there[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int pieces = p.heads * p.splits, index = blockIdx.x / pieces, rest = blockIdx.x - index * pieces, head = rest / p.splits, split = rest - head * p.splits;
  PromptBlock b;
  if (!prompt_block<ROWS, PAGED>(p, index, b)) return;
  const int end = prompt_limit(p, b, b.row0 + b.rows - 1);
  const PromptShare share = prompt_share(end, p.splits);
  const int first_tile = split * share.tiles, last_tile = min(first_tile + share.tiles, (end + PROMPT_KEYS - 1) / PROMPT_KEYS);
  if (split >= share.pieces) return;

  // This wavefront's rows; those past the end repeat the last one.
  int row[QT], limit[QT];
  bf16x8_t q[QT][STEPS];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    row[t] = b.row0 + min(32 * (QT * wave + t) + col, b.rows - 1);
    limit[t] = prompt_limit(p, b, row[t]);
    const int j = paged_quotient(p.by_group, row[t]), g = row[t] - j * p.group;
    const uint16_t* src = p.q + (b.begin + j) * p.q_token + (int64_t)(head * p.group + g) * p.q_head + 8 * half;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      u32x4_t x = *reinterpret_cast<const u32x4_t*>(src + 16 * s);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] ^= p.flip;
      q[t][s] = __builtin_bit_cast(bf16x8_t, x);
    }
  }
  const int least = __builtin_amdgcn_readfirstlane(prompt_limit(p, b, b.row0 + min(32 * QT * wave, b.rows - 1)));
  const int most = __builtin_amdgcn_readfirstlane(prompt_limit(p, b, b.row0 + min(32 * QT * (wave + 1), b.rows) - 1));
  const bool mine = 32 * QT * wave < b.rows;      // the wavefront has rows at all

  // Copies: wavefront w has keys 16 w .. + 15 of a tile.
  const int copy_row = lane / LANES, granule = lane % LANES;
  auto copy_swizzle_k = [&](int r) { return D == 64 ? r >> 1 & 7 : r & 15; };
  auto copy_swizzle_v = [&](int r) { return D == 64 ? 2 * (r >> 1 & 3) : 2 * (r & 7); };
  uint32_t k_off[COPIES], v_off[COPIES];
#pragma unroll
  for (int c = 0; c < COPIES; ++c) {
    const int r = ROWS_A_COPY * c + copy_row;
    k_off[c] = (uint32_t)(r * p.k_token * 2) + 16 * (granule ^ copy_swizzle_k(r));
    v_off[c] = (uint32_t)(r * p.v_token * 2) + 16 * (granule ^ copy_swizzle_v(r));
  }
  const uint32_t lds = lds_address(&tiles[0][0][0]);
  int64_t table_row = 0;
  bool has_row = true;
  const int32_t* pages = nullptr;
  if constexpr (PAGED) {
    table_row = p.mapping ? prompt_index(p.mapping, p.mapping_wide, b.n) : b.n;
    has_row = table_row >= 0 && table_row < p.table_rows;
    pages = uniform_pointer(p.table + (has_row ? table_row : 0) * p.table_row);
  }
  const int sequence_keys = min((int64_t)b.keys, p.positions);
  auto group_of = [&](int tile) { return min(tile * PROMPT_KEYS + 16 * wave, max(sequence_keys - 1, 0) & ~15); };
  auto page_entry = [&](int tile) {
    if (!PAGED || !has_row || sequence_keys == 0) return -1;
    return *(const __attribute__((address_space(4))) int32_t*)(pages + paged_quotient(p.page_of, group_of(tile)));
  };
  auto copy_tile = [&](int tile, int buffer, int entry) {
    const int key0 = group_of(tile);
    int last = sequence_keys - 1 - key0;          // of the 16 keys; those behind repeat it
    const uint16_t *k, *v;
    if constexpr (PAGED) {
      const bool ok = entry >= 0 && entry < p.blocks;
      const int place = key0 - paged_quotient(p.page_of, key0) * p.block_size;
      const int64_t at = ok ? entry * p.kv_block + place * p.k_token : 0;
      k = p.k + at + head * p.k_head;
      v = p.v + at + head * p.v_head;
      if (!ok) last = 15;
      if (lane == 0) reinterpret_cast<unsigned char*>(&there[buffer])[wave] = ok;
    } else {
      k = p.k + (b.key_begin + key0) * p.k_token + head * p.k_head;
      v = p.v + (b.key_begin + key0) * p.v_token + head * p.v_head;
    }
    const uint32_t to = lds + buffer * 2 * TILE + wave * 16 * PITCH;
    const char *kb = uniform_pointer(reinterpret_cast<const char*>(k)), *vb = uniform_pointer(reinterpret_cast<const char*>(v));
    if (last >= 15) {
#pragma unroll
      for (int c = 0; c < COPIES; ++c) dma16(kb, k_off[c], to + 1024 * c);
#pragma unroll
      for (int c = 0; c < COPIES; ++c) dma16(vb, v_off[c], to + TILE + 1024 * c);
    } else {
#pragma unroll
      for (int c = 0; c < COPIES; ++c) {
        const int r = ROWS_A_COPY * c + copy_row, back = max(r - last, 0);
        dma16(kb, k_off[c] - (uint32_t)(back * p.k_token * 2), to + 1024 * c);
        dma16(vb, v_off[c] - (uint32_t)(back * p.v_token * 2), to + TILE + 1024 * c);
      }
    }
  };
  // Operands: K rows are keys, lane (col, half) reads granule 2 s + half of key 32 t + col; values four keys and sixteen channels a
  // group of 16 lanes.
  const uint32_t k_at = lds + col * PITCH + 16 * (half ^ copy_swizzle_k(col));
  const int v_row = 4 * half + ((lane & 15) >> 2);
  const uint32_t v_at = lds + TILE + v_row * PITCH + 16 * ((2 * (lane >> 4 & 1) + ((lane & 3) >> 1)) ^ copy_swizzle_v(v_row)) + 8 * (lane & 1);

  f32x16_t o[QT][TILES];
  float top[QT], sum[QT];

  auto pass = [&](auto careful) {
    constexpr bool CAREFUL = decltype(careful)::value;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      top[t] = -INFINITY;
      sum[t] = 0.f;
#pragma unroll
      for (int c = 0; c < TILES; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][c][i] = 0.f;
    }
    int entry = page_entry(first_tile);
    if (first_tile < last_tile) copy_tile(first_tile, 0, entry);
    entry = page_entry(first_tile + 1);
    for (int tile = first_tile; tile < last_tile; ++tile) {
      const int buffer = (tile - first_tile) & 1, key0 = tile * PROMPT_KEYS;
      wait_vmcnt<0>();
      lds_barrier();
      if (tile + 1 < last_tile) {
        copy_tile(tile + 1, buffer ^ 1, entry);
        entry = page_entry(tile + 2);
      }
      if (!mine || key0 >= most) continue;
      uint32_t flags = 0x01010101u;
      if constexpr (PAGED) flags = __builtin_amdgcn_readfirstlane(there[buffer]);
      const uint32_t kb = k_at + buffer * 2 * TILE, vb = v_at + buffer * 2 * TILE;
      f32x16_t s[QT][2];
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[t][h][i] = 0.f;
#pragma unroll
      for (int c = 0; c < STEPS; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bf16x8_t k = lds_operand((kb ^ (32u * c)) + h * 32 * PITCH);
#pragma unroll
          for (int t = 0; t < QT; ++t) s[t][h] = mfma32<act_t>(k, q[t][c], s[t][h]);
        }
      const bool masked = key0 + PROMPT_KEYS > least || flags != 0x01010101u;
      auto sees = [&](int t, int h, int i) {
        const int key = 32 * h + 8 * (i / 4) + 4 * half + (i & 3);
        return (key0 + key < limit[t]) & ((flags >> (8 * (2 * h + i / 8)) & 1) != 0);
      };
      bf16x8_t weight[QT][4];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        if (masked) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][h][i] = sees(t, h, i) ? s[t][h][i] : -INFINITY;
        }
        float high = fmaxf(s[t][0][0], s[t][1][0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) high = fmaxf(fmaxf(s[t][0][i], s[t][1][i]), high);
        high = halves_max(high) * p.scale_log2;
        if (__ballot(high > top[t] + PROMPT_SLACK) != 0) {
          const float now = fmaxf(top[t], high), f = step_factor(top[t], now);
          top[t] = now;
          sum[t] *= f;
#pragma unroll
          for (int c = 0; c < TILES; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][c][i] *= f;
        }
        const float zero = (top[t] == -INFINITY ? 0.f : top[t]) - PROMPT_SHIFT<act_t>;
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            s[t][h][i] = __builtin_amdgcn_exp2f(fmaf(s[t][h][i], p.scale_log2, -zero));
            part[h] += s[t][h][i];
          }
        sum[t] += part[0] + part[1];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          u32x4_t w;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = pack2<act_t>(s[t][x / 2][8 * (x & 1) + 2 * i], s[t][x / 2][8 * (x & 1) + 2 * i + 1]);
          weight[t][x] = __builtin_bit_cast(bf16x8_t, w);
        }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
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
#pragma unroll
              for (int t = 0; t < QT; ++t) {
                u32x4_t marks;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  marks[i] = one & ((sees(t, x / 2, 8 * (x & 1) + 2 * i) ? 0xffffu : 0u) | (sees(t, x / 2, 8 * (x & 1) + 2 * i + 1) ? 0xffff0000u : 0u));
                f32x16_t up, down;
#pragma unroll
                for (int i = 0; i < 16; ++i) up[i] = down[i] = 0.f;
                up = mfma32<act_t>(__builtin_bit_cast(bf16x8_t, plus), __builtin_bit_cast(bf16x8_t, marks), up);
                down = mfma32<act_t>(__builtin_bit_cast(bf16x8_t, minus), __builtin_bit_cast(bf16x8_t, marks), down);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][c][i] += (up[i] > 0.f ? INFINITY : 0.f) + (down[i] > 0.f ? -INFINITY : 0.f);
              }
            }
          }
#pragma unroll
          for (int t = 0; t < QT; ++t) o[t][c] = mfma32<act_t>(v, weight[t][x], o[t][c]);
        }
    }
  };
  pass(std::false_type{});
  // A NaN may be one of the formula's, or an infinite or NaN value whose weight is zero: once more, with such values apart.
  float check = 0.f;
#pragma unroll
  for (int t = 0; t < QT; ++t)
#pragma unroll
    for (int c = 0; c < TILES; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) check += o[t][c][i] * 0.f;
  if (__syncthreads_or(check != check)) pass(std::true_type{});
  if (!mine) return;

#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const bool real = 32 * (QT * wave + t) + col < b.rows;
    const int j = paged_quotient(p.by_group, row[t]), g = row[t] - j * p.group;
    const int64_t token = b.begin + j;
    const int query_head = head * p.group + g;
    const float total = halves_sum(sum[t]);
    if (p.tops && (share.pieces > 1 || !p.offsets)) {
      const int64_t at = ((int64_t)split * p.tokens + token) * (p.heads * p.group) + query_head;
      if (real) {
#pragma unroll
        for (int c = 0; c < TILES; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(p.partial + at * D + 32 * c + 8 * i + 4 * half) =
                float4{o[t][c][4 * i], o[t][c][4 * i + 1], o[t][c][4 * i + 2], o[t][c][4 * i + 3]};
        if (half == 0) p.tops[at] = float2{top[t] - PROMPT_SHIFT<act_t>, total};
      }
      continue;
    }
    const float norm = total == 0.f ? 0.f : 1.0f / total;         // no key: zeros
#pragma unroll
    for (int c = 0; c < TILES; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        // lane half 0 gets channels 16 x .. + 7 of the 32, half 1 the next eight
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float low = o[t][c][8 * x + i], high = o[t][c][8 * x + 4 + i];
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

// Pieces of a row block to its output: a wavefront a row at a time, a lane D / 64 channels.
template <typename act_t, int D, int ROWS, bool PAGED>
__global__ __launch_bounds__(256) void prompt_join_kernel(const PromptAttention p) {
  constexpr int LANE = D / 64;
  typedef float lane_t __attribute__((ext_vector_type(LANE)));
  const int index = blockIdx.x / p.heads, head = blockIdx.x - index * p.heads;
  PromptBlock b;
  if (!prompt_block<ROWS, PAGED>(p, index, b)) return;
  const PromptShare share = prompt_share(prompt_limit(p, b, b.row0 + b.rows - 1), p.splits);
  if (share.pieces < 2) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int r = blockIdx.y * 4 + wave; r < b.rows; r += 4 * gridDim.y) {
    const int j = paged_quotient(p.by_group, b.row0 + r), query_head = head * p.group + b.row0 + r - j * p.group;
    const int64_t token = b.begin + j;
    float top = -INFINITY, sum = 0.f;
    lane_t o = {};
    for (int s = 0; s < share.pieces; ++s) {
      const int64_t at = ((int64_t)s * p.tokens + token) * (p.heads * p.group) + query_head;
      const float2 y = p.tops[at];
      const lane_t x = *reinterpret_cast<const lane_t*>(p.partial + at * D + LANE * lane);
      const float now = fmaxf(top, y.x), back = step_factor(top, now), f = step_factor(y.x, now);
      sum = fmaf(y.y, f, sum * back);
#pragma unroll
      for (int c = 0; c < LANE; ++c) o[c] = fmaf(x[c], f, o[c] * back);
      top = now;
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
  const dim3 grid((unsigned)(l.blocks * p.heads * l.splits));
  if constexpr (D != 256) {
    if (l.rows == 256) prompt_attention_kernel<act_t, D, 2, PAGED><<<grid, 256, 0, s>>>(p);
  }
  if (l.rows == 128) prompt_attention_kernel<act_t, D, 1, PAGED><<<grid, 256, 0, s>>>(p);
  if (l.splits > 1 && p.offsets) {
    const dim3 join((unsigned)(l.blocks * p.heads), (unsigned)(l.rows / 16));
    if (l.rows == 256) prompt_join_kernel<act_t, D, 256, PAGED><<<join, 256, 0, s>>>(p);
    else prompt_join_kernel<act_t, D, 128, PAGED><<<join, 256, 0, s>>>(p);
  }
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

PromptLaunch prompt_launch(int batch, int64_t tokens, int HQ, int HKV, int D, int64_t keys) {
  PromptLaunch l{};
  const int64_t rows = tokens * (HQ / HKV);
  l.rows = D != 256 && (rows / 256 + batch) * HKV >= 256 ? 256 : 128;
  // a sequence has a block that is not full, and there are no more blocks than rows
  l.blocks = rows / l.rows + batch;
  if (l.blocks > rows) l.blocks = rows;
  const int64_t groups = l.blocks * HKV, most = (keys + 4 * PROMPT_KEYS - 1) / (4 * PROMPT_KEYS);
  l.splits = (int)(groups >= 256 ? 1 : (511 / groups < most ? 511 / groups : most));
  if (l.splits < 1) l.splits = 1;
  return l;
}

int check_prompt(int batch, int64_t tokens, int HQ, int HKV, int D) {
  PLA_REQUIRE(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256, got %d", D);
  PLA_REQUIRE(HKV > 0 && HQ >= HKV && HQ % HKV == 0, "query heads must be a positive multiple of key-value heads");
  PLA_REQUIRE(batch >= 0 && tokens >= 0 && tokens * HQ <= (1 << 30), "too many rows");
  PLA_REQUIRE((tokens * (HQ / HKV) / 128 + batch) * HKV < (1 << 24), "too many sequences");
  return 0;
}

int64_t prompt_tops_at(const PromptLaunch& l, int64_t tokens, int HQ, int D) { return l.splits * tokens * HQ * D * 4; }
int64_t prompt_bytes(const PromptLaunch& l, int64_t tokens, int HQ, int D, bool always) {
  return l.splits > 1 || always ? (prompt_tops_at(l, tokens, HQ, D) + l.splits * tokens * HQ * 8 + 255) / 256 * 256 : 0;
}

int launch_prompt(PromptAttention p, const PromptLaunch& l, bool paged, int HQ, int D, float scale, int act, void* workspace, int64_t workspace_bytes,
                         hipStream_t s) {
  const int64_t bytes = prompt_bytes(l, p.tokens, HQ, D, !p.offsets);
  PLA_REQUIRE(workspace_bytes >= bytes && (bytes == 0 || workspace), "workspace too small: %lld bytes needed", (long long)bytes);
  PLA_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "the workspace must be 16-byte aligned");
  for (const int64_t x : {p.q_token, p.q_head, p.k_token, p.k_head, p.v_token, p.v_head, p.kv_block, p.gate_token, p.gate_head, p.out_token, p.out_head})
    PLA_REQUIRE(x % 8 == 0, "rows must be 16-byte aligned");
  for (const void* x : {(const void*)p.q, (const void*)p.k, (const void*)p.v, (const void*)p.gate, (const void*)p.out})
    PLA_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0, "rows must be 16-byte aligned");
  PLA_REQUIRE(p.k_token >= 0 && p.k_token < (1 << 24) && p.v_token >= 0 && p.v_token < (1 << 24), "token strides of keys and values must be below 2^24");
  // The kernel takes a maximum of scores before it scales them: the sign goes to the queries, and a scale of zero becomes one that
  // leaves finite scores equal.
  p.flip = scale < 0.f ? 0x80008000u : 0u;
  p.scale_log2 = scale == 0.f ? 1e-38f : fabsf(scale) * 1.44269504088896341f;
  p.splits = l.splits;
  char* ws = static_cast<char*>(workspace);
  p.partial = bytes ? reinterpret_cast<float*>(ws) : nullptr;
  p.tops = bytes ? reinterpret_cast<float2*>(ws + prompt_tops_at(l, p.tokens, HQ, D)) : nullptr;
  if (paged) launch_prompt<true>(p, l, D, act, s);
  else launch_prompt<false>(p, l, D, act, s);
  return check_launch("prompt_attention_kernel");
}

}  // namespace pla

extern "C" int64_t pla_prompt_attention_workspace_bytes(int batch, int64_t tokens, int HQ, int HKV, int head_dim, int64_t keys) {
  using namespace pla;
  if (check_prompt(batch, tokens, HQ, HKV, head_dim) || keys < 0) return -1;
  if (batch == 0 || tokens == 0) return 0;
  return prompt_bytes(prompt_launch(batch, tokens, HQ, HKV, head_dim, keys), tokens, HQ, head_dim, false);
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
  return launch_prompt(p, prompt_launch(batch, tokens, HQ, HKV, head_dim, keys), false, HQ, head_dim, scale, act_dtype, workspace, workspace_bytes,
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
  return launch_prompt(p, prompt_launch(batch, tokens, HQ, HKV, head_dim, positions), true, HQ, head_dim, scale, act_dtype, workspace, workspace_bytes,
                       static_cast<hipStream_t>(stream));
}
