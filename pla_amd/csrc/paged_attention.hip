// Attention of one new token, or of a window of draft tokens, over a paged key-value cache:
//
//   o = sum_p softmax_p(scale q.k_p) v_p  [* sigmoid(gate)]      over the keys p that the token sees: p < length - window + j + 1
//
// for token j of a request's window.  The query heads of a key-value head and the tokens of the window are the rows of one
// product, in blocks of 16, 32 or (D 64 and 128) 64 rows; keys and values are read once for a block.  16 windows of eight over 8000
// keys, 64 rows a head of 128, take 88.5 us as blocks of 32 and 79.8 as one of 64, windows of sixteen (two blocks) 129; 64 rows of 256
// channels do not fit the registers.
//
// Each wavefront takes 32 keys at a time: keys and values go from memory to the registers in which the matrix instructions want them,
// through no LDS.  The wavefronts of a workgroup work together, one 32 keys after the other's, and put their rows together at the
// end of a run.  Or (ALONE; 16 rows, many runs) each has runs of its own, with the queries in registers, and writes what it has whole
// from registers: nothing waits for another wavefront before the end of the kernel, where what they share is put together.  256
// requests of 300 to 4000 keys (D 128, 8 heads) take 251 us together and 245 alone, 1000 of 50 keys 82.6 and 67.3 (D 64: 74.7
// and 40.1), 64 of 200 to 4000 (D 256, 2 heads) 43.2 and 38.8.  Few runs, which wavefronts would have to share all the same, lose
// by it (one request of 60 000 keys, D 64, 2 heads, 20.1 and 22.0), so they stay together.
//
//   S^T = K Q^T    keys are the rows: lane (r, kb) loads 16 bytes of key r a step, any channels, as Q holds the same ones.
//                  It gets the scores of query r at keys 4 kb .. 4 kb + 3 of both halves of the 32 keys,
//   O^T = V^T P^T  which is the operand that the second product wants, if its contraction runs over the keys in that order:
//                  lane (r, kb) loads channels 8 r .. 8 r + 7 of those eight keys, eight loads of which sixteen lanes cover a
//                  row, and one v_perm_b32 a pair of values turns them into rows of V^T.  No value crosses a lane.
//
// A row's maximum and sum run along, in FP32.  For the product a weight goes in two parts of the cache's type, what remains of it
// in the second: off by up to 2^-16 of itself (fp16 2^-22; weights are scaled by 2^14 there), and by up to two least parts, 2^-37 of
// the largest weight in fp16.  One part alone would be off by 2^-8, as much as the output's own rounding where values cancel.
//
// Values that no row of a block sees are replaced by zeros: their weight is zero, but zero times what an unused place of the
// cache may hold need not be.  Within a window some rows see values that others do not.  Where one of those is infinite or NaN,
// these values (at most 31, of two steps) are set aside and added row by row at the end of the run, to the rows that see them.
//
// Bound by HBM: 4 D bytes a key and head are needed once, for 4 D flops a row and 2 D for the weights' second part.  32 rows at
// 6 TB/s are 290 TFLOP/s of products, a quarter of what a large product reaches here; blocks of 64 rows, of which a SIMD has one
// wavefront, wait for the products and the exponentials too.
//
// Caches of 8-bit numbers (e4m3) with a scale a token and head are widened to the queries' type on the way to the matrix instructions,
// which is exact; a key's scale multiplies its scores, a value's scale its weights, which then go in two parts of bf16 with either type of
// queries, as a scale may be anything FP32 holds.  2 D + 8 bytes a key and head: 256 requests of 300 to 4000 keys (D 128, 8 heads) 143 us
// (5.4 TB/s) against 245 over 16 bits; 40 windows of four over 500 to 30 000 keys (D 256, 2 heads, 32 rows) 77 against 87: of the one
// wavefront's cycles on a SIMD 40 % issue vector instructions there and 30 % wait for keys, LDS or a barrier, with nothing to cover them.
//
// A prefix that all requests share is attended to first, for all token rows together (the kernel over prompts, which reads it once), and what
// it gives for a row, (maximum, sum, outputs) in FP32, is put in where a run's rows or pieces are put together: 64 requests of 40 to 1500
// keys after a prefix of 8000 (D 128, 8 heads) 56 us, 27 of them for the prefix and 28 for the own keys.  It is compiled in apart (PREFIX):
// as a branch it cost calls without a prefix 1.4 us of 30.

#include "decode_common.h"
#include "mfma_bf16.h"
#include "paged_schedule.h"
#include "prompt_attention.h"

namespace pla {

// A run in pieces, for the kernel that joins them.
struct PagedRun {
  int pieces;                                     // below 2: it is whole, or there is no such run
  int worker;                                     // of the first piece
  int begin, head, row0, rows;                    // first token row of the request, key-value head, rows of the run
  int unused[2];
};

struct PagedAttention {
  const uint16_t* q; int64_t q_token, q_head;
  const void *k, *v; int64_t kv_block, kv_token, kv_head;         // 16 bits a number, or 8
  const int32_t* table; int64_t table_row;
  const void* mapping; int mapping_wide;
  const void* offsets; int offsets_wide;          // NULL: token row n is request n
  const void* lengths; int lengths_wide;
  const uint16_t* gate; int64_t gate_token, gate_head;
  uint16_t* out; int64_t out_token, out_head;
  PagedShape shape;
  int batch, blocks, block_size, table_rows;
  PagedDivisor page_of;                           // position to page
  float scale_log2;
  int by_run, row_blocks;                         // runs in pieces are listed by run, or by worker; row blocks of the longest window
  float* partial; float2* tops; PagedRun* runs;
  const float *k_scales, *v_scales; int64_t scale_block, scale_head;     // of numbers of 8 bits: [block][head][place]
  // attention over a prefix that all rows share: outputs and their references and sums [token][query head]
  const float* prefix; const float2* prefix_tops;

  __device__ int64_t at(const void* base, int wide, int64_t i) const {
    return wide ? static_cast<const int64_t*>(base)[i] : (int64_t) static_cast<const int32_t*>(base)[i];
  }
  __device__ PagedRequest request(int n) const {
    const int64_t begin = offsets ? at(offsets, offsets_wide, n) : n, end = offsets ? at(offsets, offsets_wide, n + 1) : n + 1;
    return paged_request(shape, begin, end, at(lengths, lengths_wide, n));
  }
};

// Index vectors and block tables through the scalar cache, where the index is the same for a wavefront: nothing writes them while
// the kernel runs, and a vector load would be waited for behind all keys and values in flight.
__device__ __forceinline__ int32_t scalar_load(const int32_t* p) { return *(const __attribute__((address_space(4))) int32_t*)p; }
__device__ __forceinline__ int64_t scalar_at(const void* base, int wide, int n) {
  const int32_t* p = static_cast<const int32_t*>(base) + (wide ? 2 * (int64_t)n : n);
  return wide ? (int64_t)((uint64_t)(uint32_t)scalar_load(p) | (uint64_t)(uint32_t)scalar_load(p + 1) << 32) : (int64_t)scalar_load(p);
}
__device__ __forceinline__ PagedRequest scalar_request(const PagedAttention& p, int n) {
  const int64_t begin = p.offsets ? scalar_at(p.offsets, p.offsets_wide, n) : n;
  const int64_t end = p.offsets ? scalar_at(p.offsets, p.offsets_wide, n + 1) : n + 1;
  return paged_request(p.shape, begin, end, scalar_at(p.lengths, p.lengths_wide, n));
}

template <typename act_t> __device__ __forceinline__ f32x4_t mfma_act(bf16x8_t a, bf16x8_t b, f32x4_t c);
template <> __device__ __forceinline__ f32x4_t mfma_act<bf16_t>(bf16x8_t a, bf16x8_t b, f32x4_t c) { return mfma16(a, b, c); }
template <> __device__ __forceinline__ f32x4_t mfma_act<f16_t>(bf16x8_t a, bf16x8_t b, f32x4_t c) { return mfma16h(a, b, c); }

template <typename act_t> constexpr float WEIGHT_SHIFT = 0.f;
template <> constexpr float WEIGHT_SHIFT<f16_t> = 14.f;

// What a cache holds: numbers of the queries' type, or e4m3 numbers of 8 bits with a factor a key and head.  The latter are widened to
// the queries' type for the scores and to bf16 for the values, both without an error; keys' factors go to the scores and values' to the
// weights, so a weight may be larger than one there, which bf16 holds.
struct e4m3_t { uint8_t bits; };
template <typename act_t, typename kv_t> struct Cached { using raw_t = uint16_t; using value_t = act_t; static constexpr bool SCALED = false; };
template <typename act_t> struct Cached<act_t, e4m3_t> { using raw_t = uint8_t; using value_t = bf16_t; static constexpr bool SCALED = true; };
// Two of the four numbers of a word, widened.
template <typename T> __device__ __forceinline__ uint32_t widen2(uint32_t word, int second);
template <> __device__ __forceinline__ uint32_t widen2<bf16_t>(uint32_t word, int second) {
  return second ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.f, false));
}
template <> __device__ __forceinline__ uint32_t widen2<f16_t>(uint32_t word, int second) {
  return second ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.f, false));
}
template <typename act_t> __device__ __forceinline__ float cached_number(const uint16_t* p) { return to_float(act_t{*p}); }
template <typename act_t> __device__ __forceinline__ float cached_number(const uint8_t* p) { return __builtin_amdgcn_cvt_f32_fp8((int)*p, 0); }

// Over the four lanes that hold a query's scores.
__device__ __forceinline__ float query_max(float x) {
  const LanePair a = swap_rows16(x);
  const float y = fmaxf(a.lo, a.hi);
  const LanePair b = swap_halves(y);
  return fmaxf(b.lo, b.hi);
}
__device__ __forceinline__ float query_sum(float x) {
  const LanePair a = swap_rows16(x);
  const float y = a.lo + a.hi;
  const LanePair b = swap_halves(y);
  return b.lo + b.hi;
}

// The factor from maximum `m` to maximum `top` >= m; equal infinities are no step.  Never zero: an infinite output stays one.
__device__ __forceinline__ float rescale(float m, float top) { return m == top ? 1.f : fmaxf(__builtin_amdgcn_exp2f(m - top), 0x1p-126f); }

// Two weights as packed pairs of a first part, cut off, and of what remains, rounded.  Neither part is negative (the cut sees to it)
// nor zero: a key that a row sees has some weight, so that an infinite value there makes the output infinite, as in the formula, by
// whichever way it comes into the sum.
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
template <typename act_t> constexpr float LEAST_PART = 0x1p-126f;
template <> constexpr float LEAST_PART<f16_t> = 0x1p-24f;
template <typename act_t>
__device__ __forceinline__ uint32_t at_least_least(uint32_t pair) {         // of numbers that are not negative: they are ordered as their bits
  const uint16_t least = __is_same(act_t, bf16_t) ? 0x0080 : 0x0001;
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, pair), u16x2_t{least, least}));
}
template <typename act_t>
__device__ __forceinline__ void weight_parts(float x, float y, uint32_t& high, uint32_t& low) {
  high = __is_same(act_t, bf16_t) ? __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302u)
                                  : pack2_rtz(x, y);
  low = at_least_least<act_t>(pack2<act_t>(x - lo16<act_t>(high), y - hi16<act_t>(high)));
  high = at_least_least<act_t>(high);
}

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
template <int D> struct ValueWords { static constexpr int N = D == 64 ? 2 : 4; };      // 32-bit words of a lane's channels, a chunk

// Keys in flight, values in flight and the state of the rows of one wavefront.
template <typename act_t, typename kv_t, int D, int RT>
struct Wave {
  using raw_t = typename Cached<act_t, kv_t>::raw_t;
  static constexpr bool SCALED = Cached<act_t, kv_t>::SCALED;
  static constexpr int STEPS = D / 32;                        // of the contraction of K Q^T
  static constexpr int WORDS = ValueWords<D>::N, CHUNKS = D == 256 ? 2 : 1, TILES = 2 * WORDS;
  static constexpr int LANE_CHANNELS = 2 * WORDS;             // channels of a value that a lane loads, a chunk of 16 times as many
  static constexpr int KEY_LOADS = SCALED ? STEPS / 2 : STEPS, RAW_WORDS = SCALED ? WORDS / 2 : WORDS;
  u32x4_t k[2][KEY_LOADS];
  uint32_t v[8][CHUNKS][RAW_WORDS];
  f32x4_t k_scale[SCALED ? 2 : 1], v_scale[SCALED ? 2 : 1];   // of the lane's keys
  f32x4_t o[RT][CHUNKS][TILES];
  float top[RT], sum[RT];
  int limit[RT];
  int set_aside;                                              // first key of the step whose partly seen values are added at the end, + 1 if those
                                                              // of the next are too (a wavefront alone may have both), or -1
  __device__ __forceinline__ bf16x8_t key(int h, int c) const {
    if constexpr (SCALED) {
      u32x4_t x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = widen2<act_t>(k[h][c / 2][2 * (c & 1) + i / 2], i & 1);
      return __builtin_bit_cast(bf16x8_t, x);
    } else {
      return __builtin_bit_cast(bf16x8_t, k[h][c]);
    }
  }
  __device__ __forceinline__ uint32_t value(int i, int c, int j) const {
    if constexpr (SCALED) return widen2<bf16_t>(v[i][c][j / 2], j & 1);
    else return v[i][c][j];
  }
};

// Keys and values from where the two halves of a step's keys lie (`place`, and `at` of their factors), in elements.
template <typename W, typename raw_t>
__device__ __forceinline__ void load_keys(W& w, const raw_t* base, const float* scales, const int64_t (&place)[2], const int64_t (&at)[2], uint32_t lane_offset) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const auto p = as_global(reinterpret_cast<const char*>(base + place[h]));
#pragma unroll
    for (int c = 0; c < W::KEY_LOADS; ++c) w.k[h][c] = *reinterpret_cast<global_ptr<const u32x4_t>>(p + lane_offset + 64 * c);
    if constexpr (W::SCALED) w.k_scale[h] = *reinterpret_cast<global_ptr<const f32x4_t>>(as_global(scales + at[h]) + 4 * ((threadIdx.x & 63) >> 4));
  }
}

template <typename W, typename raw_t>
__device__ __forceinline__ void load_values(W& w, const raw_t* base, const float* scales, const int64_t (&place)[2], const int64_t (&at)[2], uint32_t lane_offset,
                                            int64_t token_bytes) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const auto p = as_global(reinterpret_cast<const char*>(base + place[i / 4])) + (i & 3) * token_bytes;
#pragma unroll
    for (int c = 0; c < W::CHUNKS; ++c) {
      if constexpr (W::RAW_WORDS == 4) {
        const u32x4_t x = __builtin_nontemporal_load(reinterpret_cast<global_ptr<const u32x4_t>>(p + lane_offset + 256 * c));
#pragma unroll
        for (int y = 0; y < 4; ++y) w.v[i][c][y] = x[y];
      } else if constexpr (W::RAW_WORDS == 2) {
        const u32x2_t x = __builtin_nontemporal_load(reinterpret_cast<global_ptr<const u32x2_t>>(p + lane_offset + 128 * c));
        w.v[i][c][0] = x[0]; w.v[i][c][1] = x[1];
      } else {
        w.v[i][c][0] = __builtin_nontemporal_load(reinterpret_cast<global_ptr<const uint32_t>>(p + lane_offset));
      }
    }
  }
  if constexpr (W::SCALED) {
#pragma unroll
    for (int h = 0; h < 2; ++h) w.v_scale[h] = *reinterpret_cast<global_ptr<const f32x4_t>>(as_global(scales + at[h]) + 4 * ((threadIdx.x & 63) >> 4));
  }
}

// For v_perm_b32 on the words of two keys that hold channels 2 j and 2 j + 1 of one each: channel 2 j (odd: 2 j + 1) of both,
// zero where a key is left out.
__device__ __forceinline__ uint32_t selection(int odd, bool first, bool second) {
  return (first ? odd ? 0x0302u : 0x0100u : 0x0c0cu) | (second ? odd ? 0x07060000u : 0x05040000u : 0x0c0c0000u);
}
// Bit 15 or 31 is set if all bits of the exponent of that half are.
template <typename act_t>
__device__ __forceinline__ uint32_t not_finite(uint32_t pair) {
  return __is_same(act_t, bf16_t) ? (pair & 0x7f807f80u) + 0x00800080u : (pair & 0x7c007c00u) + 0x04000400u;
}

// The same of words of four numbers of 8 bits, of which the NaN is the one with all bits set but the sign; bit 7, 15, 23 or 31.
__device__ __forceinline__ uint32_t not_a_number8(uint32_t word) { return (word & 0x7f7f7f7fu) + 0x01010101u; }

// One step of a wavefront: scores of 32 keys from key0 on, their weights, and the weighted values.  `next`: issues the loads of
// the step after (keys once these are used, values once those are).
template <typename act_t, typename kv_t, int D, int RT, typename Queries, typename NextKeys, typename NextValues>
__device__ __forceinline__ void attend(Wave<act_t, kv_t, D, RT>& w, Queries queries, float scale_log2, const bool (&there)[2],
                                       int key0, int least, int end, NextKeys next_keys, NextValues next_values) {
  using W = Wave<act_t, kv_t, D, RT>;
  using value_t = typename Cached<act_t, kv_t>::value_t;
  const int kb = (threadIdx.x & 63) >> 4;
  f32x4_t s[RT][2];
#pragma unroll
  for (int t = 0; t < RT; ++t) s[t][0] = s[t][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < W::STEPS; ++c) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const bf16x8_t q = __builtin_bit_cast(bf16x8_t, queries(t, c));
#pragma unroll
      for (int h = 0; h < 2; ++h) s[t][h] = mfma_act<act_t>(w.key(h, c), q, s[t][h]);
    }
    if (D == 256) __builtin_amdgcn_sched_barrier(0);          // queries of all steps at once would not fit the registers
  }
  f32x4_t factor[2];                              // of the lane's keys, to the scores
  if constexpr (W::SCALED) {
    factor[0] = w.k_scale[0] * scale_log2;
    factor[1] = w.k_scale[1] * scale_log2;
  }
  next_keys();

  const bool masked = key0 + 32 > least || !there[0] || !there[1];          // some row does not see some key
  auto sees = [&](int t, int i) { return (key0 + 16 * (i / 4) + 4 * kb + (i & 3) < w.limit[t]) & there[i / 4]; };
  bf16x8_t high[RT], low[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = s[t][i / 4][i & 3] * (W::SCALED ? factor[i / 4][i & 3] : scale_log2);
    if (masked) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = sees(t, i) ? x[i] : -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    top = fmaxf(query_max(top), w.top[t]);
    if (__ballot(top > w.top[t]) != 0) {
      const float f = rescale(w.top[t], top);
      w.sum[t] *= f;
#pragma unroll
      for (int c = 0; c < W::CHUNKS; ++c)
#pragma unroll
        for (int j = 0; j < W::TILES; ++j) w.o[t][c][j] *= f;
      w.top[t] = top;
    }
    const float zero = (top == -INFINITY ? 0.f : top) - WEIGHT_SHIFT<value_t>;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_exp2f(x[i] - zero);
    u32x4_t a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w.sum[t] += x[2 * i] + x[2 * i + 1];
      uint32_t first, second;
      if constexpr (W::SCALED) {
        // numbers of 8 bits have no infinity that a weight of zero would hide
        const float y0 = x[2 * i] * w.v_scale[i / 2][2 * (i & 1)], y1 = x[2 * i + 1] * w.v_scale[i / 2][2 * (i & 1) + 1];
        first = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y1), __builtin_bit_cast(uint32_t, y0), 0x07060302u);
        second = pack2<bf16_t>(y0 - lo16<bf16_t>(first), y1 - hi16<bf16_t>(first));
      } else {
        weight_parts<act_t>(x[2 * i], x[2 * i + 1], first, second);
      }
      a[i] = first;
      b[i] = second;
    }
    if (masked) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t seen = (sees(t, 2 * i) ? 0xffffu : 0u) | (sees(t, 2 * i + 1) ? 0xffff0000u : 0u);
        a[i] &= seen;
        b[i] &= seen;
      }
    }
    high[t] = __builtin_bit_cast(bf16x8_t, a);
    low[t] = __builtin_bit_cast(bf16x8_t, b);
  }

  // Values of two keys are turned by one byte selection, which also puts zeros in the place of values that no row sees.
  const int key = key0 + 4 * kb;
  uint32_t select[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    select[0][i] = 0x05040100u;
    select[1][i] = 0x07060302u;
  }
  if (masked) {
    int stop = end;
    if (least < end && key0 + 32 > least) {       // some rows see values that others do not
      uint32_t odd = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = key + 16 * (i / 4) + (i & 3);
        const bool partly = (at >= least) & (at < end) & there[i / 4];
#pragma unroll
        for (int c = 0; c < W::CHUNKS; ++c)
#pragma unroll
          for (int j = 0; j < W::RAW_WORDS; ++j) odd |= !partly ? 0u : W::SCALED ? not_a_number8(w.v[i][c][j]) : not_finite<act_t>(w.v[i][c][j]);
      }
      if (__ballot((odd & (W::SCALED ? 0x80808080u : 0x80008000u)) != 0) != 0) {
        stop = least;
        w.set_aside = w.set_aside < 0 ? key0 : w.set_aside | 1;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = key + 16 * (i / 2) + 2 * (i & 1);
      const bool first = (at < stop) & there[i / 2], second = (at + 1 < stop) & there[i / 2];
#pragma unroll
      for (int x = 0; x < 2; ++x) select[x][i] = selection(x, first, second);
    }
  }
#pragma unroll
  for (int c = 0; c < W::CHUNKS; ++c)
#pragma unroll
    for (int j = 0; j < W::TILES; ++j) {
      u32x4_t a;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = __builtin_amdgcn_perm(w.value(2 * i + 1, c, j / 2), w.value(2 * i, c, j / 2), select[j & 1][i]);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        w.o[t][c][j] = mfma_act<value_t>(__builtin_bit_cast(bf16x8_t, a), high[t], w.o[t][c][j]);
        w.o[t][c][j] = mfma_act<value_t>(__builtin_bit_cast(bf16x8_t, a), low[t], w.o[t][c][j]);
      }
    }
  next_values();
}

// The weighted values of keys [first, last) into the D / TEAM channels of a row that a thread has (the sum has the weights already);
// the TEAM threads of a row form its scores together.
template <typename act_t, typename kv_t, int D, int TEAM>
__device__ __forceinline__ void add_set_aside(const PagedAttention& p, const PagedRequest& req, int kv_head, int row, int channel,
                                              const int32_t* pages, int first, int last, float top, float (&o)[D / TEAM]) {
  const int j = paged_quotient(p.shape.by_group, row), head = kv_head * p.shape.group + row - j * p.shape.group;
  const uint16_t* q = p.q + (req.begin + j) * p.q_token + head * p.q_head + channel;
  using cached = Cached<act_t, kv_t>;
  using value_t = typename cached::value_t;
  const auto *keys = static_cast<const typename cached::raw_t*>(p.k), *values = static_cast<const typename cached::raw_t*>(p.v);
  last = min(last, paged_limit(p.shape, req, row));
  for (int key = first; key < last; ++key) {
    const int page = paged_quotient(p.page_of, key), place = key - page * p.block_size;
    int64_t at = paged_place(pages[page], place, p.blocks, p.kv_block, p.kv_token);
    if (at < 0) continue;
    at += kv_head * p.kv_head + channel;
    float score = 0.f;
    for (int i = 0; i < D / TEAM; ++i) score = fmaf(to_float(act_t{q[i]}), cached_number<act_t>(keys + at + i), score);
    score = TEAM == 16 ? row16_allreduce(score) : row32_allreduce(score);
    const int64_t scale = cached::SCALED ? pages[page] * p.scale_block + kv_head * p.scale_head + place : 0;
    if constexpr (cached::SCALED) score *= p.k_scales[scale];
    score = score * p.scale_log2 - ((top == -INFINITY ? 0.f : top) - WEIGHT_SHIFT<value_t>);
    float weight = fmaxf(__builtin_amdgcn_exp2f(score), LEAST_PART<value_t>);
    if constexpr (cached::SCALED) weight *= p.v_scales[scale];
#pragma unroll
    for (int i = 0; i < D / TEAM; ++i) o[i] = fmaf(weight, cached_number<act_t>(values + at + i), o[i]);
  }
}

// Wavefronts a workgroup and workgroups a CU, so that 96 to 128 KiB of keys and values are in flight there (64 with blocks of 64
// rows).  More want more of the memory system than it has: 50 requests of 8000 keys (D 128, 1.64 GB) take 265 us with two workgroups of
// four wavefronts, 285 with three and 447 with four (all working together; two working alone 262).  D 64: 37 windows of up to 9000 keys
// (10 heads, 104 MB) take 31.2 us as two workgroups of eight wavefronts and 34.5 as four of four (together; alone 29.9); 32 rows do not
// fit the registers of that (64 windows of eight over 1000 to 16 000 keys, 8 heads, 208 us), and take 147 as one workgroup of eight and
// 150 as three of four.  64 rows of 128 channels need 450 registers: one workgroup.
constexpr int waves(int D, int row_tiles) { return D == 64 && row_tiles == 1 ? 8 : 4; }
constexpr int residency(int D, int row_tiles) {
  return D == 256 || (D == 128 && row_tiles == 4) ? 1 : D == 64 && row_tiles == 2 ? 3 : 2;
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
                   (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32);
}

__device__ __forceinline__ PagedRequest uniform(const PagedRequest& r) {
  return PagedRequest{uniform64(r.begin), __builtin_amdgcn_readfirstlane(r.window), __builtin_amdgcn_readfirstlane(r.length),
                      __builtin_amdgcn_readfirstlane(r.keys), __builtin_amdgcn_readfirstlane(r.blocks), __builtin_amdgcn_readfirstlane(r.tiles)};
}

// A segment as a wavefront takes it.
struct Part {
  PagedRequest req;
  PagedSegment seg;
  int row0, rows;                         // of the window
  int least, end;                         // keys that all rows see, that any row sees
  int key, steps;                         // first key and steps of this wavefront
  int64_t last;                           // unit of the run
  int index;                              // of the request
  const int32_t* pages;
};

// With a prefix it matters whether a row sees a key of its own at all: if it sees some whose scores are all minus infinity, it is the
// attention over the prefix, if none, zeros.  So such sums are not left at zero but made this, which nothing is added to that it would
// change: beside any other maximum it is zero.
constexpr float SUM_OF_NOTHING = 0x1p-126f;

// What a row has of the prefix, joined with what it has of its own keys: a common reference and the factors of both.  A row that sees no
// key of its own (sum 0) has no part in the prefix.
struct PrefixPart {
  int64_t row;                                    // of the prefix's outputs, -1: no part
  float own, prefix;
};
template <typename value_t>
__device__ __forceinline__ PrefixPart prefix_part(const PagedAttention& p, int64_t token, int head, float top, float& sum) {
  PrefixPart x{token * (p.shape.heads * p.shape.group) + head, 1.f, 0.f};
  const float2 y = p.prefix_tops[x.row];
  if (sum == 0.f) {
    x.row = -1;
    return x;
  }
  const float mine = top - WEIGHT_SHIFT<value_t>, reference = fmaxf(mine, y.x);
  x.own = 0.5f * step_factor(mine, reference);          // half of each, as the sum of two numbers may pass 32 bits
  x.prefix = 0.5f * step_factor(y.x, reference);
  sum = fmaf(y.y, x.prefix, sum * x.own);
  if (reference == -INFINITY && sum == sum) sum = 0.f;      // nothing in the prefix either
  return x;
}
template <int CHANNELS>
__device__ __forceinline__ void add_prefix(const PagedAttention& p, const PrefixPart& x, int D, int channel, float (&o)[CHANNELS]) {
  if (x.row < 0) return;
  const float* part = p.prefix + x.row * D + channel;
#pragma unroll
  for (int i = 0; i < CHANNELS; ++i) o[i] = add_brought(brought(o[i], x.own), part[i], x.prefix);
}

// CHANNELS channels of a row's output from their sums.
template <typename act_t, int D, bool PREFIX, int CHANNELS>
__device__ __forceinline__ void write_row(const PagedAttention& p, int64_t token, int head, int channel, float top, float sum, float (&o)[CHANNELS]) {
  if constexpr (PREFIX) add_prefix(p, prefix_part<act_t>(p, token, head, top, sum), D, channel, o);
  const float norm = sum == 0.f ? 0.f : 1.0f / sum;         // no key: zeros
  uint32_t word[CHANNELS / 2];
#pragma unroll
  for (int i = 0; i < CHANNELS; i += 2) {
    float x = o[i] * norm, y = o[i + 1] * norm;
    if (p.gate) {
      const uint32_t g = *reinterpret_cast<const uint32_t*>(p.gate + token * p.gate_token + head * p.gate_head + channel + i);
      x *= 1.0f / (1.0f + __expf(-lo16<act_t>(g)));
      y *= 1.0f / (1.0f + __expf(-hi16<act_t>(g)));
    }
    word[i / 2] = pack2<act_t>(x, y);
  }
  uint16_t* dst = p.out + token * p.out_token + head * p.out_head + channel;
#pragma unroll
  for (int i = 0; i < CHANNELS / 2; ++i) reinterpret_cast<uint32_t*>(dst)[i] = word[i];
}

// The same as add_set_aside for all 16 rows at once, by a wavefront alone: lane (r, kb) has a quarter of row r's channels, from
// `o` on in LDS.  row < 0: none.
template <typename act_t, typename kv_t, int D>
__device__ __forceinline__ void add_set_aside_alone(const PagedAttention& p, const PagedRequest& req, int kv_head, int row, int kb,
                                                    const int32_t* pages, int first, int last, float top, float* o) {
  const int j = row < 0 ? 0 : paged_quotient(p.shape.by_group, row), head = kv_head * p.shape.group + (row < 0 ? 0 : row - j * p.shape.group);
  const uint16_t* q = p.q + (req.begin + j) * p.q_token + head * p.q_head + kb * (D / 4);
  using cached = Cached<act_t, kv_t>;
  using value_t = typename cached::value_t;
  const auto *keys = static_cast<const typename cached::raw_t*>(p.k), *values = static_cast<const typename cached::raw_t*>(p.v);
  const int limit = row < 0 ? 0 : paged_limit(p.shape, req, row);
  for (int key = first; key < last; ++key) {
    const int page = paged_quotient(p.page_of, key), place = key - page * p.block_size;
    int64_t at = paged_place(pages[page], place, p.blocks, p.kv_block, p.kv_token);
    if (at < 0) continue;
    at += kv_head * p.kv_head + kb * (D / 4);
    float score = 0.f;
#pragma nounroll
    for (int i = 0; i < D / 4; ++i) score = fmaf(to_float(act_t{q[i]}), cached_number<act_t>(keys + at + i), score);
    score = query_sum(score);
    const int64_t scale = cached::SCALED ? pages[page] * p.scale_block + kv_head * p.scale_head + place : 0;
    if constexpr (cached::SCALED) score *= p.k_scales[scale];
    score = score * p.scale_log2 - ((top == -INFINITY ? 0.f : top) - WEIGHT_SHIFT<value_t>);
    if (key >= limit) continue;
    float weight = fmaxf(__builtin_amdgcn_exp2f(score), LEAST_PART<value_t>);
    if constexpr (cached::SCALED) weight *= p.v_scales[scale];
#pragma nounroll
    for (int i = 0; i < D / 4; ++i) o[kb * (D / 4) + i] = fmaf(weight, cached_number<act_t>(values + at + i), o[kb * (D / 4) + i]);
  }
}

// Order of this wavefront's own LDS accesses: the LDS serves one wavefront in order, the compiler has to keep it.
__device__ __forceinline__ void own_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Where the stretch of a workgroup starts, or (STARTS > 1) the shares of its wavefronts.
template <int WAVES, int STARTS>
struct StartRoom {
  int64_t sums[WAVES];
  PagedRequest request[STARTS];
  int index[STARTS], offset[STARTS];
};
__device__ __forceinline__ int64_t share_of(int64_t length, int parts, int i) {
  const int64_t each = (int64_t)((uint64_t)length / (uint32_t)parts);
  return each * i + min(i, (int)(length - each * parts));
}

// The line of work, and this workgroup's place in it: all workgroups add up the whole batch, a thread a contiguous share of the
// requests.  Returns the worker, -1 if there is nothing for it.
template <int WAVES, int STARTS>
__device__ __forceinline__ int take_stretch(const PagedAttention& p, StartRoom<WAVES, STARTS>& room, PagedLine& line) {
  constexpr int THREADS = 64 * WAVES;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int share = (p.batch + THREADS - 1) / THREADS, first = min(tid * share, p.batch), last = min(first + share, p.batch);
  int64_t mine = 0;
  PagedRequest own{};
  for (int n = first; n < last; ++n) {
    own = p.request(n);
    mine += paged_weight(p.shape, own);
    if (p.by_run && p.runs && blockIdx.x == 0)    // runs that nobody has
      for (int h = 0; h < p.shape.heads; ++h)
        for (int b = own.blocks; b < p.row_blocks; ++b) p.runs[(n * p.shape.heads + h) * p.row_blocks + b].pieces = 0;
  }
  int64_t below = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t x = __shfl_up(below, d);
    if (lane >= d) below += x;
  }
  if (lane == 63) room.sums[wave] = below;
  __syncthreads();
  int64_t total = 0;
  below -= mine;
  for (int i = 0; i < WAVES; ++i) {
    if (i < wave) below += room.sums[i];
    total += room.sums[i];
  }
  line = paged_line(p.shape, gridDim.x, uniform64(total));
  // neighbours in the line on one XCD: row blocks of the same keys share its L2
  const int block = blockIdx.x, worker = block >= line.workers || line.workers % 8 ? block : (block & 7) * (line.workers / 8) + (block >> 3);
  if (!p.by_run && p.runs && tid == 0) p.runs[worker].pieces = 0;
  if (worker >= line.workers) return -1;
  const int64_t begin = paged_stretch(line, worker), end = paged_stretch(line, worker + 1);
  if (below < end && below + mine > begin) {      // these requests have some of it
    const int64_t length = end - begin;
#pragma nounroll
    for (int i = 0; i < STARTS; ++i) {
      int64_t left = begin + share_of(length, STARTS, i) - below;
      if (left < 0 || left >= mine) continue;
      int n = first;
      if (share > 1)
        for (;; ++n) {
          own = p.request(n);
          if (left < paged_weight(p.shape, own)) break;
          left -= paged_weight(p.shape, own);
        }
      room.request[i] = own;
      room.index[i] = n;
      room.offset[i] = (int)left;
    }
  }
  __syncthreads();
  return worker;
}

// What a wavefront leaves of a run that it did not have alone.
struct PieceOfRun {
  int there, open;                        // open: the run goes on behind this wavefront's keys
  int begin, index, head, block, rows;    // first token row of its request, the request, ...
  int64_t last;                           // unit of the line
};

template <typename act_t, typename kv_t, int D, int RT, bool ALONE, bool PREFIX>
__global__ __launch_bounds__(64 * waves(D, RT), residency(D, RT) * waves(D, RT) / 4) void paged_attention_kernel(const PagedAttention p) {
  using W = Wave<act_t, kv_t, D, RT>;
  using raw_t = typename W::raw_t;
  constexpr int WAVES = waves(D, RT), THREADS = 64 * WAVES, TILE = 32 * WAVES;
  constexpr int TEAM = THREADS / 16, CHANNELS = D / TEAM;       // threads that put a row's outputs together, and channels of each
  constexpr int PITCH = D + 4;                    // floats of a row in LDS: rows of a quad of lanes start in different banks
  constexpr int PIECES = 16 * RT * D / 8, MINE = ALONE ? D / 32 : (PIECES + THREADS - 1) / THREADS;          // 16-byte pieces of the queries, and of a thread
  constexpr int STRIDE = ALONE ? 32 : TILE;       // keys from a wavefront's step to its next
  __shared__ __align__(16) float outs[ALONE ? 2 : 1][WAVES][16][PITCH];
  __shared__ __align__(16) u32x4_t queries[ALONE ? 1 : PIECES];
  __shared__ float2 tops[ALONE ? 2 : 1][WAVES][16 * RT];
  __shared__ int aside[WAVES];
  __shared__ PieceOfRun left[2][ALONE ? WAVES : 1];
  __shared__ StartRoom<WAVES, ALONE ? WAVES : 1> room;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, kb = lane >> 4;
  PagedLine line;
  const int worker = take_stretch(p, room, line);
  if (worker < 0) return;
  int64_t unit = paged_stretch(line, worker), stretch_end = paged_stretch(line, worker + 1);
  if (ALONE) {
    const int64_t length = stretch_end - unit;
    stretch_end = unit + share_of(length, WAVES, wave + 1);
    unit += share_of(length, WAVES, wave);
  }
  const int start = ALONE ? wave : 0;
  int n = __builtin_amdgcn_readfirstlane(room.index[start]);

  const uint32_t key_lane = (uint32_t)(r * p.kv_token) * sizeof(raw_t) + 16 * kb;
  const uint32_t value_lane = (uint32_t)(4 * kb * p.kv_token + W::LANE_CHANNELS * r) * sizeof(raw_t);
  const raw_t *keys = static_cast<const raw_t*>(p.k), *values = static_cast<const raw_t*>(p.v);
  auto key_scales_of = [&](int head) { return W::SCALED ? p.k_scales + head * p.scale_head : nullptr; };
  auto value_scales_of = [&](int head) { return W::SCALED ? p.v_scales + head * p.scale_head : nullptr; };

  // The part of the stretch at `at` in request n, `req`.
  auto part_at = [&](const PagedRequest& req, const PagedStart& at) {
    Part a;
    a.req = req;
    a.index = n;
    a.seg = paged_segment(line, req, at, unit, stretch_end, worker);
    a.last = unit - at.tile + req.tiles - 1;
    unit += a.seg.tiles;
    a.row0 = a.seg.block << p.shape.row_bits;
    a.rows = min(req.window * p.shape.group - a.row0, 16 * RT);
    a.least = paged_limit(p.shape, req, a.row0);
    a.end = paged_limit(p.shape, req, a.row0 + a.rows - 1);
    const int64_t table_row = p.mapping ? scalar_at(p.mapping, p.mapping_wide, n) : n;
    const bool has_row = table_row >= 0 && table_row < p.table_rows;
    a.pages = p.table + (has_row ? table_row : 0) * p.table_row;
    // steps of this wavefront: those of its keys that are below `end`
    a.key = (a.seg.tile << p.shape.tile_bits) + (ALONE ? 0 : 32 * wave);
    const int stop = min(a.end, (a.seg.tile + a.seg.tiles) << p.shape.tile_bits);
    a.steps = has_row && stop > a.key ? (stop - a.key - 1) / STRIDE + 1 : 0;
    return a;
  };
  // The one after it: the next run, of the next request that has any where this one has no more.
  auto part_after = [&](const Part& a) {
    PagedStart at{a.seg.head, a.seg.block + 1, 0};
    PagedRequest req = a.req;
    if (at.block == req.blocks) {
      at.block = 0;
      ++at.head;
    }
    if (at.head == p.shape.heads) {
      at.head = 0;
      do req = scalar_request(p, ++n);
      while (req.blocks == 0);
    }
    return part_at(req, at);
  };
  // Where the two halves of a step's keys lie: the table's entries first (always two loads, of anything where there is no such
  // step: a branch would wait for them), then, when they are there, the places.  Place 0, some block's first keys, serves loads
  // whose results do not count.
  struct Entries { int block[2]; };
  auto look_up = [&](const Part& a, int step) {
    Entries x;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = min(a.key + step * STRIDE + 16 * h, a.end - 1);
      x.block[h] = scalar_load(a.steps > 0 ? a.pages + paged_quotient(p.page_of, key) : static_cast<const int32_t*>(p.lengths));
    }
    return x;
  };
  auto place_of = [&](const Part& a, int step, const Entries& x, int64_t (&place)[2], int64_t (&at)[2], bool (&there)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = a.key + step * STRIDE + 16 * h;
      place[h] = paged_place(x.block[h], key - paged_quotient(p.page_of, key) * p.block_size, p.blocks, p.kv_block, p.kv_token);
      there[h] = a.steps > 0 && key < a.end && place[h] >= 0;
      if (!there[h]) place[h] = 0;
      if constexpr (W::SCALED) at[h] = there[h] ? x.block[h] * p.scale_block + key - paged_quotient(p.page_of, key) * p.block_size : 0;
    }
  };
  // The queries: a wavefront alone keeps its operands, row r at channels 32 c + 8 kb, in registers.  Together a thread has pieces of
  // 16 bytes, which go to where lane 16 kb + r of step c of row tile t reads its operand.
  auto load_queries = [&](const Part& a, u32x4_t (&x)[MINE]) {
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int piece = tid + THREADS * i, row = ALONE ? r : piece / (D / 8);
      const int channel = !ALONE ? piece % (D / 8) * 8 : W::SCALED ? 64 * (i / 2) + 16 * kb + 8 * (i & 1) : 32 * i + 8 * kb;
      x[i] = u32x4_t{0, 0, 0, 0};
      if (row < a.rows) {
        const int j = paged_quotient(p.shape.by_group, a.row0 + row), g = a.row0 + row - j * p.shape.group;
        x[i] = *reinterpret_cast<const u32x4_t*>(p.q + (a.req.begin + j) * p.q_token + (a.seg.head * p.shape.group + g) * p.q_head + channel);
      }
    }
  };
  auto store_queries = [&](const u32x4_t (&x)[MINE]) {
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int piece = tid + THREADS * i, row = piece / (D / 8), chunk = piece % (D / 8);
      // chunks of a step: those whose keys lie in one load of a lane (of 8-bit numbers, which are half as long, every other chunk)
      const int step = W::SCALED ? (chunk >> 3) * 2 + (chunk & 1) : chunk >> 2, group = W::SCALED ? chunk >> 1 & 3 : chunk & 3;
      if (piece < PIECES) queries[((row >> 4) * W::STEPS + step) * 64 + 16 * group + (row & 15)] = x[i];
    }
  };

  W w;
  u32x4_t q_words[MINE];
  int64_t place[2], next_place[2], scale_at[2] = {0, 0}, next_scale_at[2] = {0, 0};
  bool there[2], next_there[2];
  if (ALONE && lane < 2) left[lane][wave] = PieceOfRun{};
  if (!ALONE || unit < stretch_end) {
  const PagedRequest first_request = uniform(room.request[start]);
  Part a = part_at(first_request, paged_start(first_request, __builtin_amdgcn_readfirstlane(room.offset[start])));
  const Entries entries = look_up(a, 0);
  if (a.steps > 0) {
    place_of(a, 0, entries, place, scale_at, there);
    load_keys(w, keys + a.seg.head * p.kv_head, key_scales_of(a.seg.head), place, scale_at, key_lane);
  }
  load_queries(a, q_words);
  if (a.steps > 0) load_values(w, values + a.seg.head * p.kv_head, value_scales_of(a.seg.head), place, scale_at, value_lane, p.kv_token * (int)sizeof(raw_t));
  u32x4_t q_now[ALONE ? MINE : 1];
  if constexpr (ALONE) {
#pragma unroll
    for (int i = 0; i < MINE; ++i) q_now[i] = q_words[i];
  } else {
    store_queries(q_words);
    __syncthreads();
  }
  auto query = [&](int t, int c) { return ALONE ? q_now[ALONE ? c : 0] : queries[ALONE ? 0 : (t * W::STEPS + c) * 64 + lane]; };

  for (;;) {
    // The part after this one is worked out now, and its first keys and values are fetched by this part's last step.
    const bool more_parts = unit < stretch_end;
    Part b = a;
    if (more_parts) {
      b = part_after(a);
      load_queries(b, q_words);
    } else {
      b.steps = 0;
    }
    [[maybe_unused]] int first_key = INT32_MAX;   // with a page, of those that this wavefront has; pages hold whole sixteens
    // entries of the step after the one in flight
    Entries coming = a.steps > 1 ? look_up(a, 1) : look_up(b, 0);
    w.set_aside = -1;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int row = 16 * t + r;
      w.limit[t] = row < a.rows ? paged_limit(p.shape, a.req, a.row0 + row) : 0;
      w.top[t] = -INFINITY;
      w.sum[t] = 0.f;
#pragma unroll
      for (int c = 0; c < W::CHUNKS; ++c)
#pragma unroll
        for (int x = 0; x < W::TILES; ++x) w.o[t][c][x] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    for (int step = 0; step < a.steps; ++step) {
      // The wavefronts of a CU's workgroups take turns: the older ones would always go first, end early and leave the others alone
      // with half of the requests in flight (D 64, 64 windows of four over 4000 keys 124.8 -> 121.2 us, of eight over 1000 to 16 000
      // 167 -> 150).
      if ((step + (blockIdx.x >> 8)) & 1) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
      const bool more = step + 1 < a.steps;
      if constexpr (PREFIX) first_key = min(first_key, there[0] ? a.key + step * STRIDE : there[1] ? a.key + step * STRIDE + 16 : INT32_MAX);
      // The very last step fetches some block's first keys, the same for all, from the caches: a branch around the loads costs the
      // compiler the registers.
      // The entries for the step after next are asked for behind the keys of the next: a wait for queries in LDS is one for them too.
      const int kv_head = more ? a.seg.head : b.seg.head;
      const int64_t head = (more ? a.seg.head : b.seg.head) * p.kv_head;
      attend(w, query, p.scale_log2, there, a.key + step * STRIDE, a.least, a.end,
             [&] {
               place_of(more ? a : b, more ? step + 1 : 0, coming, next_place, next_scale_at, next_there);
               load_keys(w, keys + head, key_scales_of(kv_head), next_place, next_scale_at, key_lane);
               coming = step + 2 < a.steps ? look_up(a, step + 2) : look_up(b, 0);
             },
             [&] { load_values(w, values + head, value_scales_of(kv_head), next_place, next_scale_at, value_lane, p.kv_token * (int)sizeof(raw_t)); });
#pragma unroll
      for (int h = 0; h < 2; ++h) { place[h] = next_place[h]; scale_at[h] = next_scale_at[h]; there[h] = next_there[h]; }
    }
    if (a.steps == 0 && b.steps > 0) {
      place_of(b, 0, coming, place, scale_at, there);
      load_keys(w, keys + b.seg.head * p.kv_head, key_scales_of(b.seg.head), place, scale_at, key_lane);
      load_values(w, values + b.seg.head * p.kv_head, value_scales_of(b.seg.head), place, scale_at, value_lane, p.kv_token * (int)sizeof(raw_t));
    }

    if constexpr (ALONE) {
      const int row = a.row0 + r, j = paged_quotient(p.shape.by_group, row), head = a.seg.head * p.shape.group + row - j * p.shape.group;
      float sum = query_sum(w.sum[0]);
      if constexpr (PREFIX) sum = sum == 0.f && first_key < w.limit[0] ? SUM_OF_NOTHING : sum;
      // this lane's channels of row r: LANE_CHANNELS at a time from these on
      auto channel_of = [&](int c, int e) { return 128 * c + W::LANE_CHANNELS * (4 * kb + e); };
      auto park = [&](float* to) {
#pragma unroll
        for (int c = 0; c < W::CHUNKS; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int x = 0; x < W::TILES; x += 4)
              *reinterpret_cast<float4*>(to + channel_of(c, e) + x) =
                  float4{w.o[0][c][x][e], w.o[0][c][x + 1][e], w.o[0][c][x + 2][e], w.o[0][c][x + 3][e]};
      };
      if (w.set_aside >= 0) {
        float* mine = &outs[1][wave][r][0];               // not in use before the wavefront's last run
        park(mine);
        own_lds_order();
        add_set_aside_alone<act_t, kv_t, D>(p, a.req, a.seg.head, r < a.rows ? row : -1, kb, a.pages, max(w.set_aside & ~31, a.least),
                                      min((w.set_aside & ~31) + (w.set_aside & 1 ? 64 : 32), a.end), w.top[0], mine);
        own_lds_order();
#pragma unroll
        for (int c = 0; c < W::CHUNKS; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int x = 0; x < W::TILES; ++x) w.o[0][c][x][e] = mine[channel_of(c, e) + x];
        own_lds_order();
      }
      if (a.seg.tiles == a.req.tiles) {
        if (r < a.rows) {
          const int64_t token = a.req.begin + j;
          if constexpr (PREFIX) {
            const PrefixPart part = prefix_part<act_t>(p, token, head, w.top[0], sum);
#pragma unroll
            for (int c = 0; c < W::CHUNKS; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float y[W::TILES];
#pragma unroll
                for (int x = 0; x < W::TILES; ++x) y[x] = w.o[0][c][x][e];
                add_prefix(p, part, D, channel_of(c, e), y);
#pragma unroll
                for (int x = 0; x < W::TILES; ++x) w.o[0][c][x][e] = y[x];
              }
          }
          const float norm = sum == 0.f ? 0.f : 1.0f / sum;         // no key: zeros
#pragma unroll
          for (int c = 0; c < W::CHUNKS; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t word[W::WORDS];
#pragma unroll
              for (int x = 0; x < W::WORDS; ++x) {
                float y0 = w.o[0][c][2 * x][e] * norm, y1 = w.o[0][c][2 * x + 1][e] * norm;
                if (p.gate) {
                  const uint32_t g = *reinterpret_cast<const uint32_t*>(p.gate + token * p.gate_token + head * p.gate_head + channel_of(c, e) + 2 * x);
                  y0 *= 1.0f / (1.0f + __expf(-lo16<act_t>(g)));
                  y1 *= 1.0f / (1.0f + __expf(-hi16<act_t>(g)));
                }
                word[x] = pack2<act_t>(y0, y1);
              }
              uint16_t* dst = p.out + token * p.out_token + head * p.out_head + channel_of(c, e);
              if constexpr (W::WORDS == 4) *reinterpret_cast<uint4*>(dst) = make_uint4(word[0], word[1], word[2], word[3]);
              else *reinterpret_cast<uint2*>(dst) = make_uint2(word[0], word[1]);
            }
        }
        if (p.by_run && p.runs && lane == 0) p.runs[(a.index * p.shape.heads + a.seg.head) * p.row_blocks + a.seg.block].pieces = 1;
      } else {
        const int kind = a.seg.tile == 0;
        park(&outs[kind][wave][r][0]);
        if (kb == 0) tops[kind][wave][r] = float2{w.top[0], sum};
        if (lane == 0)
          left[kind][wave] = PieceOfRun{1, a.seg.tile + a.seg.tiles < a.req.tiles, (int)a.req.begin, a.index, a.seg.head, a.seg.block, a.rows, a.last};
      }
    } else {
    // The wavefronts' rows together.
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float sum = query_sum(w.sum[t]);
      if constexpr (PREFIX) sum = sum == 0.f && first_key < w.limit[t] ? SUM_OF_NOTHING : sum;
      if (kb == 0) tops[0][wave][16 * t + r] = float2{w.top[t], sum};
    }
    if (lane == 0) aside[wave] = w.set_aside;
    __syncthreads();
    if (more_parts) store_queries(q_words);
    const int out_row = tid / TEAM, out_channel = tid % TEAM * CHANNELS;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if (16 * t >= a.rows) break;
      float top = -INFINITY;
#pragma unroll
      for (int x = 0; x < WAVES; ++x) top = fmaxf(top, tops[0][x][16 * t + r].x);
      const float f = rescale(w.top[t], top);
#pragma unroll
      for (int c = 0; c < W::CHUNKS; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int j = 0; j < W::TILES; j += 4) {
            const int channel = 128 * c + W::LANE_CHANNELS * (4 * kb + e) + j;
            *reinterpret_cast<float4*>(&outs[0][wave][r][channel]) =
                float4{w.o[t][c][j][e] * f, w.o[t][c][j + 1][e] * f, w.o[t][c][j + 2][e] * f, w.o[t][c][j + 3][e] * f};
          }
      __syncthreads();
      if (16 * t + out_row < a.rows) {
        float row_top = -INFINITY, row_sum = 0.f;
#pragma unroll
        for (int x = 0; x < WAVES; ++x) row_top = fmaxf(row_top, tops[0][x][16 * t + out_row].x);
#pragma unroll
        for (int x = 0; x < WAVES; ++x) row_sum += tops[0][x][16 * t + out_row].y * rescale(tops[0][x][16 * t + out_row].x, row_top);
        float o[CHANNELS];
#pragma unroll
        for (int i = 0; i < CHANNELS; ++i) {
          o[i] = 0.f;
#pragma unroll
          for (int x = 0; x < WAVES; ++x) o[i] += outs[0][x][out_row][out_channel + i];
        }
        const int row = a.row0 + 16 * t + out_row;
        for (int x = 0; x < WAVES; ++x)
          if (aside[x] >= 0)
            add_set_aside<act_t, kv_t, D, TEAM>(p, a.req, a.seg.head, row, out_channel, a.pages, max(aside[x], a.least), min(aside[x] + 32, a.end), row_top, o);
        if (a.seg.slot < 0) {
          const int j = paged_quotient(p.shape.by_group, row), head = a.seg.head * p.shape.group + row - j * p.shape.group;
          write_row<act_t, D, PREFIX, CHANNELS>(p, a.req.begin + j, head, out_channel, row_top, row_sum, o);
        } else {
          const int64_t at = (int64_t)a.seg.slot * (16 * RT) + 16 * t + out_row;
#pragma unroll
          for (int i = 0; i < CHANNELS; ++i) p.partial[at * D + out_channel + i] = o[i];
          if (tid % TEAM == 0) p.tops[at] = float2{row_top, row_sum};
        }
      }
      __syncthreads();
    }
    if (tid == 0 && p.runs && a.seg.tile == 0 && (p.by_run || a.seg.pieces > 1)) {
      // in pieces or not: with a list by run somebody has to say
      PagedRun* run = p.runs + (p.by_run ? (a.index * p.shape.heads + a.seg.head) * p.row_blocks + a.seg.block : worker);
      *run = PagedRun{a.seg.pieces, worker, (int)a.req.begin, a.seg.head, a.row0, a.rows, {0, 0}};
    }
    }
    if (!more_parts) break;
    a = b;
    if constexpr (ALONE) {
#pragma unroll
      for (int i = 0; i < MINE; ++i) q_now[i] = q_words[i];
    }
  }
  }
  if constexpr (ALONE) {
    // Runs that wavefronts of this workgroup share, and what it has of runs that it shares with others: one begun before its stretch
    // (g < 0), and those begun by wavefront g, each with the pieces of the wavefronts behind, which share its rows.
    __syncthreads();
    const bool has = lane < WAVES;
    const bool from_before = has && left[0][lane].there != 0, to_behind = from_before && left[0][lane].open != 0;
    const uint32_t goes_on = (uint32_t)__ballot(from_before), closed = (uint32_t)__ballot(from_before && !to_behind);
    const uint32_t begins = (uint32_t)__ballot(has && left[1][lane].there != 0);
    constexpr int LANES = D / 8, ROWS = 64 / LANES;           // lanes a row, rows at a time
    for (int kind = 0; kind < 2; ++kind) {        // the run that this wavefront's keys begin in, the one that they end in
      if (!((kind ? begins : goes_on) >> wave & 1)) continue;
      const uint32_t before = begins & ((1u << wave) - 1);
      const int g = kind ? wave : before ? 31 - __clz(before) : -1, first = max(g, 0), from = wave + kind;
      const bool more = kind == 0 || (goes_on >> from & 1);
      const uint32_t close = more ? closed >> from : 0;
      const bool open = close == 0;
      const int last = !open ? from + __ffs(close) - 1 : more ? 31 - __clz(goes_on) : wave;
      const PieceOfRun& run = left[g >= 0][first];
      const int rows = run.rows, row0 = run.block << p.shape.row_bits;
      for (int base = (wave - first) * ROWS; base < rows; base += (last - first + 1) * ROWS) {
        const int mine = base + lane / LANES, channel = lane % LANES * 8;
        if (mine >= rows) continue;
        float2 y[WAVES];
        float row_top = -INFINITY, row_sum = 0.f, o[8];
#pragma unroll
        for (int x = 0; x < WAVES; ++x) {
          y[x] = tops[x == g][x][mine];
          if (x < first || x > last) y[x] = float2{-INFINITY, 0.f};
          row_top = fmaxf(row_top, y[x].x);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = 0.f;
#pragma unroll
        for (int x = 0; x < WAVES; ++x) {
          if (x < first || x > last) continue;
          const float f = rescale(y[x].x, row_top);
          row_sum = fmaf(y[x].y, f, row_sum);
          const float4* part = reinterpret_cast<const float4*>(&outs[x == g][x][mine][channel]);
          const float4 low = part[0], high = part[1];
          o[0] = fmaf(low.x, f, o[0]); o[1] = fmaf(low.y, f, o[1]); o[2] = fmaf(low.z, f, o[2]); o[3] = fmaf(low.w, f, o[3]);
          o[4] = fmaf(high.x, f, o[4]); o[5] = fmaf(high.y, f, o[5]); o[6] = fmaf(high.z, f, o[6]); o[7] = fmaf(high.w, f, o[7]);
        }
        if (g >= 0 && !open) {
          const int row = row0 + mine, j = paged_quotient(p.shape.by_group, row), head = run.head * p.shape.group + row - j * p.shape.group;
          write_row<act_t, D, PREFIX, 8>(p, run.begin + j, head, channel, row_top, row_sum, o);
        } else {
          const int64_t at = (int64_t)(2 * worker + (g >= 0)) * 16 + mine;
          float4* dst = reinterpret_cast<float4*>(p.partial + at * D + channel);
          dst[0] = float4{o[0], o[1], o[2], o[3]};
          dst[1] = float4{o[4], o[5], o[6], o[7]};
          if (channel == 0) p.tops[at] = float2{row_top, row_sum};
        }
      }
      if (kind && lane == 0 && p.runs && (p.by_run || open)) {
        PagedRun* list = p.runs + (p.by_run ? (run.index * p.shape.heads + run.head) * p.row_blocks + run.block : worker);
        *list = PagedRun{open ? paged_worker_of(line, run.last) - worker + 1 : 1, worker, run.begin, run.head, row0, run.rows, {0, 0}};
      }
    }
  }
}

// Pieces of a run to its output: a workgroup a run and every gridDim.y-th of its rows.  The wavefronts share the rows, or
// (PER_ROW; many pieces) the pieces of a row; a lane has D / 64 channels.  Everything that a row takes is asked for at once, as
// far as it is no more than AHEAD pieces a wavefront.
template <typename act_t, int D, bool PER_ROW, int WAVES, bool PREFIX>
__global__ __launch_bounds__(64 * WAVES) void paged_join_kernel(const PagedAttention p) {
  constexpr int LANE = D / 64, AHEAD = !PER_ROW ? 8 : D == 256 ? 10 : 18;
  typedef float lane_t __attribute__((ext_vector_type(LANE)));
  __shared__ float outs[PER_ROW ? WAVES : 1][D];
  __shared__ float2 parts[PER_ROW ? WAVES : 1];
  const PagedRun run = p.runs[blockIdx.x];
  const int pieces = run.pieces;
  if (pieces < 2) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), R = 1 << p.shape.row_bits;
  const int first = PER_ROW ? wave : 0, stride = PER_ROW ? WAVES : 1;
  for (int row = PER_ROW ? blockIdx.y : blockIdx.y * WAVES + wave; row < run.rows; row += PER_ROW ? gridDim.y : gridDim.y * WAVES) {
    const int j = paged_quotient(p.shape.by_group, run.row0 + row), head = run.head * p.shape.group + run.row0 + row - j * p.shape.group;
    const int64_t token = run.begin + j;
    uint16_t gate[LANE] = {};
    if (p.gate) {
#pragma unroll
      for (int c = 0; c < LANE; ++c) gate[c] = p.gate[token * p.gate_token + head * p.gate_head + LANE * lane + c];
    }
    // the wavefront's pieces, AHEAD at a time, with a maximum and a sum that run along
    float top = -INFINITY, sum = 0.f;
    lane_t o = {};
    for (int i = first; i < pieces; i += AHEAD * stride) {
      lane_t x[AHEAD];
      float2 y[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int piece = min(i + a * stride, pieces - 1);
        const int64_t at = (int64_t)(piece == 0 ? 2 * run.worker + 1 : 2 * (run.worker + piece)) * R + row;
        x[a] = *reinterpret_cast<const lane_t*>(p.partial + at * D + LANE * lane);
        y[a] = p.tops[at];
      }
      float high = top;
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) high = fmaxf(high, y[a].x);          // one piece twice does no harm here
      const float back = rescale(top, high);
      sum *= back;
      o *= back;
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const bool counts = i + a * stride < pieces;
        const float f = rescale(y[a].x, high);
        sum = counts ? fmaf(y[a].y, f, sum) : sum;
#pragma unroll
        for (int c = 0; c < LANE; ++c) o[c] = counts ? fmaf(x[a][c], f, o[c]) : o[c];
      }
      top = high;
    }
    if constexpr (PER_ROW) {
      *reinterpret_cast<lane_t*>(&outs[wave][LANE * lane]) = o;
      if (lane == 0) parts[wave] = float2{top, sum};
      __syncthreads();
      if (wave == 0) {
        for (int x = 0; x < WAVES; ++x) top = fmaxf(top, parts[x].x);
        sum = 0.f;
        o = lane_t{};
        for (int x = 0; x < WAVES; ++x) {
          const float f = rescale(parts[x].x, top);
          sum = fmaf(parts[x].y, f, sum);
          const lane_t y = *reinterpret_cast<const lane_t*>(&outs[x][LANE * lane]);
#pragma unroll
          for (int c = 0; c < LANE; ++c) o[c] = fmaf(y[c], f, o[c]);
        }
      }
    }
    if (!PER_ROW || wave == 0) {
      float x[LANE];
#pragma unroll
      for (int c = 0; c < LANE; ++c) x[c] = o[c];
      if constexpr (PREFIX) add_prefix(p, prefix_part<act_t>(p, token, head, top, sum), D, LANE * lane, x);
      const float norm = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
      for (int c = 0; c < LANE; ++c) {
        x[c] *= norm;
        if (p.gate) x[c] *= 1.0f / (1.0f + __expf(-to_float(act_t{gate[c]})));
      }
      uint16_t* dst = p.out + token * p.out_token + head * p.out_head + LANE * lane;
      if constexpr (LANE == 1) *dst = from_float<act_t>(x[0]).bits;
      else if constexpr (LANE == 2) *reinterpret_cast<uint32_t*>(dst) = pack2<act_t>(x[0], x[1]);
      else *reinterpret_cast<uint2*>(dst) = uint2{pack2<act_t>(x[0], x[1]), pack2<act_t>(x[2], x[3])};
    }
    if constexpr (PER_ROW) __syncthreads();
  }
}

// How a call is launched: host arithmetic from what the host knows.
struct PagedLaunch {
  int row_tiles, rows, tile, units, extra, row_blocks, workers, by_run, per_row, join_rows;
  bool alone;                             // wavefronts have stretches of their own
  bool split;                             // whether a run can be cut at all
  int64_t runs, bytes, tops_at, runs_at;  // workspace: partial outputs, maxima and sums, runs
};

static int bits_of(int power) {
  int bits = 0;
  while (1 << bits < power) ++bits;
  return bits;
}

static PagedLaunch paged_launch(int batch, int HQ, int HKV, int D, int max_query, int64_t positions) {
  PagedLaunch l{};
  const int window_rows = max_query * (HQ / HKV);
  l.row_tiles = window_rows <= 16 ? 1 : window_rows <= 32 || D == 256 ? 2 : 4;
  l.rows = 16 * l.row_tiles;
  l.row_blocks = (window_rows + l.rows - 1) / l.rows;
  l.runs = (int64_t)batch * HKV * l.row_blocks;
  // Wavefronts alone from a run for every 32 of them on: D 128 with 64 runs 21.8 us together and 21.1 alone, with 32 19.8 and 20.7; D 64
  // with 128 runs 22.3 and 22.3, with 64 17.0 and 18.6; D 256 with 32 runs 26.6 and 22.6, with 16 18.9 and 19.0.  But not where every
  // run is one tile and gets a workgroup: then no run is cut, and no join runs (64 requests of one head, D 128, up to 112 keys, 13.3
  // alone and 9.1).
  // A run counts a unit more than it has: without it 200 ragged windows (4 heads, D 64) take 60.2 us, with it 53.0, with two 52.4
  // (but the 256 requests above 249 in place of 245).
  const int64_t most = 256 * residency(D, l.row_tiles);
  const int waves_of = waves(D, l.row_tiles);
  l.alone = l.row_tiles == 1 && l.runs >= most * waves_of / 32 && !(positions <= 32 * waves_of && l.runs <= most);
  l.tile = l.alone ? 32 : 32 * waves_of;
  l.units = l.alone ? waves_of : 1;
  l.extra = l.alone ? 1 : 0;
  const int64_t tiles = (positions > 0 ? (positions - 1) / l.tile + 1 : 1) + l.extra;
  l.workers = (int)(l.runs * tiles < most * l.units ? (l.runs * tiles + l.units - 1) / l.units : most);
  l.split = tiles > 1;
  l.by_run = l.runs <= l.workers;
  // Join: where few runs share all workers each is in many pieces, and a workgroup takes one row of one run; else a wavefront does.
  const int used = window_rows < l.rows ? window_rows : l.rows;
  l.per_row = l.runs * 16 <= l.workers;
  l.join_rows = l.per_row ? used : (used + 3) / 4;
  if (l.split) {
    const int64_t slots = 2 * (int64_t)l.workers;
    l.tops_at = slots * l.rows * D * 4;
    l.runs_at = l.tops_at + slots * l.rows * 8;
    l.bytes = (l.runs_at + l.workers * (int64_t)sizeof(PagedRun) + 255) / 256 * 256;
  }
  return l;
}

template <typename act_t, typename kv_t, int D, bool PREFIX>
static void launch_paged_attention(const PagedAttention& p, const PagedLaunch& l, hipStream_t s) {
  if (l.alone) paged_attention_kernel<act_t, kv_t, D, 1, true, PREFIX><<<l.workers, 64 * waves(D, 1), 0, s>>>(p);
  else if (l.row_tiles == 1) paged_attention_kernel<act_t, kv_t, D, 1, false, PREFIX><<<l.workers, 64 * waves(D, 1), 0, s>>>(p);
  else if (l.row_tiles == 2) paged_attention_kernel<act_t, kv_t, D, 2, false, PREFIX><<<l.workers, 64 * waves(D, 2), 0, s>>>(p);
  else if constexpr (D != 256) paged_attention_kernel<act_t, kv_t, D, 4, false, PREFIX><<<l.workers, 64 * waves(D, 4), 0, s>>>(p);
  if (!l.split) return;
  const dim3 grid((unsigned)(l.by_run ? l.runs : l.workers), l.join_rows);
  if (l.per_row) paged_join_kernel<act_t, D, true, 16, PREFIX><<<grid, 1024, 0, s>>>(p);
  else paged_join_kernel<act_t, D, false, 4, PREFIX><<<grid, 256, 0, s>>>(p);
}

template <typename act_t, typename kv_t, bool PREFIX>
static void launch_paged_attention(const PagedAttention& p, const PagedLaunch& l, int D, hipStream_t s) {
  if (D == 64) launch_paged_attention<act_t, kv_t, 64, PREFIX>(p, l, s);
  else if (D == 128) launch_paged_attention<act_t, kv_t, 128, PREFIX>(p, l, s);
  else launch_paged_attention<act_t, kv_t, 256, PREFIX>(p, l, s);
}
template <typename act_t>
static void launch_paged_attention(const PagedAttention& p, const PagedLaunch& l, int D, hipStream_t s) {
  if (p.k_scales) launch_paged_attention<act_t, e4m3_t, false>(p, l, D, s);
  else if (p.prefix_tops) launch_paged_attention<act_t, act_t, true>(p, l, D, s);
  else launch_paged_attention<act_t, act_t, false>(p, l, D, s);
}

static int check_shape(int batch, int HQ, int HKV, int D, int max_query, int64_t positions) {
  PLA_REQUIRE(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256, got %d", D);
  PLA_REQUIRE(HKV > 0 && HQ >= HKV && HQ % HKV == 0, "query heads must be a positive multiple of key-value heads");
  PLA_REQUIRE(max_query >= 1 && max_query <= 32, "max_query_len must be between 1 and 32");
  PLA_REQUIRE(max_query * (int64_t)(HQ / HKV) <= (1 << 30), "too many query heads");
  PLA_REQUIRE(batch >= 0 && (int64_t)batch * HKV * ((max_query * (int64_t)(HQ / HKV) + 15) / 16) <= INT32_MAX, "too many requests");
  PLA_REQUIRE(positions >= 0 && positions <= (1 << 30), "a row of the block table must hold at most 2^30 positions");
  // the most units that a request can have: a run's tiles of 32 keys and the one more that it counts where wavefronts work alone
  const int64_t units = (positions > 0 ? (positions - 1) / 32 + 1 : 1) + 1;
  PLA_REQUIRE(units * HKV * ((max_query * (int64_t)(HQ / HKV) + 15) / 16) <= INT32_MAX, "a request with too many heads for its positions");
  return 0;
}

}  // namespace pla

extern "C" int64_t pla_paged_attention_workspace_bytes(int batch, int HQ, int HKV, int head_dim, int max_query_len, int64_t positions) {
  using namespace pla;
  if (check_shape(batch, HQ, HKV, head_dim, max_query_len, positions)) return -1;
  return batch == 0 ? 0 : paged_launch(batch, HQ, HKV, head_dim, max_query_len, positions).bytes;
}

extern "C" int pla_paged_attention_segments(
    const int32_t* offsets, const int32_t* seq_lens, int batch, int tokens, int HQ, int HKV, int head_dim, int max_query_len,
    int64_t positions, int worker, int64_t* segments, int capacity) {
  using namespace pla;
  if (check_shape(batch, HQ, HKV, head_dim, max_query_len, positions) || batch == 0 || !offsets || !seq_lens) return -1;
  const PagedLaunch l = paged_launch(batch, HQ, HKV, head_dim, max_query_len, positions);
  const PagedShape shape{HKV, HQ / HKV, paged_divisor(HQ / HKV), bits_of(l.rows), bits_of(l.tile), l.units, l.extra, max_query_len, tokens, positions};
  auto request = [&](int n) { return paged_request(shape, offsets[n], offsets[n + 1], seq_lens[n]); };
  int64_t total = 0;
  for (int n = 0; n < batch; ++n) total += paged_weight(shape, request(n));
  const PagedLine line = paged_line(shape, l.workers, total);
  if (worker < 0 || worker >= line.workers) return 0;
  int64_t unit = paged_stretch(line, worker), offset = unit;
  const int64_t end = paged_stretch(line, worker + 1);
  int found = 0;
  for (int n = 0; unit < end;) {
    const PagedRequest r = request(n);
    if (offset >= paged_weight(shape, r)) {
      offset -= paged_weight(shape, r);
      ++n;
      continue;
    }
    const PagedSegment s = paged_segment(line, r, paged_start(r, (int)offset), unit, end, worker);
    if (found < capacity) {
      const int64_t row[7] = {n, s.head, s.block, s.tile, s.tiles, s.slot, s.pieces};
      for (int i = 0; i < 7; ++i) segments[7 * found + i] = row[i];
    }
    ++found;
    unit += s.tiles;
    offset += s.tiles;
  }
  return found;
}

namespace pla {

// What a call has beyond the plain one: factors of a cache of 8-bit numbers, a prefix that all rows share.
struct PagedExtras {
  const float *k_scales, *v_scales;
  int64_t scale_block, scale_head;
  const int32_t* prefix_blocks;
  int prefix_pages;
  const void* prefix_len;
  int prefix_len_wide;
};

static int paged_attention(
    const void* q, int64_t q_token, int64_t q_head, const void* k_cache, const void* v_cache,
    int64_t kv_block, int64_t kv_token, int64_t kv_head, int blocks, int block_size,
    const int32_t* block_table, int64_t table_row_stride, int table_rows, int table_cols,
    const void* mapping, int mapping_wide, const void* offsets, int offsets_wide, const void* seq_lens, int seq_lens_wide,
    const void* gate, int64_t gate_token, int64_t gate_head, void* out, int64_t out_token, int64_t out_head,
    float scale, int batch, int tokens, int max_query_len, int HQ, int HKV, int head_dim, int act_dtype, const PagedExtras& extras,
    void* workspace, int64_t workspace_bytes, void* stream) {
  PLA_REQUIRE(block_size > 0 && block_size % 16 == 0, "block_size must be a multiple of 16");
  const int64_t positions = (int64_t)table_cols * block_size;
  if (const int bad = check_shape(batch, HQ, HKV, head_dim, max_query_len, positions)) return bad;
  PLA_REQUIRE(act_dtype == PLA_BF16 || act_dtype == PLA_F16, "activations must be bf16 or fp16");
  PLA_REQUIRE(tokens >= 0 && table_rows >= 0 && table_cols >= 0 && table_row_stride >= table_cols, "invalid dimensions");
  PLA_REQUIRE(offsets || max_query_len >= 1, "invalid dimensions");
  if (batch == 0 || tokens == 0) return 0;
  PLA_REQUIRE(offsets || batch <= tokens, "more requests than token rows");
  PLA_REQUIRE(mapping || batch <= table_rows, "more requests than rows of the block table");
  PLA_REQUIRE(q && k_cache && v_cache && seq_lens && out, "null tensor pointer");
  PLA_REQUIRE(block_table || table_rows == 0 || table_cols == 0, "null tensor pointer");
  PLA_REQUIRE(blocks > 0, "the cache must hold a block");
  const bool scaled = extras.k_scales != nullptr;
  for (const int64_t s : {q_token, q_head, kv_block, kv_token, kv_head, gate_token, gate_head, out_token, out_head})
    PLA_REQUIRE(s % 8 == 0, "rows must be 16-byte aligned");
  for (const void* x : {q, k_cache, v_cache, gate, (const void*)out})
    PLA_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0, "rows must be 16-byte aligned");
  if (scaled) {
    for (const int64_t s : {kv_block, kv_token, kv_head}) PLA_REQUIRE(s % 16 == 0, "rows must be 16-byte aligned");
    PLA_REQUIRE(extras.v_scales && extras.scale_block % 4 == 0 && extras.scale_head % 4 == 0 &&
                    (reinterpret_cast<uintptr_t>(extras.k_scales) | reinterpret_cast<uintptr_t>(extras.v_scales)) % 16 == 0,
                "scales of a block's head must be 16-byte aligned");
  }
  PLA_REQUIRE(kv_token >= 0 && kv_token < (1 << 24), "the cache's token stride must be below 2^24");
  const PagedLaunch l = paged_launch(batch, HQ, HKV, head_dim, max_query_len, positions);
  char* ws = static_cast<char*>(workspace);
  PLA_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "the workspace must be 16-byte aligned");
  PagedAttention p{};
  int64_t taken = 0;
  if (extras.prefix_len) {
    PLA_REQUIRE(!scaled, "a shared prefix stands in a cache of the queries' type");
    PLA_REQUIRE(extras.prefix_pages >= 0 && (int64_t)extras.prefix_pages * block_size <= (1 << 30), "a prefix must have at most 2^30 positions");
    PLA_REQUIRE(extras.prefix_blocks || extras.prefix_pages == 0, "null tensor pointer");
    if (const int bad = check_prompt(1, tokens, HQ, HKV, head_dim)) return bad;
    PromptAttention x{};
    x.q = (const uint16_t*)q; x.q_token = q_token; x.q_head = q_head;
    x.k = (const uint16_t*)k_cache; x.k_token = kv_token; x.k_head = kv_head;
    x.v = (const uint16_t*)v_cache; x.v_token = kv_token; x.v_head = kv_head;
    x.kv_block = kv_block; x.blocks = blocks; x.block_size = block_size; x.page_of = paged_divisor(block_size);
    x.table = extras.prefix_blocks; x.table_rows = extras.prefix_pages ? 1 : 0;
    x.lengths = extras.prefix_len; x.lengths_wide = extras.prefix_len_wide;
    x.batch = 1; x.tokens = tokens; x.heads = HKV; x.group = HQ / HKV; x.by_group = paged_divisor(HQ / HKV);
    x.positions = (int64_t)extras.prefix_pages * block_size;
    const PromptLaunch prompt = prompt_launch(1, tokens, HQ, HKV, head_dim, x.positions, true);
    taken = prompt.bytes;
    if (const int bad = launch_prompt(x, prompt, true, head_dim, scale, act_dtype, workspace, workspace_bytes - l.bytes, static_cast<hipStream_t>(stream)))
      return bad;
    p.prefix = reinterpret_cast<const float*>(ws + prompt.rows_at);
    p.prefix_tops = reinterpret_cast<const float2*>(ws + prompt.row_tops_at);
  }
  PLA_REQUIRE(workspace_bytes >= taken + l.bytes && (taken + l.bytes == 0 || workspace), "workspace too small: %lld bytes needed", (long long)(taken + l.bytes));
  ws += taken;
  p.q = (const uint16_t*)q; p.q_token = q_token; p.q_head = q_head;
  p.k = k_cache; p.v = v_cache; p.kv_block = kv_block; p.kv_token = kv_token; p.kv_head = kv_head;
  p.k_scales = extras.k_scales; p.v_scales = extras.v_scales; p.scale_block = extras.scale_block; p.scale_head = extras.scale_head;
  p.table = block_table; p.table_row = table_row_stride;
  p.mapping = mapping; p.mapping_wide = mapping_wide;
  p.offsets = offsets; p.offsets_wide = offsets_wide;
  p.lengths = seq_lens; p.lengths_wide = seq_lens_wide;
  p.gate = (const uint16_t*)gate; p.gate_token = gate_token; p.gate_head = gate_head;
  p.out = (uint16_t*)out; p.out_token = out_token; p.out_head = out_head;
  p.shape = PagedShape{HKV, HQ / HKV, paged_divisor(HQ / HKV), bits_of(l.rows), bits_of(l.tile), l.units, l.extra, max_query_len, tokens, positions};
  p.batch = batch; p.blocks = blocks; p.block_size = block_size; p.table_rows = table_rows;
  p.page_of = paged_divisor(block_size);
  p.scale_log2 = scale * 1.44269504088896341f;
  p.by_run = l.by_run; p.row_blocks = l.row_blocks;
  if (l.split) {
    p.partial = reinterpret_cast<float*>(ws);
    p.tops = reinterpret_cast<float2*>(ws + l.tops_at);
    p.runs = reinterpret_cast<PagedRun*>(ws + l.runs_at);
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (act_dtype == PLA_BF16) launch_paged_attention<bf16_t>(p, l, head_dim, s);
  else launch_paged_attention<f16_t>(p, l, head_dim, s);
  return check_launch("paged_attention_kernel");
}

}  // namespace pla

extern "C" int pla_paged_attention_launch(
    const void* q, int64_t q_token, int64_t q_head, const void* k_cache, const void* v_cache,
    int64_t kv_block, int64_t kv_token, int64_t kv_head, int blocks, int block_size,
    const int32_t* block_table, int64_t table_row_stride, int table_rows, int table_cols,
    const void* mapping, int mapping_wide, const void* offsets, int offsets_wide, const void* seq_lens, int seq_lens_wide,
    const void* gate, int64_t gate_token, int64_t gate_head, void* out, int64_t out_token, int64_t out_head,
    float scale, int batch, int tokens, int max_query_len, int HQ, int HKV, int head_dim, int act_dtype,
    void* workspace, int64_t workspace_bytes, void* stream) {
  return pla::paged_attention(q, q_token, q_head, k_cache, v_cache, kv_block, kv_token, kv_head, blocks, block_size, block_table, table_row_stride,
                              table_rows, table_cols, mapping, mapping_wide, offsets, offsets_wide, seq_lens, seq_lens_wide, gate, gate_token,
                              gate_head, out, out_token, out_head, scale, batch, tokens, max_query_len, HQ, HKV, head_dim, act_dtype,
                              pla::PagedExtras{}, workspace, workspace_bytes, stream);
}

extern "C" int pla_paged_attention_fp8_launch(
    const void* q, int64_t q_token, int64_t q_head, const void* k_cache, const void* v_cache,
    int64_t kv_block, int64_t kv_token, int64_t kv_head, int blocks, int block_size,
    const float* k_scales, const float* v_scales, int64_t scale_block, int64_t scale_head,
    const int32_t* block_table, int64_t table_row_stride, int table_rows, int table_cols,
    const void* mapping, int mapping_wide, const void* offsets, int offsets_wide, const void* seq_lens, int seq_lens_wide,
    const void* gate, int64_t gate_token, int64_t gate_head, void* out, int64_t out_token, int64_t out_head,
    float scale, int batch, int tokens, int max_query_len, int HQ, int HKV, int head_dim, int act_dtype,
    void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace pla;
  PLA_REQUIRE(k_scales && v_scales, "null tensor pointer");
  PagedExtras extras{};
  extras.k_scales = k_scales; extras.v_scales = v_scales; extras.scale_block = scale_block; extras.scale_head = scale_head;
  return paged_attention(q, q_token, q_head, k_cache, v_cache, kv_block, kv_token, kv_head, blocks, block_size, block_table, table_row_stride,
                         table_rows, table_cols, mapping, mapping_wide, offsets, offsets_wide, seq_lens, seq_lens_wide, gate, gate_token,
                         gate_head, out, out_token, out_head, scale, batch, tokens, max_query_len, HQ, HKV, head_dim, act_dtype,
                         extras, workspace, workspace_bytes, stream);
}

extern "C" int64_t pla_paged_attention_prefix_workspace_bytes(int batch, int tokens, int HQ, int HKV, int head_dim, int max_query_len, int64_t positions,
                                                              int64_t prefix_positions) {
  using namespace pla;
  if (check_shape(batch, HQ, HKV, head_dim, max_query_len, positions) || check_prompt(1, tokens, HQ, HKV, head_dim) || prefix_positions < 0) return -1;
  if (batch == 0 || tokens == 0) return 0;
  return paged_launch(batch, HQ, HKV, head_dim, max_query_len, positions).bytes +
         prompt_launch(1, tokens, HQ, HKV, head_dim, prefix_positions, true).bytes;
}

extern "C" int pla_paged_attention_prefix_launch(
    const void* q, int64_t q_token, int64_t q_head, const void* k_cache, const void* v_cache,
    int64_t kv_block, int64_t kv_token, int64_t kv_head, int blocks, int block_size,
    const int32_t* prefix_blocks, int prefix_pages, const void* prefix_len, int prefix_len_wide,
    const int32_t* block_table, int64_t table_row_stride, int table_rows, int table_cols,
    const void* mapping, int mapping_wide, const void* offsets, int offsets_wide, const void* seq_lens, int seq_lens_wide,
    const void* gate, int64_t gate_token, int64_t gate_head, void* out, int64_t out_token, int64_t out_head,
    float scale, int batch, int tokens, int max_query_len, int HQ, int HKV, int head_dim, int act_dtype,
    void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace pla;
  PLA_REQUIRE(prefix_len, "null tensor pointer");
  PagedExtras extras{};
  extras.prefix_blocks = prefix_blocks; extras.prefix_pages = prefix_pages; extras.prefix_len = prefix_len; extras.prefix_len_wide = prefix_len_wide;
  return paged_attention(q, q_token, q_head, k_cache, v_cache, kv_block, kv_token, kv_head, blocks, block_size, block_table, table_row_stride,
                         table_rows, table_cols, mapping, mapping_wide, offsets, offsets_wide, seq_lens, seq_lens_wide, gate, gate_token,
                         gate_head, out, out_token, out_head, scale, batch, tokens, max_query_len, HQ, HKV, head_dim, act_dtype,
                         extras, workspace, workspace_bytes, stream);
}
