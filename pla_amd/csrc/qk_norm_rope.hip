// Norms of queries and keys for each head, the position rotation and the write into the paged cache, in one pass:
//
//   y = x rsqrt(mean(x^2) + eps) (weight + offset)                     (no weight: y = x)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t) attention_factor  with t = position * inv_freq[i]
//
// for the pairs (i, i + rot/2) or (2i, 2i + 1) of the first `rot` channels; the other channels pass.  Queries go to q_out, keys
// to k_out and / or the cache row of the token's slot, values to the cache as they are.  FP32 throughout, one rounding at the end.
//
// Angles: at position 10^6 a product in FP32 is off by 0.06 radians, and at 2^40 one in FP64 by 0.001.  Position and frequency are
// multiplied in two FP64 words, as revolutions, and only the part below one revolution is narrowed, for v_sin_f32 and v_cos_f32, which
// take revolutions and are off by at most 1.3e-7 between minus and plus a half (measured at 2^20 places).  So an angle is as exact at
// any position up to 2^53, which FP64 holds, as at the first.
//
// Bound by HBM, if the instructions stay out of its way: every row is read once and written once, 16 bytes a lane, D / 8 lanes a row.
// A wavefront takes a step of 64 / (D / 8) heads of one kind (q, k or v) at a time, so pointers, strides and kind are scalars, and
// all of a token's steps in a large call: a lane works out an angle, the pairs go through LDS of the wavefront's own without a
// barrier, and weight, cosine and sine become two factors a channel once for all rows of a kind.  The sum of squares is a few DPP
// steps, the partner channels of the split layout sit in another lane of the row.  16 384 tokens of 32 + 8 heads (D 128, 336 MB) take
// 64 us (5.3 TB/s; a large copy runs at 4.75), with norms 65.5, with norms and both caches (403 MB) 78; a workgroup a token, whose
// wavefronts each worked out the factors for two or three rows, took 65, 85 and 100.  Without the hint that rows go past the caches
// 84, 81 and 97.
// Small calls take a step a wavefront, for the shortest chain: 8 tokens 5.8 us a call, launch bound (kernel 4.6).

#include "decode_common.h"

namespace pla {

struct QkNormRope {
  const uint16_t *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  const void* positions; int positions_wide;
  const void *q_weight, *k_weight; int weights_f32;
  float eps, weight_offset;
  const float* inv_freq; int rot; float attention_factor; int interleaved;
  uint16_t *q_out, *k_out;
  int64_t qo_token, qo_head, ko_token, ko_head;
  uint16_t *k_cache, *v_cache;
  int64_t kc_block, kc_token, kc_head, vc_block, vc_token, vc_head;
  const void* slots; int slots_wide; int block, cache_slots;
  int tokens, HQ, HKV;
  int q_steps, k_steps, steps;        // of a token: for queries, for keys, and with those for values
  int chunk, chunks;                  // steps a wavefront, wavefronts a token
};

template <int LANES>
__device__ __forceinline__ float lanes_allreduce(float x) {
  static_assert(LANES == 8 || LANES == 16 || LANES == 32, "lanes a row");
  if constexpr (LANES == 32) return row32_allreduce(x);
  if constexpr (LANES == 16) return row16_allreduce(x);
  x += dpp_mov<0xB1>(x);
  x += dpp_mov<0x4E>(x);
  x += dpp_mov<0x141>(x);
  return x;
}

template <typename act_t>
__device__ __forceinline__ void widen8(uint4 w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = lo16<act_t>(u[i]); x[2 * i + 1] = hi16<act_t>(u[i]); }
}

// Eight channels of a weight vector, offset added.
template <typename act_t>
__device__ __forceinline__ void weights8(const void* weight, int f32, int channel, float offset, float (&w)[8]) {
  if (f32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(weight) + channel);
    const float4 a = p[0], b = p[1];
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
    widen8<act_t>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(weight) + channel), w);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] += offset;
}

// Through the scalar cache, where the address is one for the wavefront.
__device__ __forceinline__ int64_t scalar_index(const void* base, int wide, int i) {
  typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
  const int32_t* p = static_cast<const int32_t*>(base) + (wide ? 2 * (int64_t)i : i);
  const int32_t low = *(scalar_ptr)p;
  return wide ? (int64_t)((uint64_t)(uint32_t)low | (uint64_t)(uint32_t)*(scalar_ptr)(p + 1) << 32) : (int64_t)low;
}

// position * frequency / (2 pi) without its whole revolutions: what the first word of each product leaves goes on in the second.
__device__ __forceinline__ float part_of_turn(int64_t position, float frequency) {
#pragma clang fp contract(off)
  constexpr double INVERSE_TURN = 0x1.45f306dc9c883p-3, INVERSE_TURN_REST = -0x1.6b01ec5417056p-57;      // of 1 / (2 pi)
  const double p = (double)position, f = (double)frequency;
  const double rate = f * INVERSE_TURN, rate_rest = fma(f, INVERSE_TURN_REST, fma(f, INVERSE_TURN, -rate));
  const double turns = p * rate, turns_rest = fma(p, rate_rest, fma(p, rate, -turns));
  return (float)((turns - rint(turns)) + turns_rest);
}

// Bytes of q and k from which on a call's rows go past the caches; below, whoever reads them next finds them there, which is not in
// these figures.  Through the caches and past them, 32 + 8 heads of 128 channels (us, inputs that change): 1024 tokens 8.4 and 7.1,
// 2048 12.7 and 12.3, 4096 (42 MB) 20.3 and 20.3, 6000 (61 MB) 35.0 and 27.6, 8192 52.5 and 38.1; with norms and both caches, whose
// values and copies are not counted, 1024 10.6 and 9.3, 2048 16.4 and 15.6, 4096 29.2 and 23.9, 6000 44.4 and 35.7.
constexpr int64_t PAST_CACHES = 48ll << 20;
constexpr int WAVES_RESIDENT = 8192;  // on the chip, about

template <typename act_t, int D, bool PAST>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const QkNormRope p) {
  constexpr int LANES = D / 8, HEADS = 64 / LANES, AHEAD = 2;            // heads of a step, steps whose rows are asked for together
  __shared__ __align__(16) float turn[4][2][D / 2];                      // cosines and sines of a wavefront's token
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), item = blockIdx.x * 4 + wave;
  const int token = item / p.chunks, begin = (item - token * p.chunks) * p.chunk, end = min(begin + p.chunk, p.steps);
  if (token >= p.tokens) return;
  const int here = threadIdx.x & 63, lane = here & (LANES - 1), channel = 8 * lane, head = here / LANES;

  // Kind of a step (0 q, 1 k, 2 v) and the head that this lane has of it.
  auto kind_of = [&](int step) { return step < p.q_steps ? 0 : step < p.q_steps + p.k_steps ? 1 : 2; };
  auto head_of = [&](int step, int kind) { return (step - (kind == 0 ? 0 : kind == 1 ? p.q_steps : p.q_steps + p.k_steps)) * HEADS + head; };
  auto load_row = [&](int step) {
    uint4 x = {0, 0, 0, 0};
    if (step >= end) return x;
    const int kind = kind_of(step), h = head_of(step, kind);
    const uint16_t* base = kind == 0 ? p.q + token * p.q_token : kind == 1 ? p.k + token * p.k_token : p.v + token * p.v_token;
    const int64_t stride = kind == 0 ? p.q_head : kind == 1 ? p.k_head : p.v_head;
    if (h < (kind == 0 ? p.HQ : p.HKV)) {
      const uint16_t* row = base + h * stride + channel;
      x = PAST ? __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const v4i_t*>(row))) : *reinterpret_cast<const uint4*>(row);
    }
    return x;
  };
  auto store_row = [&](uint16_t* row, uint4 x) {
    if (PAST) __builtin_nontemporal_store(__builtin_bit_cast(v4i_t, x), reinterpret_cast<v4i_t*>(row + channel));
    else *reinterpret_cast<uint4*>(row + channel) = x;
  };
  // The longest chain first: position, angle, LDS, factors.  Then the rows, then where they go.
  constexpr int FREQUENCIES = D > 128 ? D / 128 : 1;
  float frequency[FREQUENCIES];
  int64_t position = 0;
  if (p.rot) {
    position = scalar_index(p.positions, p.positions_wide, token);
#pragma unroll
    for (int i = 0; i < FREQUENCIES; ++i) frequency[i] = p.inv_freq[min(here + 64 * i, p.rot / 2 - 1)];
  }
  uint4 raw[AHEAD];
#pragma unroll
  for (int a = 0; a < AHEAD; ++a) raw[a] = load_row(begin + a);
  // the token's cache row; negative: nowhere
  int64_t slot = p.slots ? scalar_index(p.slots, p.slots_wide, token) : -1;
  if (slot >= p.cache_slots) slot = -1;
  const int block = slot >= 0 ? (int)slot / p.block : 0, place = slot >= 0 ? (int)slot - block * p.block : 0;
  if (p.rot) {
#pragma unroll
    for (int i = 0; i < FREQUENCIES; ++i) {
      const float part = part_of_turn(position, frequency[i]);
      if (here + 64 * i < p.rot / 2) {
        turn[wave][0][here + 64 * i] = __builtin_amdgcn_cosf(part) * p.attention_factor;
        turn[wave][1][here + 64 * i] = __builtin_amdgcn_sinf(part) * p.attention_factor;
      }
    }
    // other lanes read them: the LDS serves a wavefront in order, the compiler has to keep it
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  // out = rstd (x straight + partner cross)
  const bool turns = channel < p.rot;
  const int half = p.rot / 2;
  const bool split = p.rot && !p.interleaved, upper = split && channel >= half;
  const int partner = !turns || !split ? here : upper ? here - half / 8 : here + half / 8;
  float straight[8], cross[8];
  auto prepare = [&](int kind) {
    const void* weight = kind ? p.k_weight : p.q_weight;
    float w[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = v[i] = 1.f;
    if (weight) {
      weights8<act_t>(weight, p.weights_f32, channel, p.weight_offset, w);
      if (split) weights8<act_t>(weight, p.weights_f32, channel + 8 * (partner - here), p.weight_offset, v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      straight[i] = w[i];
      cross[i] = 0.f;
      if (turns) {
        const int f = split ? channel + i - (upper ? half : 0) : (channel + i) / 2;
        const float s = (split ? upper : (i & 1) != 0) ? turn[wave][1][f] : -turn[wave][1][f];
        straight[i] = w[i] * turn[wave][0][f];
        cross[i] = (split ? v[i] : w[i ^ 1]) * s;
      }
    }
  };

  int prepared = -1;
  for (int step0 = begin; step0 < end; step0 += AHEAD) {
    uint4 now[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) now[a] = raw[a];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) raw[a] = load_row(step0 + AHEAD + a);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int step = step0 + a;
      if (step >= end) break;
      const int kind = kind_of(step), h = head_of(step, kind);
      uint4 result = now[a];
      if (kind < 2) {
        if (kind != prepared) {
          prepare(kind);
          prepared = kind;
        }
        float x[8], y[8];
        widen8<act_t>(now[a], x);
        if (split) {
          uint4 other;
          other.x = __shfl(now[a].x, partner); other.y = __shfl(now[a].y, partner);
          other.z = __shfl(now[a].z, partner); other.w = __shfl(now[a].w, partner);
          widen8<act_t>(other, y);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
        }
        float rstd = 1.f;
        if (kind ? p.k_weight : p.q_weight) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
          rstd = fast_rsqrt(lanes_allreduce<LANES>(sum) * (1.0f / D) + p.eps);
        }
        // (a channel that does not turn has no partner: what stands in its place must not meet the factor of zero)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float along = x[i] * straight[i];
          x[i] = (turns ? fmaf(y[i], cross[i], along) : along) * rstd;
        }
        result = make_uint4(pack2<act_t>(x[0], x[1]), pack2<act_t>(x[2], x[3]), pack2<act_t>(x[4], x[5]), pack2<act_t>(x[6], x[7]));
      }
      if (h >= (kind == 0 ? p.HQ : p.HKV)) continue;
      if (kind == 0) {
        store_row(p.q_out + token * p.qo_token + h * p.qo_head, result);
      } else {
        if (kind == 1 && p.k_out) store_row(p.k_out + token * p.ko_token + h * p.ko_head, result);
        if (slot >= 0)
          store_row(kind == 1 ? p.k_cache + block * p.kc_block + place * p.kc_token + h * p.kc_head
                              : p.v_cache + block * p.vc_block + place * p.vc_token + h * p.vc_head, result);
      }
    }
  }
}

template <typename act_t, int D>
static void launch_qk_norm_rope(QkNormRope p, hipStream_t s) {
  constexpr int HEADS = 64 / (D / 8);
  p.q_steps = (p.HQ + HEADS - 1) / HEADS;
  p.k_steps = (p.HKV + HEADS - 1) / HEADS;
  p.steps = p.q_steps + (p.v_cache ? 2 : 1) * p.k_steps;
  // As many steps a wavefront as leave the chip its wavefronts; a token's angles are worked out by each of its wavefronts.
  const int64_t share = ((int64_t)p.tokens * p.steps + WAVES_RESIDENT - 1) / WAVES_RESIDENT;
  p.chunk = (int)(share < p.steps ? share : p.steps);
  p.chunks = (p.steps + p.chunk - 1) / p.chunk;
  const dim3 grid((unsigned)(((int64_t)p.tokens * p.chunks + 3) / 4));
  if ((int64_t)p.tokens * (p.HQ + p.HKV) * D * 2 > PAST_CACHES) qk_norm_rope_kernel<act_t, D, true><<<grid, 256, 0, s>>>(p);
  else qk_norm_rope_kernel<act_t, D, false><<<grid, 256, 0, s>>>(p);
}

template <typename act_t>
static void launch_qk_norm_rope(const QkNormRope& p, int D, hipStream_t s) {
  if (D == 64) launch_qk_norm_rope<act_t, 64>(p, s);
  else if (D == 128) launch_qk_norm_rope<act_t, 128>(p, s);
  else launch_qk_norm_rope<act_t, 256>(p, s);
}

}  // namespace pla

extern "C" int pla_qk_norm_rope_launch(
    const void* q, const void* k, const void* v, const int64_t* strides, const void* positions, int positions_wide,
    const void* q_weight, const void* k_weight, int weights_f32, float eps, float weight_offset,
    const float* inv_freq, int rotary_dim, float attention_factor, int interleaved,
    void* q_out, void* k_out, void* k_cache, void* v_cache, const void* slots, int slots_wide, int blocks, int block_size,
    int tokens, int HQ, int HKV, int D, int act_dtype, void* stream) {
  using namespace pla;
  PLA_REQUIRE(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256, got %d", D);
  PLA_REQUIRE(act_dtype == PLA_BF16 || act_dtype == PLA_F16, "activations must be bf16 or fp16");
  PLA_REQUIRE(tokens >= 0 && HQ > 0 && HKV > 0, "invalid token or head counts");
  PLA_REQUIRE(rotary_dim >= 0 && rotary_dim <= D && rotary_dim % 16 == 0, "rotary_dim must be a multiple of 16 up to head_dim");
  const int heads = HQ + 2 * HKV;
  PLA_REQUIRE((int64_t)tokens * heads <= INT32_MAX, "too many rows");
  if (tokens == 0) return 0;
  PLA_REQUIRE(q && k && q_out && strides, "null tensor pointer");
  PLA_REQUIRE(rotary_dim == 0 || (positions && inv_freq), "a rotation needs positions and inv_freq");
  PLA_REQUIRE((k_cache != nullptr) == (slots != nullptr) && (v_cache == nullptr || (v && k_cache)),
              "k_cache and slots come together, v_cache with v and both");
  PLA_REQUIRE(k_cache || k_out, "keys need a cache or an output");
  PLA_REQUIRE(k_cache == nullptr || (blocks >= 0 && block_size > 0 && (int64_t)blocks * block_size <= INT32_MAX),
              "a cache must have at most 2^31 - 1 slots");
  for (int i = 0; i < 16; ++i) PLA_REQUIRE(strides[i] % 8 == 0, "rows must be 16-byte aligned");
  for (const void* x : {q, k, v, q_weight, k_weight, (const void*)q_out, (const void*)k_out, (const void*)k_cache, (const void*)v_cache})
    PLA_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0, "rows must be 16-byte aligned");
  const int64_t* t = strides;
  const QkNormRope p{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, t[0], t[1], t[2], t[3], t[4], t[5],
                     positions, positions_wide, q_weight, k_weight, weights_f32, eps, weight_offset, inv_freq, rotary_dim,
                     attention_factor, interleaved, (uint16_t*)q_out, (uint16_t*)k_out, t[6], t[7], t[8], t[9],
                     (uint16_t*)k_cache, (uint16_t*)v_cache, t[10], t[11], t[12], t[13], t[14], t[15],
                     slots, slots_wide, block_size, k_cache ? blocks * block_size : 0, tokens, HQ, HKV, 0, 0, 0, 0, 0};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (act_dtype == PLA_BF16) launch_qk_norm_rope<bf16_t>(p, D, s);
  else launch_qk_norm_rope<f16_t>(p, D, s);
  return check_launch("qk_norm_rope_kernel");
}
