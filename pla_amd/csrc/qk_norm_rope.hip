// Norms of queries and keys for each head, the position rotation and the write into the paged cache, in one pass:
//
//   y = x rsqrt(mean(x^2) + eps) (weight + offset)                     (no weight: y = x)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t) attention_factor  with t = position * inv_freq[i]
//
// for the pairs (i, i + rot/2) or (2i, 2i + 1) of the first `rot` channels; the other channels pass.  Queries go to q_out, keys
// to k_out and / or the cache row of the token's slot, values to the cache as they are.  FP32 throughout, one rounding at the end.
//
// Angles: at position 10^6 a product in FP32 is off by 0.06 radians.  Position and frequency are multiplied in FP64, as
// revolutions, and only the part below one revolution is narrowed: sine and cosine are then good to FP32's own rounding.  A
// workgroup works out the rot/2 pairs of its token once and leaves them in LDS for all of its heads.
//
// Bound by HBM: every row is read once and written once, 16 bytes a lane.  D / 8 lanes hold a row, so its sum of squares is a
// few DPP steps, and the partner channels of the split layout sit in another lane of the same wavefront.

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
  int tokens, HQ, HKV, chunks;        // chunks: workgroups a token
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

// ROWS rows a group of D / 8 lanes, all of one token; their loads go out together, before the angles are worked out.
template <typename act_t, int D, int ROWS>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const QkNormRope p) {
  constexpr int LANES = D / 8, GROUPS = 256 / LANES;
  __shared__ __align__(16) float cosines[D / 2], sines[D / 2];
  const int token = blockIdx.x / p.chunks, chunk = blockIdx.x - token * p.chunks;
  const int group = threadIdx.x / LANES, lane = threadIdx.x & (LANES - 1), channel = 8 * lane;
  const int heads = p.HQ + (p.v_cache ? 2 : 1) * p.HKV;
  const int first = chunk * GROUPS * ROWS + group;

  // the token's cache row, -1: nowhere
  int64_t slot = -1;
  if (p.slots) {
    slot = p.slots_wide ? static_cast<const int64_t*>(p.slots)[token] : (int64_t) static_cast<const int32_t*>(p.slots)[token];
    if (slot >= p.cache_slots) slot = -1;
  }
  uint4 raw[ROWS] = {};
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int h = first + r * GROUPS;
    if (h >= heads) continue;
    const uint16_t* row = h < p.HQ ? p.q + token * p.q_token + h * p.q_head
                        : h < p.HQ + p.HKV ? p.k + token * p.k_token + (h - p.HQ) * p.k_head
                                           : p.v + token * p.v_token + (h - p.HQ - p.HKV) * p.v_head;
    raw[r] = *reinterpret_cast<const uint4*>(row + channel);
  }
  if (p.rot) {
    const int half = p.rot / 2;
    for (int i = threadIdx.x; i < half; i += 256) {
      const int64_t position = p.positions_wide ? static_cast<const int64_t*>(p.positions)[token]
                                                : (int64_t) static_cast<const int32_t*>(p.positions)[token];
      const double turns = (double)position * ((double)p.inv_freq[i] * 0.15915494309189533577);     // 1 / (2 pi)
      float s, c;
      sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
      cosines[i] = c * p.attention_factor;
      sines[i] = s * p.attention_factor;
    }
    __syncthreads();
  }
  // this lane's part of the rotation: out = x * cos + partner * sin, sin with the sign of its side
  const bool turns = channel < p.rot;
  const int half = p.rot / 2, side = p.interleaved ? 0 : half / 8;          // lanes to the partner
  const bool upper = !p.interleaved && channel >= half;
  float cosine[8], sine[8];
  if (turns) {
    const int i0 = p.interleaved ? channel / 2 : upper ? channel - half : channel;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int f = p.interleaved ? i0 + i / 2 : i0 + i;
      cosine[i] = cosines[f];
      sine[i] = (p.interleaved ? (i & 1) != 0 : upper) ? sines[f] : -sines[f];
    }
  }
  const int here = threadIdx.x & 63, partner_lane = !turns || p.interleaved ? here : upper ? here - side : here + side;
  const int partner_channel = channel + 8 * (partner_lane - here);

#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int h = first + r * GROUPS;
    // all lanes of a wavefront take part in the exchange
    uint4 other;
    other.x = __shfl(raw[r].x, partner_lane); other.y = __shfl(raw[r].y, partner_lane);
    other.z = __shfl(raw[r].z, partner_lane); other.w = __shfl(raw[r].w, partner_lane);
    float x[8], y[8];
    widen8<act_t>(raw[r], x);
    widen8<act_t>(other, y);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
    sum = lanes_allreduce<LANES>(sum);
    if (h >= heads) continue;
    const bool is_q = h < p.HQ, is_v = h >= p.HQ + p.HKV;
    uint4 result = raw[r];
    if (!is_v) {
      const void* weight = is_q ? p.q_weight : p.k_weight;
      if (weight) {
        const float rstd = 1.0f / sqrtf(sum * (1.0f / D) + p.eps);
        float w[8];
        weights8<act_t>(weight, p.weights_f32, channel, p.weight_offset, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= rstd * w[i];
        if (turns && !p.interleaved) {
          weights8<act_t>(weight, p.weights_f32, partner_channel, p.weight_offset, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] *= rstd * w[i];
        }
      }
      if (turns) {
        if (p.interleaved) {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], cosine[i], y[i] * sine[i]);
      }
      result = make_uint4(pack2<act_t>(x[0], x[1]), pack2<act_t>(x[2], x[3]), pack2<act_t>(x[4], x[5]), pack2<act_t>(x[6], x[7]));
    }
    const int kv = is_v ? h - p.HQ - p.HKV : h - p.HQ;
    if (is_q) {
      *reinterpret_cast<uint4*>(p.q_out + token * p.qo_token + h * p.qo_head + channel) = result;
    } else if (!is_v && p.k_out) {
      *reinterpret_cast<uint4*>(p.k_out + token * p.ko_token + kv * p.ko_head + channel) = result;
    }
    if (!is_q && slot >= 0) {
      const int block = (int)slot / p.block, place = (int)slot - block * p.block;
      uint16_t* row = is_v ? p.v_cache + block * p.vc_block + place * p.vc_token + kv * p.vc_head
                           : p.k_cache + block * p.kc_block + place * p.kc_token + kv * p.kc_head;
      *reinterpret_cast<uint4*>(row + channel) = result;
    }
  }
}

template <typename act_t, int D>
static void launch_qk_norm_rope(QkNormRope p, hipStream_t s) {
  constexpr int GROUPS = 256 / (D / 8);
  const int heads = p.HQ + (p.v_cache ? 2 : 1) * p.HKV;
  // Few rows: one a group, for the shortest chain.  Many: up to four a group share the token's angles.
  const int per_token = (heads + GROUPS - 1) / GROUPS;
  const int rows = (int64_t)p.tokens * per_token <= 1024 ? 1 : per_token < 4 ? per_token : 4;
  p.chunks = (per_token + rows - 1) / rows;
  const dim3 grid((unsigned)p.tokens * p.chunks);
  switch (rows) {
    case 1: qk_norm_rope_kernel<act_t, D, 1><<<grid, 256, 0, s>>>(p); break;
    case 2: qk_norm_rope_kernel<act_t, D, 2><<<grid, 256, 0, s>>>(p); break;
    case 3: qk_norm_rope_kernel<act_t, D, 3><<<grid, 256, 0, s>>>(p); break;
    default: qk_norm_rope_kernel<act_t, D, 4><<<grid, 256, 0, s>>>(p); break;
  }
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
                     slots, slots_wide, block_size, k_cache ? blocks * block_size : 0, tokens, HQ, HKV, 1};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (act_dtype == PLA_BF16) launch_qk_norm_rope<bf16_t>(p, D, s);
  else launch_qk_norm_rope<f16_t>(p, D, s);
  return check_launch("qk_norm_rope_kernel");
}
