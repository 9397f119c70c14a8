// pla.decode.paged._C: the compiled host layer of the paged softmax-attention operators.  It holds every check of their
// arguments, allocates outputs and workspaces that the caller does not bring from torch's allocator, and launches through the
// C ABI of libpla_gfx950.so on torch's current stream of the tensors' device.  Nothing here computes, synchronises or reads a
// tensor's values, so every call can be captured.  A failed check raises RuntimeError before any launch; shapes and types are
// judged before devices.

#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <initializer_list>
#include <optional>
#include <tuple>

#include "../../include/pla_gfx950.h"

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
void launched(int rc) { TORCH_CHECK(rc == 0, pla_last_error()); }
bool bypass() {                                   // read once, as in the other namespaces
  static const bool on = [] { const char* v = std::getenv("PLA_BYPASS_EXEC"); return v && v[0] == '1' && v[1] == 0; }();
  return on;
}
int wide(const Tensor& t) { return t.scalar_type() == at::kLong ? 1 : 0; }
int wide(const OptTensor& t) { return t ? wide(*t) : 0; }
const void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
int count(int64_t n, const char* what) {
  TORCH_CHECK(n <= INT32_MAX, "too many ", what, ": ", n);
  return (int)n;
}
bool finite(double x) { return std::isfinite((float)x); }
int act_code(const Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, name, " must be bf16 or fp16, got ", t.scalar_type());
  return t.scalar_type() == at::kHalf ? PLA_F16 : PLA_BF16;
}

// Dense int32 / int64 vector of n entries (a strided one is copied).
Tensor index_vector(const Tensor& t, const char* name, int64_t n) {
  TORCH_CHECK(t.dim() == 1 && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong), name, " must be an int32 or int64 vector");
  TORCH_CHECK(t.numel() == n, name, " must have ", n, " entries, got ", t.numel());
  return t.contiguous();
}
void dense_ints(const Tensor& t, const char* name, at::ScalarType type, int64_t n) {
  TORCH_CHECK(t.dim() == 1 && t.scalar_type() == type && t.is_contiguous(), name, " must be a contiguous ", type, " vector");
  TORCH_CHECK(t.numel() == n, name, " must have ", n, " entries, got ", t.numel());
}
void block_table_form(const Tensor& t) {
  TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kInt && (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)),
              "block_table must be int32 [requests, blocks] with dense rows");
}
int64_t table_pitch(const Tensor& t) { return std::max(t.stride(0), t.size(1)); }

void on_one_gpu(const Tensor& ref, const char* name, std::initializer_list<std::pair<const char*, const OptTensor*>> others) {
  for (const auto& [what, t] : others)
    if (*t) TORCH_CHECK((*t)->device() == ref.device(), what, " must be on the device of ", name);
  TORCH_CHECK(ref.is_cuda(), name, " must be a CUDA tensor");
}

// Whether two tensors may share memory.  Views of one buffer interleave (q, k and v of a projection row; K and V of a block): where
// both step by the same stride, what counts is where one lies within a step of the other, dimension by dimension.
struct Dim { int64_t size, stride; };          // bytes
struct Dims { Dim d[8]; int n; };              // of a tensor, largest stride first, without those of one entry or stride 0
int64_t extent(const Dims& t, int from, int64_t element) {
  int64_t n = element;
  for (int i = from; i < t.n; ++i) n += (t.d[i].size - 1) * t.d[i].stride;
  return n;
}
bool lap(const Dims& a, const Dims& b, int i, int j, int64_t ahead, int64_t ea, int64_t eb) {
  // `ahead`: of b's first byte to a's
  if (ahead >= extent(a, i, ea) || -ahead >= extent(b, j, eb)) return false;
  if (i == a.n || j == b.n || a.d[i].stride != b.d[j].stride) return true;
  const int64_t step = a.d[i].stride, rest = ((ahead % step) + step) % step;
  return lap(a, b, i + 1, j + 1, rest, ea, eb) || lap(a, b, i + 1, j + 1, rest - step, ea, eb);
}
Dims dims_of(const Tensor& t) {
  Dims r{{}, 0};
  TORCH_CHECK(t.dim() <= 8, "too many dimensions");
  const int64_t element = t.element_size();
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.size(i) <= 1 || t.stride(i) <= 0) continue;
    int at = r.n++;
    for (; at > 0 && r.d[at - 1].stride < t.stride(i) * element; --at) r.d[at] = r.d[at - 1];
    r.d[at] = {t.size(i), t.stride(i) * element};
  }
  return r;
}
// A step of a dimension leaves the smaller ones behind, or not.
bool folds(const Dims& d, int64_t element) {
  for (int i = 0; i < d.n; ++i)
    if (d.d[i].stride < extent(d, i + 1, element)) return true;
  return false;
}
bool may_overlap(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto base_a = reinterpret_cast<intptr_t>(a.data_ptr()), base_b = reinterpret_cast<intptr_t>(b.data_ptr());
  const int64_t ahead = base_b - base_a;
  if (a.is_contiguous() && ahead >= (int64_t)(a.numel() * a.element_size())) return false;        // the usual case, quickly
  if (b.is_contiguous() && -ahead >= (int64_t)(b.numel() * b.element_size())) return false;
  const Dims x = dims_of(a), y = dims_of(b);
  const int64_t ex = a.element_size(), ey = b.element_size();
  // of rows that lie on each other there may be another one anywhere within a step: what counts is the whole extent
  if (folds(x, ex) || folds(y, ey)) return ahead < extent(x, 0, ex) && -ahead < extent(y, 0, ey);
  return lap(x, y, 0, 0, ahead, ex, ey);
}
bool overlaps_itself(const Tensor& t) {
  if (t.numel() == 0 || t.is_contiguous()) return false;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) return true;
  return folds(dims_of(t), t.element_size());
}
bool same_rows(const Tensor& a, const Tensor& b) { return a.data_ptr() == b.data_ptr() && a.strides() == b.strides(); }
void apart(std::initializer_list<std::pair<const char*, const OptTensor*>> written,
           std::initializer_list<std::pair<const char*, const OptTensor*>> read) {
  for (auto w = written.begin(); w != written.end(); ++w) {
    if (!*w->second) continue;
    TORCH_CHECK(!overlaps_itself(**w->second), w->first, " must not share memory with itself");
    for (auto o = written.begin(); o != w; ++o)
      TORCH_CHECK(!*o->second || !may_overlap(**w->second, **o->second), w->first, " must not share memory with ", o->first);
    for (const auto& [what, t] : read)
      TORCH_CHECK(!*t || !may_overlap(**w->second, **t), w->first, " must not share memory with ", what);
  }
}

// ---- block tables and slot maps ----------------------------------------------------------------------------------

std::tuple<Tensor, Tensor, Tensor, Tensor> paged_kv_plan(
    const Tensor& block_table, const Tensor& held_blocks, const Tensor& free_blocks, const Tensor& free_count, int64_t block_size,
    const Tensor& context_lens, const Tensor& query_lens, const OptTensor& request_indices, int64_t token_capacity,
    const OptTensor& out_offsets, const OptTensor& out_seq_lens, const OptTensor& out_positions, const OptTensor& out_slots) {
  block_table_form(block_table);
  const int64_t rows = block_table.size(0), cols = block_table.size(1);
  TORCH_CHECK(context_lens.dim() == 1, "context_lens must be an int32 or int64 vector");
  const int64_t batch = context_lens.numel();
  const Tensor context = index_vector(context_lens, "context_lens", batch), query = index_vector(query_lens, "query_lens", batch);
  OptTensor mapping;
  if (request_indices) mapping = index_vector(*request_indices, "request_indices", batch);
  dense_ints(held_blocks, "held_blocks", at::kInt, rows);
  TORCH_CHECK(free_blocks.dim() == 1 && free_blocks.scalar_type() == at::kInt && free_blocks.is_contiguous(), "free_blocks must be a contiguous Int vector");
  dense_ints(free_count, "free_count", at::kInt, 1);
  TORCH_CHECK(block_size > 0 && block_size <= (1 << 30) && cols * block_size <= (1 << 30), "block_size must be positive and a row's positions at most 2^30");
  TORCH_CHECK(token_capacity >= 0 && token_capacity <= (1 << 30), "token_capacity must be between 0 and 2^30");
  TORCH_CHECK(mapping || batch <= rows, "more batch entries than rows of the block table");
  const int table_rows = count(rows, "rows of the block table"), entries = count(batch, "batch entries"),
            stack_size = count(free_blocks.numel(), "places for free blocks");
  if (out_offsets) {
    TORCH_CHECK(out_seq_lens && out_positions && out_slots, "the four outputs come together");
    dense_ints(*out_offsets, "query_start_loc", at::kInt, batch + 1);
    dense_ints(*out_seq_lens, "seq_lens", at::kInt, batch);
    dense_ints(*out_positions, "positions", at::kInt, token_capacity);
    dense_ints(*out_slots, "slot_mapping", at::kLong, token_capacity);
  }
  const OptTensor table(block_table), held(held_blocks), stack(free_blocks), height(free_count), ctx(context), qry(query);
  on_one_gpu(block_table, "block_table", {{"held_blocks", &held}, {"free_blocks", &stack}, {"free_count", &height},
                                          {"context_lens", &ctx}, {"query_lens", &qry}, {"request_indices", &mapping},
                                          {"query_start_loc", &out_offsets}, {"seq_lens", &out_seq_lens},
                                          {"positions", &out_positions}, {"slot_mapping", &out_slots}});
  apart({{"block_table", &table}, {"held_blocks", &held}, {"free_blocks", &stack}, {"free_count", &height},
         {"query_start_loc", &out_offsets}, {"seq_lens", &out_seq_lens}, {"positions", &out_positions}, {"slot_mapping", &out_slots}},
        {{"context_lens", &ctx}, {"query_lens", &qry}, {"request_indices", &mapping}});
  const c10::DeviceGuard guard(block_table.device());
  const auto ints = block_table.options();
  Tensor offsets = out_offsets ? *out_offsets : at::empty({batch + 1}, ints);
  Tensor seq_lens = out_offsets ? *out_seq_lens : at::empty({batch}, ints);
  Tensor positions = out_offsets ? *out_positions : at::empty({token_capacity}, ints);
  Tensor slots = out_offsets ? *out_slots : at::empty({token_capacity}, ints.dtype(at::kLong));
  if (!bypass())
    launched(pla_paged_kv_plan_launch(
        context.data_ptr(), wide(context), query.data_ptr(), wide(query), ptr(mapping), wide(mapping), block_table.data_ptr<int32_t>(),
        table_pitch(block_table), table_rows, (int)cols, held_blocks.data_ptr<int32_t>(), free_blocks.data_ptr<int32_t>(),
        free_count.data_ptr<int32_t>(), stack_size, entries, (int)block_size, (int)token_capacity,
        offsets.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(), positions.data_ptr<int32_t>(), slots.data_ptr<int64_t>(),
        stream_of(block_table)));
  return {offsets, seq_lens, positions, slots};
}

// ---- caches ------------------------------------------------------------------------------------------------------

// A dimension of one entry steps nowhere, whatever its stride says.
int64_t step(const Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }
int64_t step(const OptTensor& t, int64_t d) { return t ? step(*t, d) : 0; }

void head_rows(const Tensor& t, const char* name, int64_t tokens, int64_t heads, int64_t D, at::ScalarType act) {
  TORCH_CHECK(t.dim() == 3 && t.size(0) == tokens && t.size(1) == heads && t.size(2) == D, name, " must be [", tokens, ", ", heads, ", ", D,
              "], got ", t.sizes());
  TORCH_CHECK(t.scalar_type() == act, name, " must be ", act, ", got ", t.scalar_type());
  TORCH_CHECK(t.numel() == 0 || (t.stride(2) == 1 && step(t, 0) % 8 == 0 && step(t, 1) % 8 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0),
              name, " must have dense channels and 16-byte aligned rows");
}
void cache_form(const Tensor& t, const char* name, int64_t heads, int64_t D, at::ScalarType act) {
  TORCH_CHECK(t.dim() == 4 && t.size(2) == heads && t.size(3) == D, name, " must be [blocks, block_size, ", heads, ", ", D, "], got ", t.sizes());
  TORCH_CHECK(t.scalar_type() == act, name, " must be ", act, ", got ", t.scalar_type());
  TORCH_CHECK(t.size(0) > 0 && t.size(1) > 0, name, " must hold at least one block");
  const int64_t unit = 16 / t.element_size();
  TORCH_CHECK(t.stride(3) == 1 && step(t, 0) % unit == 0 && step(t, 1) % unit == 0 && step(t, 2) % unit == 0 &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              name, " must have dense channels and 16-byte aligned rows");
  TORCH_CHECK(t.size(0) * t.size(1) <= INT32_MAX, name, " must have at most 2^31 - 1 slots");
}

// Scales of a cache of 8-bit numbers, [blocks, heads, block_size] float32.
void scales_form(const Tensor& t, const char* name, const Tensor& cache) {
  TORCH_CHECK(t.dim() == 3 && t.size(0) == cache.size(0) && t.size(1) == cache.size(2) && t.size(2) == cache.size(1), name, " must be [",
              cache.size(0), ", ", cache.size(2), ", ", cache.size(1), "], got ", t.sizes());
  TORCH_CHECK(t.scalar_type() == at::kFloat, name, " must be float32, got ", t.scalar_type());
  TORCH_CHECK((t.size(2) == 1 || t.stride(2) == 1) && step(t, 0) % 4 == 0 && step(t, 1) % 4 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              name, " must have dense places and 16-byte aligned heads");
}

// Caches that attention reads.
void cache_pair(const Tensor& k_cache, const Tensor& v_cache, int64_t heads, int64_t D, at::ScalarType type) {
  cache_form(k_cache, "k_cache", heads, D, type);
  cache_form(v_cache, "v_cache", heads, D, type);
  TORCH_CHECK(v_cache.sizes() == k_cache.sizes() && step(v_cache, 0) == step(k_cache, 0) && step(v_cache, 1) == step(k_cache, 1) &&
                  step(v_cache, 2) == step(k_cache, 2),
              "k_cache and v_cache must have the same shape and strides");
  TORCH_CHECK(k_cache.size(1) % 16 == 0, "block_size must be a multiple of 16, got ", k_cache.size(1));
  TORCH_CHECK(step(k_cache, 1) < (1 << 24), "the caches' token stride must be below 2^24");
}

// ---- norms, rotation, cache write --------------------------------------------------------------------------------

std::tuple<Tensor, OptTensor> fused_qk_norm_rope(
    const Tensor& q, const Tensor& k, const OptTensor& positions_in, const OptTensor& q_weight, const OptTensor& k_weight, double eps,
    double weight_offset, const OptTensor& inv_freq, double attention_factor, bool interleaved, const OptTensor& q_out_in,
    const OptTensor& k_out_in, const OptTensor& v, const OptTensor& k_cache, const OptTensor& v_cache, const OptTensor& slots_in,
    const OptTensor& k_scales, const OptTensor& v_scales) {
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3, "q and k must be [tokens, heads, head_dim]");
  const int64_t T = q.size(0), HQ = q.size(1), HKV = k.size(1), D = q.size(2);
  TORCH_CHECK(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256, got ", D);
  TORCH_CHECK(HQ > 0 && HKV > 0, "q and k must have heads");
  const int act = act_code(q, "q");
  const at::ScalarType type = q.scalar_type();
  head_rows(q, "q", T, HQ, D, type);
  head_rows(k, "k", T, HKV, D, type);
  TORCH_CHECK(T * (HQ + 2 * HKV) <= INT32_MAX, "too many rows");
  for (const auto& [name, w] : {std::pair<const char*, const OptTensor*>{"q_weight", &q_weight}, {"k_weight", &k_weight}}) {
    if (!*w) continue;
    const Tensor& t = **w;
    TORCH_CHECK(t.dim() == 1 && t.numel() == D && t.is_contiguous() && (t.scalar_type() == type || t.scalar_type() == at::kFloat) &&
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
                name, " must be ", D, " contiguous values of q's type or float32, 16-byte aligned");
  }
  TORCH_CHECK(!q_weight || !k_weight || q_weight->scalar_type() == k_weight->scalar_type(), "q_weight and k_weight must be of one type");
  TORCH_CHECK(finite(eps) && eps >= 0 && finite(weight_offset) && finite(attention_factor),
              "eps, weight_offset and attention_factor must be finite, eps not negative");
  int64_t rot = 0;
  OptTensor positions;
  if (inv_freq) {
    TORCH_CHECK(inv_freq->dim() == 1 && inv_freq->scalar_type() == at::kFloat && inv_freq->is_contiguous(), "inv_freq must be a contiguous float32 vector");
    rot = 2 * inv_freq->numel();
    TORCH_CHECK(rot > 0 && rot <= D && rot % 16 == 0, "rotary_dim (twice the frequencies) must be a multiple of 16 up to head_dim, got ", rot);
    TORCH_CHECK(positions_in.has_value(), "a rotation needs positions");
    positions = index_vector(*positions_in, "positions", T);
  }
  TORCH_CHECK(k_cache.has_value() == slots_in.has_value(), "k_cache and slot_mapping come together");
  TORCH_CHECK(v_cache.has_value() == v.has_value() && (!v || k_cache), "v comes with v_cache, and both with k_cache");
  OptTensor slots;
  const at::ScalarType stored = k_scales ? at::kFloat8_e4m3fn : type;
  TORCH_CHECK(!k_scales || k_cache, "k_scales come with k_cache");
  TORCH_CHECK(v_scales.has_value() == (k_scales.has_value() && v.has_value()), "v_scales come with v and k_scales");
  if (k_cache) {
    cache_form(*k_cache, "k_cache", HKV, D, stored);
    if (k_scales) scales_form(*k_scales, "k_scales", *k_cache);
    slots = index_vector(*slots_in, "slot_mapping", T);
  }
  if (v) {
    head_rows(*v, "v", T, HKV, D, type);
    cache_form(*v_cache, "v_cache", HKV, D, stored);
    if (v_scales) scales_form(*v_scales, "v_scales", *v_cache);
    TORCH_CHECK(v_cache->size(0) == k_cache->size(0) && v_cache->size(1) == k_cache->size(1), "k_cache and v_cache must have the same blocks");
  }
  if (q_out_in) head_rows(*q_out_in, "q_out", T, HQ, D, type);
  if (k_out_in) head_rows(*k_out_in, "k_out", T, HKV, D, type);
  const OptTensor qt(q), kt(k);
  on_one_gpu(q, "q", {{"k", &kt}, {"v", &v}, {"positions", &positions}, {"q_weight", &q_weight}, {"k_weight", &k_weight},
                      {"inv_freq", &inv_freq}, {"q_out", &q_out_in}, {"k_out", &k_out_in}, {"k_cache", &k_cache},
                      {"v_cache", &v_cache}, {"slot_mapping", &slots}, {"k_scales", &k_scales}, {"v_scales", &v_scales}});
  // in place: the very rows of the input, each of which one group of lanes reads and writes
  const bool q_in_place = q_out_in && same_rows(*q_out_in, q), k_in_place = k_out_in && same_rows(*k_out_in, k);
  const OptTensor none, other_q = q_in_place ? none : qt, other_k = k_in_place ? none : kt;
  apart({{"q_out", &q_out_in}, {"k_out", &k_out_in}, {"k_cache", &k_cache}, {"v_cache", &v_cache}, {"k_scales", &k_scales}, {"v_scales", &v_scales}},
        {{"q", &other_q}, {"k", &other_k}, {"v", &v}, {"positions", &positions}, {"q_weight", &q_weight}, {"k_weight", &k_weight},
         {"inv_freq", &inv_freq}, {"slot_mapping", &slots}});
  TORCH_CHECK(!q_in_place || !may_overlap(*q_out_in, k), "q_out must not share memory with k");
  TORCH_CHECK(!k_in_place || !may_overlap(*k_out_in, q), "k_out must not share memory with q");

  const c10::DeviceGuard guard(q.device());
  Tensor q_out = q_out_in ? *q_out_in : at::empty({T, HQ, D}, q.options());
  OptTensor k_out = k_out_in;
  if (!k_out && !k_cache) k_out = at::empty({T, HKV, D}, q.options());
  if (bypass() || T == 0) return {q_out, k_out};
  const int64_t strides[16] = {step(q, 0), step(q, 1), step(k, 0), step(k, 1), step(v, 0), step(v, 1), step(q_out, 0), step(q_out, 1),
                               step(k_out, 0), step(k_out, 1), step(k_cache, 0), step(k_cache, 1), step(k_cache, 2),
                               step(v_cache, 0), step(v_cache, 1), step(v_cache, 2)};
  const bool f32 = (q_weight && q_weight->scalar_type() == at::kFloat) || (k_weight && k_weight->scalar_type() == at::kFloat);
  const float* frequencies = inv_freq ? inv_freq->data_ptr<float>() : nullptr;
  void *k_to = k_out ? k_out->data_ptr() : nullptr, *k_cached = k_cache ? k_cache->data_ptr() : nullptr, *v_cached = v_cache ? v_cache->data_ptr() : nullptr;
  const int blocks = k_cache ? (int)k_cache->size(0) : 0, block_size = k_cache ? (int)k_cache->size(1) : 0;
  if (k_scales) {
    const int64_t scale_strides[4] = {step(k_scales, 0), step(k_scales, 1), step(v_scales, 0), step(v_scales, 1)};
    launched(pla_qk_norm_rope_fp8_launch(
        q.data_ptr(), k.data_ptr(), ptr(v), strides, ptr(positions), wide(positions), ptr(q_weight), ptr(k_weight), f32 ? 1 : 0, (float)eps,
        (float)weight_offset, frequencies, (int)rot, (float)attention_factor, interleaved ? 1 : 0, q_out.data_ptr(), k_to, k_cached, v_cached,
        k_scales->data_ptr<float>(), v_scales ? v_scales->data_ptr<float>() : nullptr, scale_strides, ptr(slots), wide(slots), blocks, block_size,
        (int)T, (int)HQ, (int)HKV, (int)D, act, stream_of(q)));
  } else {
    launched(pla_qk_norm_rope_launch(
        q.data_ptr(), k.data_ptr(), ptr(v), strides, ptr(positions), wide(positions), ptr(q_weight), ptr(k_weight), f32 ? 1 : 0, (float)eps,
        (float)weight_offset, frequencies, (int)rot, (float)attention_factor, interleaved ? 1 : 0, q_out.data_ptr(), k_to, k_cached, v_cached,
        ptr(slots), wide(slots), blocks, block_size, (int)T, (int)HQ, (int)HKV, (int)D, act, stream_of(q)));
  }
  return {q_out, k_out};
}

// ---- attention ---------------------------------------------------------------------------------------------------

Tensor paged_attention_decode(
    const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table, const Tensor& seq_lens_in,
    const OptTensor& offsets_in, const OptTensor& request_indices, int64_t max_query_len, std::optional<double> scale,
    const OptTensor& output_gate, const OptTensor& out_in, const OptTensor& k_scales, const OptTensor& v_scales, const OptTensor& prefix_blocks,
    const OptTensor& prefix_len_in) {
  TORCH_CHECK(q.dim() == 3, "q must be [tokens, heads, head_dim]");
  const int64_t T = q.size(0), HQ = q.size(1), D = q.size(2);
  TORCH_CHECK(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256, got ", D);
  const int act = act_code(q, "q");
  const at::ScalarType type = q.scalar_type();
  head_rows(q, "q", T, HQ, D, type);
  TORCH_CHECK(k_cache.dim() == 4, "k_cache must be [blocks, block_size, heads, head_dim]");
  const int64_t HKV = k_cache.size(2), block_size = k_cache.size(1);
  TORCH_CHECK(HKV > 0 && HQ >= HKV && HQ % HKV == 0, "query heads must be a positive multiple of key-value heads, got ", HQ, " and ", HKV);
  TORCH_CHECK(k_scales.has_value() == v_scales.has_value(), "k_scales and v_scales come together");
  cache_pair(k_cache, v_cache, HKV, D, k_scales ? at::kFloat8_e4m3fn : type);
  if (k_scales) {
    scales_form(*k_scales, "k_scales", k_cache);
    scales_form(*v_scales, "v_scales", v_cache);
    TORCH_CHECK(step(k_scales, 0) == step(v_scales, 0) && step(k_scales, 1) == step(v_scales, 1), "k_scales and v_scales must have the same strides");
  }
  TORCH_CHECK(prefix_blocks.has_value() == prefix_len_in.has_value(), "prefix_blocks and prefix_len come together");
  TORCH_CHECK(!prefix_blocks || !k_scales, "a shared prefix stands in a cache of q's type");
  OptTensor prefix_len;
  if (prefix_blocks) {
    TORCH_CHECK(prefix_blocks->dim() == 1 && prefix_blocks->scalar_type() == at::kInt && prefix_blocks->is_contiguous(), "prefix_blocks must be a contiguous int32 vector");
    TORCH_CHECK(prefix_blocks->numel() * block_size <= (1 << 30), "a prefix must have at most 2^30 positions");
    prefix_len = index_vector(*prefix_len_in, "prefix_len", 1);
    TORCH_CHECK(T * HQ <= (1 << 30), "too many rows");
  }
  block_table_form(block_table);
  const int64_t rows = block_table.size(0), cols = block_table.size(1);
  TORCH_CHECK(cols * block_size <= (1 << 30), "a row of the block table must hold at most 2^30 positions");
  TORCH_CHECK(seq_lens_in.dim() == 1, "seq_lens must be an int32 or int64 vector");
  const int64_t batch = seq_lens_in.numel();
  const Tensor seq_lens = index_vector(seq_lens_in, "seq_lens", batch);
  TORCH_CHECK(max_query_len >= 1 && max_query_len <= 32, "max_query_len must be between 1 and 32, got ", max_query_len);
  OptTensor offsets, mapping;
  if (offsets_in) offsets = index_vector(*offsets_in, "query_start_loc", batch + 1);
  else TORCH_CHECK(T == batch, "without query_start_loc every request has one token row: ", batch, " requests, ", T, " rows");
  if (request_indices) mapping = index_vector(*request_indices, "request_indices", batch);
  else TORCH_CHECK(batch <= rows, "more requests than rows of the block table");
  const int requests = count(batch, "requests"), tokens = count(T, "token rows"), heads = count(HQ, "heads"), table_rows = count(rows, "rows of the block table");
  TORCH_CHECK(!scale || finite(*scale), "scale must be finite");
  if (output_gate) head_rows(*output_gate, "output_gate", T, HQ, D, type);
  if (out_in) head_rows(*out_in, "out", T, HQ, D, type);
  const OptTensor qt(q), kt(k_cache), vt(v_cache), table(block_table), lens(seq_lens);
  on_one_gpu(q, "q", {{"k_cache", &kt}, {"v_cache", &vt}, {"block_table", &table}, {"seq_lens", &lens}, {"query_start_loc", &offsets},
                      {"request_indices", &mapping}, {"output_gate", &output_gate}, {"out", &out_in}, {"k_scales", &k_scales}, {"v_scales", &v_scales},
                      {"prefix_blocks", &prefix_blocks}, {"prefix_len", &prefix_len}});
  apart({{"out", &out_in}}, {{"q", &qt}, {"k_cache", &kt}, {"v_cache", &vt}, {"block_table", &table}, {"seq_lens", &lens},
                             {"query_start_loc", &offsets}, {"request_indices", &mapping}, {"output_gate", &output_gate}, {"k_scales", &k_scales},
                             {"v_scales", &v_scales}, {"prefix_blocks", &prefix_blocks}, {"prefix_len", &prefix_len}});

  const c10::DeviceGuard guard(q.device());
  Tensor out = out_in ? *out_in : at::empty({T, HQ, D}, q.options());
  if (bypass() || T == 0 || batch == 0) return out;
  const int64_t positions = cols * block_size;
  const int64_t bytes = prefix_len ? pla_paged_attention_prefix_workspace_bytes(requests, tokens, heads, (int)HKV, (int)D, (int)max_query_len, positions,
                                                                                prefix_blocks->numel() * block_size)
                                   : pla_paged_attention_workspace_bytes(requests, heads, (int)HKV, (int)D, (int)max_query_len, positions);
  TORCH_CHECK(bytes >= 0, pla_last_error());
  Tensor workspace;
  if (bytes > 0) workspace = at::empty({bytes}, q.options().dtype(at::kByte));
  const float factor = (float)scale.value_or(1.0 / std::sqrt((double)D));
  void* ws = bytes > 0 ? workspace.data_ptr() : nullptr;
  const auto launch = [&](auto entry, auto... extras) {
    launched(entry(q.data_ptr(), step(q, 0), step(q, 1), k_cache.data_ptr(), v_cache.data_ptr(), step(k_cache, 0), step(k_cache, 1), step(k_cache, 2),
                   (int)k_cache.size(0), (int)block_size, extras..., block_table.data_ptr<int32_t>(), table_pitch(block_table), table_rows, (int)cols,
                   ptr(mapping), wide(mapping), ptr(offsets), wide(offsets), seq_lens.data_ptr(), wide(seq_lens), ptr(output_gate),
                   step(output_gate, 0), step(output_gate, 1), out.data_ptr(), step(out, 0), step(out, 1), factor, requests, tokens,
                   (int)max_query_len, heads, (int)HKV, (int)D, act, ws, bytes, stream_of(q)));
  };
  if (k_scales)
    launch(pla_paged_attention_fp8_launch, k_scales->data_ptr<float>(), v_scales->data_ptr<float>(), step(k_scales, 0), step(k_scales, 1));
  else if (prefix_len)
    launch(pla_paged_attention_prefix_launch, prefix_blocks->data_ptr<int32_t>(), (int)prefix_blocks->numel(), prefix_len->data_ptr(), wide(prefix_len));
  else
    launch(pla_paged_attention_launch);
  return out;
}

// ---- prompts -----------------------------------------------------------------------------------------------------

// Heads of q and of a tensor with key-value heads.
void query_heads(int64_t HQ, int64_t HKV) {
  TORCH_CHECK(HKV > 0 && HQ >= HKV && HQ % HKV == 0, "query heads must be a positive multiple of key-value heads, got ", HQ, " and ", HKV);
}

Tensor packed_attention_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& offsets_in, const OptTensor& key_offsets_in,
                            std::optional<double> scale, const OptTensor& output_gate, const OptTensor& out_in) {
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3, "q and k must be [tokens, heads, head_dim]");
  const int64_t T = q.size(0), HQ = q.size(1), D = q.size(2), keys = k.size(0), HKV = k.size(1);
  TORCH_CHECK(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256, got ", D);
  const int act = act_code(q, "q");
  const at::ScalarType type = q.scalar_type();
  query_heads(HQ, HKV);
  head_rows(q, "q", T, HQ, D, type);
  head_rows(k, "k", keys, HKV, D, type);
  head_rows(v, "v", keys, HKV, D, type);
  TORCH_CHECK(step(k, 0) < (1 << 24) && step(v, 0) < (1 << 24), "the token strides of k and v must be below 2^24");
  TORCH_CHECK(offsets_in.dim() == 1 && offsets_in.numel() >= 1, "cu_seqlens must be an int32 or int64 vector of at least one entry");
  const int64_t batch = offsets_in.numel() - 1;
  const Tensor offsets = index_vector(offsets_in, "cu_seqlens", batch + 1);
  OptTensor key_offsets;
  if (key_offsets_in) key_offsets = index_vector(*key_offsets_in, "cu_seqlens_k", batch + 1);
  else TORCH_CHECK(keys == T, "without cu_seqlens_k there is a key for every token: ", T, " tokens, ", keys, " keys");
  TORCH_CHECK(T * HQ <= (1 << 30) && keys <= INT32_MAX - 1024, "too many rows");
  const int sequences = count(batch, "sequences");
  TORCH_CHECK(!scale || finite(*scale), "scale must be finite");
  if (output_gate) head_rows(*output_gate, "output_gate", T, HQ, D, type);
  if (out_in) head_rows(*out_in, "out", T, HQ, D, type);
  const OptTensor qt(q), kt(k), vt(v), off(offsets);
  on_one_gpu(q, "q", {{"k", &kt}, {"v", &vt}, {"cu_seqlens", &off}, {"cu_seqlens_k", &key_offsets}, {"output_gate", &output_gate}, {"out", &out_in}});
  apart({{"out", &out_in}}, {{"q", &qt}, {"k", &kt}, {"v", &vt}, {"cu_seqlens", &off}, {"cu_seqlens_k", &key_offsets}, {"output_gate", &output_gate}});

  const c10::DeviceGuard guard(q.device());
  Tensor out = out_in ? *out_in : at::empty({T, HQ, D}, q.options());
  if (bypass() || T == 0 || batch == 0) return out;
  const int64_t bytes = pla_prompt_attention_workspace_bytes(sequences, T, (int)HQ, (int)HKV, (int)D, keys);
  TORCH_CHECK(bytes >= 0, pla_last_error());
  Tensor workspace;
  if (bytes > 0) workspace = at::empty({bytes}, q.options().dtype(at::kByte));
  launched(pla_prompt_attention_launch(
      q.data_ptr(), step(q, 0), step(q, 1), k.data_ptr(), step(k, 0), step(k, 1), v.data_ptr(), step(v, 0), step(v, 1), offsets.data_ptr(),
      wide(offsets), ptr(key_offsets), wide(key_offsets), ptr(output_gate), step(output_gate, 0), step(output_gate, 1), out.data_ptr(), step(out, 0),
      step(out, 1), (float)scale.value_or(1.0 / std::sqrt((double)D)), sequences, (int)T, keys, (int)HQ, (int)HKV, (int)D, act,
      bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_of(q)));
  return out;
}

Tensor paged_attention_prefill(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table, const Tensor& seq_lens_in,
                               const Tensor& offsets_in, const OptTensor& request_indices, std::optional<double> scale,
                               const OptTensor& output_gate, const OptTensor& out_in) {
  TORCH_CHECK(q.dim() == 3, "q must be [tokens, heads, head_dim]");
  const int64_t T = q.size(0), HQ = q.size(1), D = q.size(2);
  TORCH_CHECK(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256, got ", D);
  const int act = act_code(q, "q");
  const at::ScalarType type = q.scalar_type();
  head_rows(q, "q", T, HQ, D, type);
  TORCH_CHECK(k_cache.dim() == 4, "k_cache must be [blocks, block_size, heads, head_dim]");
  const int64_t HKV = k_cache.size(2), block_size = k_cache.size(1);
  query_heads(HQ, HKV);
  cache_pair(k_cache, v_cache, HKV, D, type);
  block_table_form(block_table);
  const int64_t rows = block_table.size(0), cols = block_table.size(1);
  TORCH_CHECK(cols * block_size <= (1 << 30), "a row of the block table must hold at most 2^30 positions");
  TORCH_CHECK(seq_lens_in.dim() == 1, "seq_lens must be an int32 or int64 vector");
  const int64_t batch = seq_lens_in.numel();
  const Tensor seq_lens = index_vector(seq_lens_in, "seq_lens", batch), offsets = index_vector(offsets_in, "query_start_loc", batch + 1);
  OptTensor mapping;
  if (request_indices) mapping = index_vector(*request_indices, "request_indices", batch);
  else TORCH_CHECK(batch <= rows, "more requests than rows of the block table");
  TORCH_CHECK(T * HQ <= (1 << 30), "too many rows");
  const int requests = count(batch, "requests"), table_rows = count(rows, "rows of the block table");
  TORCH_CHECK(!scale || finite(*scale), "scale must be finite");
  if (output_gate) head_rows(*output_gate, "output_gate", T, HQ, D, type);
  if (out_in) head_rows(*out_in, "out", T, HQ, D, type);
  const OptTensor qt(q), kt(k_cache), vt(v_cache), table(block_table), lens(seq_lens), off(offsets);
  on_one_gpu(q, "q", {{"k_cache", &kt}, {"v_cache", &vt}, {"block_table", &table}, {"seq_lens", &lens}, {"query_start_loc", &off},
                      {"request_indices", &mapping}, {"output_gate", &output_gate}, {"out", &out_in}});
  apart({{"out", &out_in}}, {{"q", &qt}, {"k_cache", &kt}, {"v_cache", &vt}, {"block_table", &table}, {"seq_lens", &lens},
                             {"query_start_loc", &off}, {"request_indices", &mapping}, {"output_gate", &output_gate}});

  const c10::DeviceGuard guard(q.device());
  Tensor out = out_in ? *out_in : at::empty({T, HQ, D}, q.options());
  if (bypass() || T == 0 || batch == 0) return out;
  const int64_t bytes = pla_prompt_attention_workspace_bytes(requests, T, (int)HQ, (int)HKV, (int)D, cols * block_size);
  TORCH_CHECK(bytes >= 0, pla_last_error());
  Tensor workspace;
  if (bytes > 0) workspace = at::empty({bytes}, q.options().dtype(at::kByte));
  launched(pla_paged_prompt_attention_launch(
      q.data_ptr(), step(q, 0), step(q, 1), k_cache.data_ptr(), v_cache.data_ptr(), step(k_cache, 0), step(k_cache, 1),
      step(k_cache, 2), (int)k_cache.size(0), (int)block_size, block_table.data_ptr<int32_t>(), table_pitch(block_table), table_rows,
      (int)cols, ptr(mapping), wide(mapping), offsets.data_ptr(), wide(offsets), seq_lens.data_ptr(), wide(seq_lens), ptr(output_gate),
      step(output_gate, 0), step(output_gate, 1), out.data_ptr(), step(out, 0), step(out, 1),
      (float)scale.value_or(1.0 / std::sqrt((double)D)), requests, (int)T, (int)HQ, (int)HKV, (int)D, act,
      bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_of(q)));
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "pla.decode.paged._C for MI355X: block tables, head norms with rotation and paged attention over libpla_gfx950.so";
  m.def("paged_kv_plan", &paged_kv_plan);
  m.def("fused_qk_norm_rope", &fused_qk_norm_rope);
  m.def("paged_attention_decode", &paged_attention_decode);
  m.def("packed_attention_fwd", &packed_attention_fwd);
  m.def("paged_attention_prefill", &paged_attention_prefill);
}
