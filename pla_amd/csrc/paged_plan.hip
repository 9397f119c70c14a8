// Block tables and slot maps of a serving step from the requests' lengths, without any value leaving the device, so that a
// step can be captured in a graph.  For entry n of the batch, with c = context[n] tokens cached, q = query[n] new ones, its
// row r = mapping[n] (or n) of the block table, h = held[r] blocks of that row in use and w = ceil((c + q) / block_size):
//
//   sound     0 <= c, 0 <= q, w <= columns, r inside the table and no earlier entry's row, its token rows within the capacity.
//   returned  the blocks [w, h) of sound entries go back on the free stack, in the order of the batch, then of the row.
//   taken     after that w - h blocks come off the stack, in the same order; an entry gets them if the running sum of what
//             was asked for, its own included, is on the stack (what a refused entry asked for counts), and none otherwise.
//   results   offsets (running sum of the q of entries with 0 <= q <= capacity, at most the capacity), sequence lengths c + q
//             (0: unsound or refused, such an entry keeps its blocks), and for every token row its position and slot
//             block * block_size + position % block_size (0 and -1 for rows of refused entries and behind the batch).
//
// Bound by latency: lengths, held counts, stack and table are four dependent trips to memory, the scans between them run in
// one workgroup, an entry per thread.  Everything whose number depends on the values (blocks moved, token rows) is dealt out
// flat: thread i finds its entry by bisection of the running sums in LDS, so that one long prompt costs no more than many
// short ones.  Steps of many token rows leave these to a second launch over the whole chip.

#include "decode_common.h"

namespace pla {

constexpr int PAGED_PLAN_THREADS = 1024;
// Token rows up to which the workgroup that makes the plan writes them as well.
constexpr int PAGED_PLAN_INLINE_ROWS = 4096;
constexpr int PAGED_PLAN_MAPPED_ROWS = 8192;      // rows whose first entry is looked up in LDS: 32 KB
constexpr int32_t PAGED_SATURATED = INT32_MAX;    // of running sums: more than any capacity

struct PagedPlan {
  const void* context; const void* query; const void* mapping;
  int context_wide, query_wide, mapping_wide;
  int32_t* table; int64_t table_stride; int rows, cols;
  int32_t* held; int32_t* stack; int32_t* height; int stack_size;
  int batch, block, capacity;
  int32_t* offsets; int32_t* seq_lens; int32_t* positions; int64_t* slots;

  __device__ int64_t at(const void* base, int wide, int64_t i) const {
    return wide ? static_cast<const int64_t*>(base)[i] : (int64_t) static_cast<const int32_t*>(base)[i];
  }
  __device__ int64_t row_of(int n) const { return mapping ? at(mapping, mapping_wide, n) : (int64_t)n; }
};

__device__ __forceinline__ int add_saturated(int a, int b) {      // of numbers that are not negative
  return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)PAGED_SATURATED);
}

// Running sum over the workgroup's threads, own value included; `total` gets the sum of all.  Sums saturate, which keeps
// them monotone.  `scratch`: one word a wavefront, free again after the caller's next barrier.
__device__ __forceinline__ int running_sum(int x, int* scratch, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int below = __shfl_up(x, d);
    if (lane >= d) x = add_saturated(x, below);
  }
  if (lane == 63) scratch[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < PAGED_PLAN_THREADS / 64; ++w) {
    const int s = scratch[w];
    if (w < wave) before = add_saturated(before, s);
    total = add_saturated(total, s);
  }
  return add_saturated(before, x);
}

// The entry whose share of a running sum holds item i: the first of `ends` above i (there is one).
__device__ __forceinline__ int entry_of(const int* ends, int n, int i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > i) hi = mid; else lo = mid + 1;
  }
  return lo;
}

struct PagedEntry {
  int64_t row, context;
  int query;              // token rows it stands for: its q, or 0 where q is no count
  int end;                // running sum of these
  int held, want;         // equal unless the entry is sound
  bool sound;
};

// Entry `n` (of one thread each; n >= batch: nothing).  `carry`: token rows of the chunks before.
__device__ __forceinline__ PagedEntry load_entry(const PagedPlan& p, const int* owner, int n, int& carry, int* scratch) {
  PagedEntry e{0, 0, 0, 0, 0, 0, false};
  int64_t query = -1;
  bool inside = false;
  if (n < p.batch) {
    e.context = p.at(p.context, p.context_wide, n);
    query = p.at(p.query, p.query_wide, n);
    e.row = p.row_of(n);
    inside = e.row >= 0 && e.row < p.rows;
    if (inside) e.held = min(max(p.held[e.row], 0), p.cols);
  }
  const bool counted = query >= 0 && query <= p.capacity;
  e.query = counted ? (int)query : 0;
  int total;
  e.end = add_saturated(carry, running_sum(e.query, scratch, total));
  carry = add_saturated(carry, total);
  e.want = e.held;
  if (inside && counted && e.context >= 0 && e.context <= (int64_t)p.cols * p.block && e.end <= p.capacity &&
      (owner == nullptr || owner[e.row] == n)) {
    const int64_t want = (e.context + query + p.block - 1) / p.block;
    e.sound = want <= p.cols;
    if (e.sound) e.want = (int)want;
  }
  return e;
}

// Position and slot of token row t: the plan's results so far say all that is needed.
__device__ __forceinline__ void write_token_row(const PagedPlan& p, int t, int n, int begin, int length, int end) {
  // length: of the entry's sequence, 0 if it was refused; its token rows are [begin, end)
  const bool live = t < end && length > 0;
  const int position = live ? length - (end - begin) + (t - begin) : 0;
  int64_t slot = -1;
  if (live) {
    const int page = position / p.block;
    slot = (int64_t)p.table[p.row_of(n) * p.table_stride + page] * p.block + (position - page * p.block);
  }
  p.positions[t] = position;
  p.slots[t] = slot;
}

template <bool TOKEN_ROWS>
__global__ __launch_bounds__(PAGED_PLAN_THREADS) void paged_plan_kernel(const PagedPlan p) {
  extern __shared__ int32_t owner_lds[];
  __shared__ int ends[2][PAGED_PLAN_THREADS];        // of blocks returned or taken | of token rows
  __shared__ int first[PAGED_PLAN_THREADS];          // page of an entry's first block that moves
  __shared__ int64_t line[PAGED_PLAN_THREADS];       // its row's start in the table
  __shared__ int length[PAGED_PLAN_THREADS];
  __shared__ int scratch[3][PAGED_PLAN_THREADS / 64];
  const int tid = threadIdx.x, chunks = (p.batch + PAGED_PLAN_THREADS - 1) / PAGED_PLAN_THREADS;
  const int* owner = nullptr;
  if (p.mapping) {
    // the first entry of a row is the row's
    for (int r = tid; r < p.rows; r += PAGED_PLAN_THREADS) owner_lds[r] = INT32_MAX;
    __syncthreads();
    for (int n = tid; n < p.batch; n += PAGED_PLAN_THREADS) {
      const int64_t row = p.row_of(n);
      if (row >= 0 && row < p.rows) atomicMin(&owner_lds[row], n);
    }
    __syncthreads();
    owner = owner_lds;
  }

  int height = min(max(*p.height, 0), p.stack_size), carry = 0;
  PagedEntry e{};
  for (int c = 0; c < chunks; ++c) {                 // blocks that go back
    const int base = c * PAGED_PLAN_THREADS, count = min(p.batch - base, PAGED_PLAN_THREADS);
    e = load_entry(p, owner, base + tid, carry, scratch[0]);
    int total;
    ends[0][tid] = running_sum(max(e.held - e.want, 0), scratch[1], total);
    first[tid] = e.want;
    line[tid] = e.row * p.table_stride;
    __syncthreads();
    for (int i = tid; i < total; i += PAGED_PLAN_THREADS) {
      const int n = entry_of(ends[0], count, i), before = n ? ends[0][n - 1] : 0;
      if (i < p.stack_size - height) p.stack[height + i] = p.table[line[n] + first[n] + (i - before)];
    }
    height = (int)min((int64_t)height + total, (int64_t)p.stack_size);
    __syncthreads();
  }

  carry = 0;
  int asked = 0, taken = 0;
  for (int c = 0; c < chunks; ++c) {                 // blocks that are taken, and the results
    const int base = c * PAGED_PLAN_THREADS, count = min(p.batch - base, PAGED_PLAN_THREADS), n = base + tid;
    if (chunks > 1) e = load_entry(p, owner, n, carry, scratch[0]);
    const int need = max(e.want - e.held, 0);
    int total, granted_total;
    const int sum = add_saturated(asked, running_sum(need, scratch[1], total));
    asked = add_saturated(asked, total);
    const bool granted = e.sound && (need == 0 || sum <= height);
    ends[0][tid] = running_sum(granted ? need : 0, scratch[2], granted_total);
    ends[1][tid] = e.end;
    first[tid] = e.held;
    line[tid] = e.row * p.table_stride;
    length[tid] = granted ? (int)(e.context + e.query) : 0;
    if (n < p.batch) {
      p.offsets[n + 1] = min(e.end, p.capacity);
      p.seq_lens[n] = length[tid];
      if (granted) p.held[e.row] = e.want;
    }
    if (n == 0) p.offsets[0] = 0;
    __syncthreads();
    for (int i = tid; i < granted_total; i += PAGED_PLAN_THREADS) {
      const int m = entry_of(ends[0], count, i), before = m ? ends[0][m - 1] : 0;
      p.table[line[m] + first[m] + (i - before)] = p.stack[height - 1 - (taken + i)];
    }
    taken += granted_total;
    __syncthreads();
    if (TOKEN_ROWS) {
      const int begin = base ? p.offsets[base] : 0, end = min(ends[1][count - 1], p.capacity);
      for (int t = begin + tid; t < end; t += PAGED_PLAN_THREADS) {
        const int m = entry_of(ends[1], count, t);
        write_token_row(p, t, base + m, m ? ends[1][m - 1] : begin, length[m], ends[1][m]);
      }
      __syncthreads();
    }
  }
  if (tid == 0) {
    *p.height = height - taken;
    if (p.batch == 0) p.offsets[0] = 0;
  }
  if (TOKEN_ROWS) {
    const int used = p.batch ? p.offsets[p.batch] : 0;
    for (int t = used + tid; t < p.capacity; t += PAGED_PLAN_THREADS) {
      p.positions[t] = 0;
      p.slots[t] = -1;
    }
  }
}

// Token rows of a step that has many: one a thread.
__global__ __launch_bounds__(256) void paged_token_rows_kernel(const PagedPlan p) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= p.capacity) return;
  int n = 0, begin = 0, end = 0, length = 0;
  if (p.batch > 0 && t < p.offsets[p.batch]) {
    n = entry_of(p.offsets + 1, p.batch, t);
    begin = p.offsets[n];
    end = p.offsets[n + 1];
    length = p.seq_lens[n];
  }
  write_token_row(p, t, n, begin, length, end);
}

}  // namespace pla

extern "C" int pla_paged_kv_plan_launch(
    const void* context, int context_wide, const void* query, int query_wide, const void* mapping, int mapping_wide,
    int32_t* block_table, int64_t table_row_stride, int table_rows, int table_cols, int32_t* held_blocks,
    int32_t* free_blocks, int32_t* free_count, int free_capacity, int batch, int block_size, int token_capacity,
    int32_t* offsets, int32_t* seq_lens, int32_t* positions, int64_t* slots, void* stream) {
  using namespace pla;
  PLA_REQUIRE(batch >= 0 && token_capacity >= 0 && token_capacity <= (1 << 30), "batch and token_capacity must be between 0 and 2^30");
  PLA_REQUIRE(table_rows >= 0 && table_cols >= 0 && table_row_stride >= table_cols, "invalid block table dimensions");
  PLA_REQUIRE(block_size > 0 && (int64_t)table_cols * block_size <= INT32_MAX, "block_size must be positive and a row's positions must fit 32 bits");
  PLA_REQUIRE(free_capacity >= 0 && free_capacity <= (1 << 30), "invalid free stack size");
  PLA_REQUIRE(mapping != nullptr || batch <= table_rows, "more batch entries than rows of the block table");
  PLA_REQUIRE(mapping == nullptr || table_rows <= PAGED_PLAN_MAPPED_ROWS, "request_indices take at most %d rows", PAGED_PLAN_MAPPED_ROWS);
  PLA_REQUIRE(free_count && offsets, "null tensor pointer");
  PLA_REQUIRE(batch == 0 || (context && query && seq_lens), "null tensor pointer");
  PLA_REQUIRE(table_rows == 0 || (held_blocks && (block_table || table_cols == 0)), "null tensor pointer");
  PLA_REQUIRE(free_capacity == 0 || free_blocks, "null tensor pointer");
  PLA_REQUIRE(token_capacity == 0 || (positions && slots), "null tensor pointer");
  const PagedPlan p{context, query, mapping, context_wide, query_wide, mapping_wide, block_table, table_row_stride, table_rows,
                    table_cols, held_blocks, free_blocks, free_count, free_capacity, batch, block_size, token_capacity,
                    offsets, seq_lens, positions, slots};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const size_t lds = mapping ? (size_t)table_rows * sizeof(int32_t) : 0;
  if (token_capacity <= PAGED_PLAN_INLINE_ROWS) {
    paged_plan_kernel<true><<<1, PAGED_PLAN_THREADS, lds, s>>>(p);
  } else {
    paged_plan_kernel<false><<<1, PAGED_PLAN_THREADS, lds, s>>>(p);
    paged_token_rows_kernel<<<(token_capacity + 255) / 256, 256, 0, s>>>(p);
  }
  return check_launch("paged_plan_kernel");
}
