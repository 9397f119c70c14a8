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
// Bound by latency in small steps: lengths and rows, held counts, then table and stack are dependent trips to memory, the two scans
// between them run in one workgroup, up to four entries a thread.  Large ones are bound by that workgroup's rate: it moves a thousand
// blocks in 0.8 to 0.9 us, 4 of the 15 us of a plan of 1500 entries that returns or takes 4600.  Everything whose number depends on
// the values (blocks moved, token rows) is dealt out flat: thread i finds its entry by bisection of the running sums in LDS, so that
// one long prompt costs no more than many short ones.  Token rows take a new block's number from the stack and do not wait for the
// table; steps of many token rows leave these to a second launch over the whole chip.

#include "decode_common.h"

namespace pla {

// Token rows up to which the workgroup that makes the plan writes them as well: a step of 1000 requests takes 8.8 us on the device
// with 2000 rows by one launch and 9.5 by two, with 4000 rows 10.9 and 9.4; one of 40 requests with 1920 rows 7.5 and 8.7, with 4000
// rows 9.0 and 8.6.
constexpr int PAGED_PLAN_INLINE_ROWS = 2048;
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

// Running sums over the workgroup's entries, E a thread, own value included; returns the sum of all.  Sums saturate, which keeps
// them monotone.  `scratch`: one word a wavefront, free again after the caller's next barrier.
template <int THREADS, int E>
__device__ __forceinline__ int running_sums(int (&x)[E], int* scratch) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 1; i < E; ++i) x[i] = add_saturated(x[i - 1], x[i]);
  int sum = x[E - 1];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int below = __shfl_up(sum, d);
    if (lane >= d) sum = add_saturated(sum, below);
  }
  if (lane == 63) scratch[wave] = sum;
  const int below = __shfl_up(sum, 1);
  __syncthreads();
  int before = lane ? below : 0, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const int s = scratch[w];
    if (w < wave) before = add_saturated(before, s);
    total = add_saturated(total, s);
  }
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] = add_saturated(before, x[i]);
  return total;
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
  int64_t row, context, query;
  int end;                // running sum of the token rows
  int held, want;         // equal unless the entry is sound
  bool inside;            // its row is one of the table's
  bool sound;
};

// What memory has of a thread's entries n .. n + E - 1 (from the batch's end on: nothing).
template <int E>
__device__ __forceinline__ void fetch_entries(const PagedPlan& p, int n, PagedEntry (&e)[E]) {
#pragma unroll
  for (int i = 0; i < E; ++i) {
    e[i] = PagedEntry{0, 0, -1, 0, 0, 0, false, false};
    if (n + i < p.batch) {
      e[i].row = p.row_of(n + i);
      e[i].context = p.at(p.context, p.context_wide, n + i);
      e[i].query = p.at(p.query, p.query_wide, n + i);
    }
    e[i].inside = n + i < p.batch && e[i].row >= 0 && e[i].row < p.rows;
  }
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (e[i].inside) e[i].held = p.held[e[i].row];
}

// What they ask for.  `carry`: token rows of the chunks before.
template <int THREADS, int E>
__device__ __forceinline__ void judge_entries(const PagedPlan& p, const int* owner, int n, int& carry, int* scratch, PagedEntry (&e)[E]) {
  bool counted[E];        // its q is a number of token rows
  int rows[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    counted[i] = e[i].query >= 0 && e[i].query <= p.capacity;
    rows[i] = counted[i] ? (int)e[i].query : 0;
  }
  const int total = running_sums<THREADS>(rows, scratch);
#pragma unroll
  for (int i = 0; i < E; ++i) {
    e[i].end = add_saturated(carry, rows[i]);
    e[i].held = min(max(e[i].held, 0), p.cols);
    e[i].want = e[i].held;
    if (e[i].inside && counted[i] && e[i].context >= 0 && e[i].context <= (int64_t)p.cols * p.block && e[i].end <= p.capacity &&
        (owner == nullptr || owner[e[i].row] == n + i)) {
      const int want = (int)(((uint32_t)e[i].context + (uint32_t)e[i].query + (uint32_t)p.block - 1) / (uint32_t)p.block);
      e[i].sound = want <= p.cols;
      if (e[i].sound) e[i].want = want;
    }
  }
  carry = add_saturated(carry, total);
}

// Position of token row t of an entry whose token rows are [begin, end), and whose sequence has `length` tokens (0: refused);
// -1: it has none.
__device__ __forceinline__ int position_of(int t, int begin, int end, int length) {
  return t < end && length > 0 ? length - (end - begin) + (t - begin) : -1;
}
__device__ __forceinline__ void write_token_row(const PagedPlan& p, int t, int position, int block) {
  p.positions[t] = max(position, 0);
  p.slots[t] = position < 0 ? -1 : (int64_t)block * p.block + position % p.block;
}

template <int THREADS, int E, bool TOKEN_ROWS>
__global__ __launch_bounds__(THREADS) void paged_plan_kernel(const PagedPlan p) {
  constexpr int CHUNK = THREADS * E;
  extern __shared__ int32_t owner_lds[];
  __shared__ int token_ends[CHUNK], back_ends[CHUNK], take_ends[CHUNK];   // running sums: token rows, blocks returned, blocks asked for
  __shared__ int first[CHUNK];                       // page of an entry's first block that moves, or its number of pages
  __shared__ int length[CHUNK], table_row[CHUNK];
  __shared__ int scratch[3][THREADS / 64], granted_end;
  const int tid = threadIdx.x, chunks = (p.batch + CHUNK - 1) / CHUNK;
  PagedEntry e[E];
  fetch_entries<E>(p, tid * E, e);
  int height = min(max(*p.height, 0), p.stack_size), carry = 0, asked_all = 0;
  const int* owner = nullptr;
  if (p.mapping) {
    // the first entry of a row is the row's
    for (int r = tid; r < p.rows; r += THREADS) owner_lds[r] = INT32_MAX;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (e[i].inside) atomicMin(&owner_lds[e[i].row], tid * E + i);
    for (int n = CHUNK + tid; n < p.batch; n += THREADS) {
      const int64_t row = p.row_of(n);
      if (row >= 0 && row < p.rows) atomicMin(&owner_lds[row], n);
    }
    __syncthreads();
    owner = owner_lds;
  }

  int take[E];
  // Running sums of a chunk; returns the blocks it gives back.
  auto load_chunk = [&](int base, int& asked) {
    if (chunks > 1) fetch_entries<E>(p, base + tid * E, e);
    judge_entries<THREADS, E>(p, owner, base + tid * E, carry, scratch[0], e);
    int back[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      back[i] = max(e[i].held - e[i].want, 0);
      take[i] = max(e[i].want - e[i].held, 0);
    }
    const int returned = running_sums<THREADS>(back, scratch[1]);
    asked = running_sums<THREADS>(take, scratch[2]);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      back_ends[tid * E + i] = back[i];
      take_ends[tid * E + i] = take[i];
      token_ends[tid * E + i] = e[i].end;
      first[tid * E + i] = min(e[i].held, e[i].want);
      table_row[tid * E + i] = (int)e[i].row;
    }
    if (tid == 0) granted_end = 0;
    __syncthreads();
    return returned;
  };
  int asked = 0;
  for (int c = 0; c < chunks; ++c) {                 // blocks that go back
    const int base = c * CHUNK, count = min(p.batch - base, CHUNK), returned = load_chunk(base, asked);
    for (int i = tid; i < min(returned, p.stack_size - height); i += THREADS) {
      const int m = entry_of(back_ends, count, i), before = m ? back_ends[m - 1] : 0;
      p.stack[height + i] = p.table[table_row[m] * p.table_stride + first[m] + (i - before)];
    }
    height = (int)min((int64_t)height + returned, (int64_t)p.stack_size);
    if (chunks > 1) __syncthreads();
  }

  carry = 0;
  int taken = 0, first_row = 0;                      // of the chunk's token rows
  for (int c = 0; c < chunks; ++c) {                 // blocks that are taken, and the results
    const int base = c * CHUNK, count = min(p.batch - base, CHUNK);
    if (chunks > 1) load_chunk(base, asked);
    // Who is granted blocks: those up to whose own the sum fits.  They come before all that are not, so the sum is also the place.
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int n = base + tid * E + i;
      const bool needs = e[i].want > e[i].held, granted = e[i].sound && (!needs || add_saturated(asked_all, take[i]) <= height);
      if (needs && granted) atomicMax(&granted_end, take[i]);
      const int tokens = granted ? (int)(e[i].context + e[i].query) : 0;
      length[tid * E + i] = tokens;
      if (n < p.batch) {
        p.offsets[n + 1] = min(e[i].end, p.capacity);
        p.seq_lens[n] = tokens;
        if (granted) p.held[e[i].row] = e[i].want;
      }
      if (n == 0) p.offsets[0] = 0;
    }
    __syncthreads();
    const int granted_total = granted_end;
    const int top = height - 1 - taken;              // of the stack, for this chunk's first block
    for (int i = tid; i < granted_total; i += THREADS) {
      const int block = p.stack[top - i], m = entry_of(take_ends, count, i), before = m ? take_ends[m - 1] : 0;
      p.table[table_row[m] * p.table_stride + first[m] + (i - before)] = block;
    }
    if (TOKEN_ROWS) {
      const int end = min(token_ends[count - 1], p.capacity);
      for (int t = first_row + tid; t < end; t += THREADS) {
        const int m = entry_of(token_ends, count, t), position = position_of(t, m ? token_ends[m - 1] : first_row, token_ends[m], length[m]);
        const int page = max(position, 0) / p.block;
        int block = 0;
        if (position >= 0)
          block = page < first[m] ? p.table[table_row[m] * p.table_stride + page]
                                  : p.stack[top - ((m ? take_ends[m - 1] : 0) + page - first[m])];
        write_token_row(p, t, position, block);
      }
      first_row = end;
    }
    taken += granted_total;
    asked_all = add_saturated(asked_all, asked);
    if (chunks > 1) __syncthreads();
  }
  if (tid == 0) {
    *p.height = height - taken;
    if (p.batch == 0) p.offsets[0] = 0;
  }
  if (TOKEN_ROWS)
    for (int t = first_row + tid; t < p.capacity; t += THREADS) write_token_row(p, t, -1, 0);
}

// Token rows of a step that has many: one a thread.  A wavefront looks for the entry of its first row with 64 probes at a time, two
// trips to memory for 4096 entries; those of the other rows are, but for runs of empty entries, among the next 64.
__global__ __launch_bounds__(256) void paged_token_rows_kernel(const PagedPlan p) {
  const int t = blockIdx.x * 256 + threadIdx.x, lane = threadIdx.x & 63, t0 = __builtin_amdgcn_readfirstlane(t);
  if (t0 >= p.capacity) return;
  const int32_t* ends = p.offsets + 1;
  const int total = p.batch > 0 ? p.offsets[p.batch] : 0;
  int position = -1, block = 0;
  if (t0 < total) {
    int from = 0;
    for (int span = p.batch; span > 64;) {
      const int step = (span + 63) / 64;
      const uint64_t above = __ballot(ends[from + min((lane + 1) * step, span) - 1] > t0);         // the last lane's is
      const int skip = (__ffsll((unsigned long long)above) - 1) * step;
      from += skip;
      span = min(step, span - skip);
    }
    const int end = ends[min(from + lane, p.batch - 1)];
    int below = 0;                          // of these 64 ends, those up to t
#pragma unroll
    for (int d = 32; d; d >>= 1) below += __shfl(end, below + d - 1) <= t ? d : 0;
    below += __shfl(end, below) <= t ? 1 : 0;
    if (t < total) {
      const int n = from + below + (below == 64 ? entry_of(ends + from + 64, p.batch - from - 64, t) : 0);
      position = position_of(t, p.offsets[n], ends[n], p.seq_lens[n]);
      if (position >= 0) block = p.table[p.row_of(n) * p.table_stride + position / p.block];
    }
  }
  if (t < p.capacity) write_token_row(p, t, position, block);
}

}  // namespace pla

extern "C" int pla_paged_kv_plan_launch(
    const void* context, int context_wide, const void* query, int query_wide, const void* mapping, int mapping_wide,
    int32_t* block_table, int64_t table_row_stride, int table_rows, int table_cols, int32_t* held_blocks,
    int32_t* free_blocks, int32_t* free_count, int free_capacity, int batch, int block_size, int token_capacity,
    int32_t* offsets, int32_t* seq_lens, int32_t* positions, int64_t* slots, void* stream) {
  using namespace pla;
  PLA_REQUIRE(batch >= 0 && batch <= (1 << 30) && token_capacity >= 0 && token_capacity <= (1 << 30), "batch and token_capacity must be between 0 and 2^30");
  PLA_REQUIRE(table_rows >= 0 && table_cols >= 0 && table_row_stride >= table_cols, "invalid block table dimensions");
  PLA_REQUIRE(block_size > 0 && block_size <= (1 << 30) && (int64_t)table_cols * block_size <= (1 << 30),
              "block_size must be positive and a row's positions at most 2^30");
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
  const bool rows_inline = token_capacity <= PAGED_PLAN_INLINE_ROWS;
  if (batch <= 256 && token_capacity <= 1024) paged_plan_kernel<256, 1, true><<<1, 256, lds, s>>>(p);
  else if (batch <= 1024 && rows_inline) paged_plan_kernel<1024, 1, true><<<1, 1024, lds, s>>>(p);
  else if (batch <= 1024) paged_plan_kernel<1024, 1, false><<<1, 1024, lds, s>>>(p);
  else if (rows_inline) paged_plan_kernel<1024, 4, true><<<1, 1024, lds, s>>>(p);
  else paged_plan_kernel<1024, 4, false><<<1, 1024, lds, s>>>(p);
  if (!rows_inline) paged_token_rows_kernel<<<(token_capacity + 255) / 256, 256, 0, s>>>(p);
  return check_launch("paged_plan_kernel");
}
