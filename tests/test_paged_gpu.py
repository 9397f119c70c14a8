"""Paged softmax attention next to the linear-attention layers: block tables from lengths, head norms with rotation and cache write,
attention over the cache - each against a plain implementation in 64 bits, then all of them together as a serving step runs them."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


# ---- block tables ------------------------------------------------------------------------------------------------

def _plan_reference(state, context, query, rows, capacity, bs):
    """The rules one entry after the other, on lists.  state: (table, held, free, count) - changed in place, count returned."""
    table, held, free, count = state
    R, cols, top = len(table), len(table[0]) if table else 0, len(free)
    count = min(max(count, 0), top)
    seen, entries, end = set(), [], 0
    for c, q, row in zip(context, query, rows):
        inside = 0 <= row < R
        counted = 0 <= q <= capacity
        end += q if counted else 0
        first = inside and row not in seen
        if inside:
            seen.add(row)
        h = min(max(held[row], 0), cols) if inside else 0
        want = -(-(c + q) // bs)
        sound = first and counted and c >= 0 and want <= cols and end <= capacity
        entries.append((c, q if counted else 0, row, h, want if sound else h, sound, end))
    for c, q, row, h, want, sound, _ in entries:
        for page in range(want, h):
            if count < top:
                free[count] = table[row][page]
                count += 1
    height, asked = count, 0
    offsets, seqs, positions, slots = [0], [], [], []
    for c, q, row, h, want, sound, end in entries:
        need = max(want - h, 0)
        asked += need
        granted = sound and (need == 0 or asked <= height)
        if granted:
            for page in range(h, want):
                count -= 1
                table[row][page] = free[count]
            held[row] = want
        for p in range(c, c + q):
            if len(slots) < capacity:
                positions.append(p if granted else 0)
                slots.append(table[row][p // bs] * bs + p % bs if granted else -1)
        offsets.append(min(end, capacity))
        seqs.append(c + q if granted else 0)
    spare = capacity - len(slots)
    return offsets, seqs, positions + [0] * spare, slots + [-1] * spare, count


def _check_plan(pool, lists, context, query, rows, capacity, index_dtype=torch.int32, out=None):
    from pla.decode.paged import paged_kv_plan
    mapping = None if rows is None else _ints(rows, index_dtype)
    plan = paged_kv_plan(pool, _ints(context, index_dtype), _ints(query, index_dtype), mapping, token_capacity=capacity, out=out)
    table, held, free, count = lists
    offsets, seqs, positions, slots, count = _plan_reference((table, held, free, count), context, query,
                                                             list(range(len(context))) if rows is None else rows, capacity, pool.block_size)
    assert plan.query_start_loc.tolist() == offsets
    assert plan.seq_lens.tolist() == seqs
    assert plan.positions.tolist() == positions
    assert plan.slot_mapping.tolist() == slots
    assert pool.free_count.item() == count
    assert pool.held_blocks.tolist() == held
    assert pool.free_blocks.tolist() == free
    assert pool.block_table.tolist() == table
    return plan, (table, held, free, count)


def _pool(num_blocks, bs, rows, cols):
    from pla.decode.paged import PagedKVBlocks
    pool = PagedKVBlocks.allocate(num_blocks, bs, rows, cols, DEV)
    return pool, (pool.block_table.tolist(), pool.held_blocks.tolist(), pool.free_blocks.tolist(), pool.free_count.item())


@pytest.mark.parametrize("batch, window, bs, mapped, index_dtype", [
    (1, 1, 16, False, torch.int32), (3, 8, 1, False, torch.int64), (64, 4, 16, True, torch.int32), (200, 8, 5, True, torch.int64),
    (1025, 3, 16, False, torch.int32), (2500, 2, 32, True, torch.int32), (9, 700, 16, False, torch.int32)])
def test_plan_over_steps_that_grow_roll_back_and_finish(batch, window, bs, mapped, index_dtype):
    """Chained steps: lengths grow, fall back and end, some steps with lengths, rows or capacities that are refused.  All integers
    equal those of the rules applied one entry after the other."""
    rng = random.Random(batch * 31 + window)
    rows = 2 * batch if mapped else batch
    cols = (60 + 3 * window) // bs + 2
    pool, lists = _pool(1 + int(batch * cols * 0.6) + 1, bs, rows, cols)
    context = [rng.randint(0, 40) for _ in range(batch)]
    for step in range(5):
        query = [rng.randint(0, window) for _ in range(batch)]
        index = rng.sample(range(rows), batch) if mapped and step == 0 else (index if mapped else None)
        used = index
        if step == 2:                                        # an overlong, a negative and a doubled entry, a row that is none
            query[0] = cols * bs + 1
            context[-1] = -1
            if mapped and batch > 3:
                used = list(index)
                used[2], used[3] = used[1], rows
        capacity = sum(q for q in query if 0 <= q) + rng.choice((0, 5))
        if step == 3:                                        # the last entries' rows do not fit
            capacity = max(0, capacity - window - 5)
        _, lists = _check_plan(pool, lists, context, query, used, capacity, index_dtype)
        context = [0 if rng.random() < 0.2 else max(0, min(cols * bs - window, (c if c >= 0 else 0) + rng.randint(-window, window)))
                   for c in context]


def test_plan_refuses_what_the_stack_does_not_hold_and_serves_the_others():
    pool, lists = _pool(6, 16, 4, 4)                         # five blocks
    _, lists = _check_plan(pool, lists, [0, 0, 0, 0], [33, 40, 16, 0], None, 100)      # 3, 3 (refused), 1 (asked for 7 by then), none
    assert pool.held_blocks.tolist() == [3, 0, 0, 0]
    # the first ends: its blocks serve the others in the same step
    _, lists = _check_plan(pool, lists, [0, 0, 0, 0], [0, 40, 16, 17], None, 100)
    assert pool.held_blocks.tolist() == [0, 3, 1, 0]


def test_plan_of_nothing_and_of_empty_steps():
    pool, lists = _pool(6, 16, 4, 4)
    _, lists = _check_plan(pool, lists, [], [], None, 3)
    _, lists = _check_plan(pool, lists, [], [], [], 0)
    _, lists = _check_plan(pool, lists, [0, 5], [0, 0], None, 0)
    _, lists = _check_plan(pool, lists, [0, 5], [0, 0], [3, 1], 2)
    assert lists[1] == [0, 1, 0, 0]                          # ceil(0 / 16) and ceil(5 / 16) blocks


def test_plan_takes_corrupt_counts_as_the_nearest_that_can_be():
    pool, lists = _pool(8, 16, 3, 2)
    for height, held in ((-5, [9, -2, 1]), (99, [0, 0, 0])):
        pool.free_count.fill_(height)
        pool.held_blocks.copy_(_ints(held))
        lists = (pool.block_table.tolist(), list(held), pool.free_blocks.tolist(), height)
        _check_plan(pool, lists, [5, 0, 20], [3, 4, 1], None, 16)
        lists = (pool.block_table.tolist(), pool.held_blocks.tolist(), pool.free_blocks.tolist(), pool.free_count.item())


def test_plan_writes_into_given_outputs_and_many_token_rows():
    from pla.decode.paged import PagedKVPlan
    pool, lists = _pool(900, 16, 5, 200)
    out = PagedKVPlan.allocate(5, 9000, DEV)
    plan, lists = _check_plan(pool, lists, [0, 100, 3, 0, 7], [3001, 0, 2500, 1, 1999], None, 9000, out=out)
    assert plan is out
    _check_plan(pool, lists, [3001, 90, 3, 0, 2006], [1, 8, 0, 0, 1], None, 4097)


@pytest.mark.parametrize("batch, mapped, capacity, blocks", [(9001, False, 4000, 14000), (9001, False, 13000, 11000), (5000, True, 12000, 12000),
                                                             (8192, True, 3000, 9000), (4097, False, 9000, 20000)])
def test_plan_of_more_entries_than_a_workgroup_holds_at_once(batch, mapped, capacity, blocks):
    """Several passes over the entries: sums, blocks and refusals (of a stack too small, of a capacity too small) go on over their ends."""
    rng = random.Random(batch + capacity)
    rows, cols, bs = 8192 if mapped else batch + 3, 5, 4
    pool, lists = _pool(blocks, bs, rows, cols)
    index = rng.sample(range(rows), batch) if mapped else None
    context = [rng.randint(0, 5) for _ in range(batch)]
    for step in range(3):
        query = [rng.choice((0, 0, 1, 1, 2, 3)) for _ in range(batch)]
        used = index
        if mapped and step == 1:                             # the same row in two passes, twice in one
            used = list(index)
            used[-1], used[-2], used[-3] = used[0], used[-4], rows
        _, lists = _check_plan(pool, lists, context, query, used, capacity)
        context = [rng.choice((0, max(0, c - 3), min(cols * bs - 3, c + q))) for c, q in zip(context, query)]


@pytest.mark.parametrize("batch", [1, 63, 64, 65, 700, 4096, 4200])
def test_token_rows_between_runs_of_empty_entries(batch):
    """More token rows than the planning workgroup writes: entries without any between long and short ones, at the ends and in runs
    of more than 64, rows without an entry behind them."""
    rng = random.Random(batch)
    cols, bs = 40, 16
    pool, lists = _pool(4000, bs, batch, cols)
    query = [0] * batch
    for n in rng.sample(range(batch), min(batch, 40)):
        query[n] = rng.choice((1, 2, 7, 64, 65, 300, 600))
    for step in range(2):
        _, lists = _check_plan(pool, lists, [rng.randint(0, 9) for _ in range(batch)], query, None, max(sum(query), 4097) + 70 * step)
        query = query[::-1] if step else [0] * (batch // 2) + [1] * (batch - batch // 2)


def test_plan_refuses_shared_memory():
    from pla.decode.paged import PagedKVPlan, paged_kv_plan
    pool, _ = _pool(9, 16, 3, 4)
    lens = _ints([1, 2, 3])
    for out in (PagedKVPlan(_ints([0] * 4), lens, _ints([0] * 8), _ints([0] * 8, torch.int64)),
                PagedKVPlan(_ints([0] * 4), pool.held_blocks, _ints([0] * 8), _ints([0] * 8, torch.int64))):
        with pytest.raises(RuntimeError, match="must not share memory"):
            paged_kv_plan(pool, lens, _ints([1, 1, 1]), token_capacity=8, out=out)


# ---- norms, rotation, cache write --------------------------------------------------------------------------------

def _rope_reference(x, weight, positions, inv_freq, *, eps, offset, factor, interleaved):
    """(result, size of the error that 32-bit arithmetic may have) in 64 bits.

    Roundings of the 32-bit form, each at most 2^-24 relative: squares and their tree of sums (D / 8 - 1 in a lane, up to 5 across;
    the root halves them), root, division, two products with the weight, sine and cosine (2 steps each and the angle's last bit),
    two products and a sum: below 16 in all, or 2^-20 of the pair's size."""
    y = x.double().cpu()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * (weight.double().cpu() + offset)
    size = y.abs()
    if inv_freq is not None:
        half = inv_freq.numel()
        angle = positions.double().cpu()[:, None, None] * inv_freq.double().cpu()
        first = torch.arange(0, 2 * half, 2) if interleaved else torch.arange(half)
        second = first + (1 if interleaved else half)
        a, b = y[..., first].clone(), y[..., second].clone()
        y[..., first] = (a * angle.cos() - b * angle.sin()) * factor
        y[..., second] = (b * angle.cos() + a * angle.sin()) * factor
        size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(factor)
    return y, size * 2.0 ** -20


def _close(got, ref, slack, what):
    """One rounding to got's type of a value that is off by at most ``slack``; subnormals step by a fixed size."""
    got, info = got.double().cpu(), torch.finfo(got.dtype)
    bound = (ref.abs() + slack) * (info.eps / 2) + slack + info.tiny * info.eps / 2
    worst = ((got - ref).abs() / bound).max().item() if got.numel() else 0.0
    assert worst <= 1.0 or math.isnan(worst) is False and (got == ref).all(), (what, worst)


def _rope_case(seed, T, HQ, HKV, D, act, *, gated=False, far=1 << 20):
    g = torch.Generator().manual_seed(seed)
    dtype = DTYPES[act]
    width = 2 * D if gated else D
    row = _randn(g, T, HQ * width + 2 * HKV * D + 8, dtype=dtype)
    q = row[:, :HQ * width].view(T, HQ, width)[..., :D]
    k = row[:, HQ * width:HQ * width + HKV * D].view(T, HKV, D)
    v = row[:, HQ * width + HKV * D:HQ * width + 2 * HKV * D].view(T, HKV, D)
    positions = torch.randint(0, far, (T,), generator=g).to(torch.int32).to(DEV)
    return g, row, q, k, v, positions


@pytest.mark.parametrize("T, HQ, HKV, D, rot, interleaved, norm, act, f32_weights", [
    (1, 1, 1, 64, 64, False, True, "bf16", False), (3, 5, 1, 64, 16, True, True, "fp16", False), (7, 16, 2, 128, 128, False, True, "bf16", True),
    (65, 32, 8, 128, 96, False, False, "fp16", False), (2, 40, 40, 128, 128, True, True, "bf16", False), (33, 16, 2, 256, 64, False, True, "bf16", True),
    (5, 8, 8, 256, 256, True, False, "fp16", False), (9, 3, 3, 256, 0, False, True, "bf16", False), (300, 16, 2, 256, 256, False, True, "fp16", False),
    (500, 64, 1, 64, 32, False, True, "bf16", False), (1200, 33, 7, 128, 64, True, True, "fp16", True), (0, 4, 2, 128, 128, False, True, "bf16", False)])
def test_norm_rotation_and_store(T, HQ, HKV, D, rot, interleaved, norm, act, f32_weights):
    from pla.decode.paged import fused_qk_norm_rope
    g, row, q, k, v, positions = _rope_case(T + D, T, HQ, HKV, D, act, gated=HQ == 16)
    dtype, before = DTYPES[act], row.clone()
    wtype = torch.float32 if f32_weights else dtype
    q_weight, k_weight = (_randn(g, D, dtype=wtype, scale=0.2) if norm else None for _ in range(2))
    inv_freq = (10000.0 ** -(torch.arange(0, rot, 2).double() / rot)).float().to(DEV) if rot else None
    how = dict(eps=1e-5, offset=1.0, factor=1.25, interleaved=interleaved)
    blocks, bs = -(-T // 16) + 2, 16
    caches = [torch.full((blocks, bs, HKV, D), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    slots = torch.randperm(blocks * bs, generator=g)[:T]
    slots[T // 2:T // 2 + 2] = torch.tensor([-1, blocks * bs])[:max(0, min(2, T - T // 2))]      # stored nowhere
    slots = slots.to(DEV)
    k_out = torch.zeros(T, HKV, D, dtype=dtype, device=DEV)
    q_out, same = fused_qk_norm_rope(q, k, positions if rot else None, q_weight=q_weight, k_weight=k_weight, eps=1e-5, weight_offset=1.0,
                                     inv_freq=inv_freq, attention_factor=1.25, interleaved=interleaved, k_out=k_out, v=v,
                                     k_cache=caches[0], v_cache=caches[1], slot_mapping=slots)
    assert same is k_out or same.data_ptr() == k_out.data_ptr()
    assert torch.equal(row, before)
    ref_q, slack_q = _rope_reference(q, q_weight, positions, inv_freq, **how)
    ref_k, slack_k = _rope_reference(k, k_weight, positions, inv_freq, **how)
    _close(q_out, ref_q, slack_q, "q")
    _close(k_out, ref_k, slack_k, "k")
    flat = [c.view(-1, HKV, D) for c in caches]
    kept = (slots >= 0) & (slots < blocks * bs)
    assert torch.equal(flat[0][slots[kept]], k_out[kept]) and torch.equal(flat[1][slots[kept]], v[kept])
    rest = torch.ones(blocks * bs, dtype=torch.bool, device=DEV)
    rest[slots[kept]] = False
    assert (flat[0][rest] == 7).all() and (flat[1][rest] == 7).all()
    if rot < D and not norm:
        assert torch.equal(q_out[..., rot:], q[..., rot:])


def test_angles_of_far_and_negative_positions():
    """At position 2^30 an angle in 32 bits would be off by whole turns."""
    from pla.decode.paged import fused_qk_norm_rope
    D = 128
    g, _, q, k, _, _ = _rope_case(5, 6, 2, 2, D, "fp16")
    positions = torch.tensor([0, 1, 2 ** 30 + 7, 2 ** 31 - 1, -5, -2 ** 31], dtype=torch.int64, device=DEV)
    inv_freq = (10000.0 ** -(torch.arange(0, D, 2).double() / D)).float().to(DEV)
    q_out, k_out = fused_qk_norm_rope(q, k, positions, inv_freq=inv_freq)
    # the 64-bit product rounds at 2^-53 of up to 2^31 radians, twice: 2^-21 of a radian on either side
    for got, x in ((q_out, q), (k_out, k)):
        ref, slack = _rope_reference(x, None, positions, inv_freq, eps=0, offset=0, factor=1.0, interleaved=False)
        _close(got, ref, slack * 3, "far")
    assert torch.equal(q_out[0], q[0])                       # position 0 turns nothing


def test_in_place_and_other_layouts():
    from pla.decode.paged import fused_qk_norm_rope
    D, T, HQ, HKV = 128, 37, 6, 2
    g, row, q, k, v, positions = _rope_case(9, T, HQ, HKV, D, "bf16")
    inv_freq = (10000.0 ** -(torch.arange(0, D, 2).double() / D)).float().to(DEV)
    weight = _randn(g, D, dtype=torch.bfloat16)
    args = dict(q_weight=weight, k_weight=weight, inv_freq=inv_freq)
    expect_q, expect_k = fused_qk_norm_rope(q, k, positions, **args)
    v_before = v.clone()
    # heads first in the cache, K and V of a block in one page
    pages = torch.zeros(4, 2, HKV, 16, D, dtype=torch.bfloat16, device=DEV)
    slots = torch.arange(T, device=DEV, dtype=torch.int32) + 3
    got_q, got_k = fused_qk_norm_rope(q, k, positions, **args, q_out=q, k_out=k, v=v, k_cache=pages[:, 0].transpose(1, 2),
                                      v_cache=pages[:, 1].transpose(1, 2), slot_mapping=slots)
    assert got_q.data_ptr() == q.data_ptr() and torch.equal(q, expect_q) and torch.equal(k, expect_k) and torch.equal(v, v_before)
    assert torch.equal(pages[:, 0].transpose(1, 2).reshape(-1, HKV, D)[3:3 + T], expect_k)
    assert torch.equal(pages[:, 1].transpose(1, 2).reshape(-1, HKV, D)[3:3 + T], v)
    # strided positions, heads first in q, keys without values, slots past 32 bits' sign
    q2, k2 = _randn(g, HQ, T, D, dtype=torch.bfloat16).transpose(0, 1), _randn(g, T, HKV, D, dtype=torch.bfloat16)
    spread = torch.stack([positions, positions + 1], 1)[:, 0]
    a, none = fused_qk_norm_rope(q2, k2, spread, **args, k_cache=pages[:, 0].transpose(1, 2), slot_mapping=slots.long())
    b, c = fused_qk_norm_rope(q2.contiguous(), k2, positions, **args)
    assert none is None and torch.equal(a, b) and torch.equal(pages[:, 0].transpose(1, 2).reshape(-1, HKV, D)[3:3 + T], c)


def test_values_that_are_not_finite_stay_in_their_heads():
    from pla.decode.paged import fused_qk_norm_rope
    D = 64
    g, _, q, k, _, positions = _rope_case(3, 4, 3, 1, D, "fp16")
    q = q.clone()
    inv_freq = (100.0 ** -(torch.arange(0, 32, 2).double() / 32)).float().to(DEV)
    clean, _ = fused_qk_norm_rope(q, k, positions, inv_freq=inv_freq)
    q[1, 2, 40] = math.inf                                   # a channel that passes
    q[2, 0, 3] = math.nan                                    # one of the pair (3, 19)
    got, _ = fused_qk_norm_rope(q, k, positions, inv_freq=inv_freq)
    assert got[1, 2, 40] == math.inf and got[2, 0, 3].isnan() and got[2, 0, 19].isnan()
    clean[1, 2, 40] = got[1, 2, 40]
    clean[2, 0, 3] = clean[2, 0, 19] = 0
    got[2, 0, 3] = got[2, 0, 19] = 0
    assert torch.equal(got, clean)


def test_norm_refuses_shared_memory():
    from pla.decode.paged import fused_qk_norm_rope
    x = torch.zeros(8, 4, 64, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(8, 4, 64, dtype=torch.bfloat16, device=DEV)
    buffer = torch.zeros(9, 4, 64, dtype=torch.bfloat16, device=DEV)
    for args in (dict(q=buffer[:8], k=k, q_out=buffer[1:]), dict(q=x, k=k, q_out=k), dict(q=x, k=k, q_out=x, k_out=x),
                 dict(q=x, k=k, k_out=torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV).expand(8, 4, 64))):
        with pytest.raises(RuntimeError, match="share memory|more than one element"):
            fused_qk_norm_rope(**args)


def test_written_tensors_that_overlap_themselves_are_refused():
    """Rows or blocks a step apart that is smaller than they are: two workgroups would write one place."""
    from pla.decode.paged import fused_qk_norm_rope, paged_attention_decode
    x = torch.zeros(8, 4, 64, dtype=torch.bfloat16, device=DEV)
    store = torch.zeros(4096, dtype=torch.bfloat16, device=DEV)
    rows, slots = store.as_strided((8, 4, 64), (128, 64, 1)), torch.arange(8, device=DEV)
    cache = torch.zeros(2, 16, 4, 64, dtype=torch.bfloat16, device=DEV)
    close = torch.zeros(8192, dtype=torch.bfloat16, device=DEV).as_strided((2, 16, 4, 64), (2048, 256, 64, 1))
    for args in (dict(q_out=rows), dict(k_out=rows), dict(k_cache=close, slot_mapping=slots),
                 dict(k_cache=cache, v_cache=close, v=x, slot_mapping=slots)):
        with pytest.raises(RuntimeError, match="must not share memory with itself"):
            fused_qk_norm_rope(x, x, **args)
    with pytest.raises(RuntimeError, match="must not share memory with itself"):
        paged_attention_decode(x, cache, cache, _ints([[0]] * 8), _ints([1] * 8), out=rows)
    # read only: a cache whose blocks lie half on each other is what it is
    got = paged_attention_decode(x, close, close, _ints([[0]] * 8), _ints([1] * 8))
    assert torch.equal(got, torch.zeros_like(got))
    # rows far enough apart in any order of the dimensions
    out = torch.zeros(64 * 4 * 9, dtype=torch.bfloat16, device=DEV).as_strided((8, 4, 64), (64, 64 * 9, 1))
    assert torch.equal(paged_attention_decode(x, cache, cache, _ints([[0]] * 8), _ints([1] * 8), out=out), got)


# ---- attention ---------------------------------------------------------------------------------------------------

class _Cache:
    """A paged cache whose every place outside of the sequences holds ``junk``."""

    def __init__(self, lengths, HKV, D, bs, act, *, seed=0, heads_first=False, rows=None, junk=math.nan, spare=2):
        g = torch.Generator().manual_seed(seed)
        dtype = DTYPES[act]
        pages = [-(-max(n, 0) // bs) for n in lengths]
        total = sum(pages) + spare
        order = torch.randperm(total, generator=g).tolist()
        cols = max(pages + [1]) + 1
        store = torch.full((total, 2, HKV, bs, D) if heads_first else (total, 2, bs, HKV, D), junk, dtype=dtype)
        self.rows = list(range(len(lengths))) if rows is None else rows
        table = torch.full((max(self.rows, default=0) + 1, cols), -7, dtype=torch.int32)
        self.k, self.v = [], []
        at = 0
        for row, n, count in zip(self.rows, lengths, pages):
            mine = order[at:at + count]
            at += count
            table[row, :count] = torch.tensor(mine, dtype=torch.int32)
            n = max(n, 0)
            k, v = (torch.randn(n, HKV, D, generator=g).to(dtype) for _ in range(2))
            self.k.append(k)
            self.v.append(v)
            for p, block in enumerate(mine):
                part = slice(p * bs, min(n, (p + 1) * bs))
                for i, x in enumerate((k, v)):
                    x = x[part]
                    if heads_first:
                        store[block, i, :, :x.size(0)] = x.transpose(0, 1)
                    else:
                        store[block, i, :x.size(0)] = x
        self.store, self.table = store.to(DEV), table.to(DEV)
        self.k_cache, self.v_cache = (self.store[:, i].transpose(1, 2) if heads_first else self.store[:, i] for i in range(2))


def _attention_reference(q, cache, lengths, windows, scale, gate=None, visible=None):
    """(outputs, size of the error that the kernel's arithmetic may have) in 64 bits.

    A weight w that is rounded by a relative u and summed as rounded moves a result by at most u sum w |v - o|, as the sum of what is
    added is zero; so does an error e of a score (2 e).  Scores: products are exact in 32 bits, their sum of D terms is off by at most
    D 2^-24 of the sum of the sizes, the factor and the exponential's argument by 2^-24 of the score each, its value by 2^-22.  Sums over
    n keys in 32 bits, regrouped a few times: at most (n + 16) 2^-24 sum w |v|; one division, one product with the gate.  Weights in
    fp16 below 2^-39 of the largest are dropped."""
    T, HQ, D = q.shape
    HKV = cache.k_cache.size(2)
    G, u = HQ // HKV, _half_step(q.dtype)
    out, slack = torch.zeros(T, HQ, D, dtype=torch.float64), torch.zeros(T, HQ, D, dtype=torch.float64)
    qd = q.double().cpu()
    token = 0
    for n, (length, window) in enumerate(zip(lengths, windows)):
        for j in range(window):
            sees = min(max(length - window + j + 1, 0), max(length, 0))
            keep = torch.arange(sees) if visible is None else torch.tensor([p for p in range(sees) if visible(n, p)], dtype=torch.long)
            if keep.numel():
                k, v = cache.k[n][keep].double().repeat_interleave(G, 1), cache.v[n][keep].double().repeat_interleave(G, 1)
                terms = qd[token][None] * k
                score = terms.sum(-1) * scale                                     # [keys, HQ]
                wrong = (terms.abs().sum(-1) * abs(scale) * D + 3 * score.abs()) * 2.0 ** -24 + 2.0 ** -22
                w = torch.softmax(score, 0)
                o = torch.einsum("nh,nhd->hd", w, v)
                spread = torch.einsum("nh,nhd->hd", w * (u * (1 + 2 * u) + 2 * wrong), (v - o).abs())
                size = torch.einsum("nh,nhd->hd", w, v.abs())
                out[token] = o
                slack[token] = spread + (keep.numel() + 16) * 2.0 ** -24 * size + keep.numel() * 2.0 ** -38 * v.abs().amax()
            token += 1
    if gate is not None:
        g = torch.sigmoid(gate.double().cpu())
        out, slack = out * g, slack * g + (out * g).abs() * 2.0 ** -20
    return out, slack


CROWD = 0                                                    # requests without a window behind those of a call


@pytest.fixture(params=[0, 160], ids=["together", "alone"])
def crowd(request, monkeypatch):
    """Calls of few runs, whose workgroups work together, and of many, whose wavefronts have runs of their own."""
    monkeypatch.setitem(globals(), "CROWD", request.param)


def _attend(cache, q, lengths, windows, *, max_query=None, index_dtype=torch.int32, gate=None, scale=None, rows=None, out=None, offsets=None):
    from pla.decode.paged import paged_attention_decode
    if offsets is None:
        offsets = [0]
        for w in windows:
            offsets.append(offsets[-1] + w)
    single = max_query is None and all(w == 1 for w in windows)
    max_query = 1 if single else max_query or max(windows)
    if CROWD:
        rows = (list(range(len(lengths))) if rows is None else list(rows)) + [0] * CROWD
        lengths, offsets, single = list(lengths) + [9] * CROWD, list(offsets) + [offsets[-1]] * CROWD, False
    return paged_attention_decode(q, cache.k_cache, cache.v_cache, cache.table, _ints(lengths, index_dtype),
                                  query_start_loc=None if single else _ints(offsets, index_dtype),
                                  request_indices=None if rows is None else _ints(rows, index_dtype),
                                  max_query_len=max_query, scale=scale, output_gate=gate, out=out)


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 130, 255, 257, 500]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("act", ["bf16", "fp16"])
@pytest.mark.parametrize("HQ, HKV, bs, heads_first, gated", [(1, 1, 16, False, False), (8, 2, 32, True, True), (7, 1, 48, False, False),
                                                             (16, 1, 528, False, True), (40, 2, 16, True, False)])
@pytest.mark.usefixtures("crowd")
def test_one_new_token_at_the_edges_of_pages_and_tiles(D, act, HQ, HKV, bs, heads_first, gated):
    cache = _Cache(EDGES, HKV, D, bs, act, seed=D + HQ, heads_first=heads_first)
    g = torch.Generator().manual_seed(HQ)
    q = _randn(g, len(EDGES), HQ, D, dtype=DTYPES[act], scale=2.0)
    gate = _randn(g, len(EDGES), HQ, D, dtype=DTYPES[act], scale=3.0) if gated else None
    out = _attend(cache, q, EDGES, [1] * len(EDGES), gate=gate)
    ref, slack = _attention_reference(q, cache, EDGES, [1] * len(EDGES), D ** -0.5, gate)
    _close(out, ref, slack, "attention")
    assert (out[0] == 0).all()                               # nothing to see


@pytest.mark.parametrize("D, act, HQ, HKV, max_query", [(64, "fp16", 4, 4, 8), (128, "bf16", 16, 2, 4), (128, "fp16", 6, 2, 32), (256, "bf16", 8, 1, 32),
                                                        (256, "fp16", 3, 1, 5), (64, "bf16", 16, 1, 17), (128, "bf16", 12, 1, 3)])
@pytest.mark.usefixtures("crowd")
def test_windows_of_draft_tokens(D, act, HQ, HKV, max_query):
    """Windows of every size against lengths that are shorter, equal, at a page's or a tile's edge; the longest split into pieces."""
    rng = random.Random(D + max_query)
    windows = [rng.randint(0, max_query) for _ in range(14)] + [max_query, 1, max_query]
    lengths = [0, 1, 2, max_query, 16, 17, 33, 127, 128, 129, 130, 140, 160, 200, 1300, 2000, 2049]
    cache = _Cache(lengths, HKV, D, 16, act, seed=max_query)
    g = torch.Generator().manual_seed(7)
    T = sum(windows)
    q = _randn(g, T + 3, HQ, D, dtype=DTYPES[act], scale=1.5)
    out = torch.full_like(q, 5.0)
    _attend(cache, q, lengths, windows, max_query=max_query, index_dtype=torch.int64, out=out)
    ref, slack = _attention_reference(q[:T], cache, lengths, windows, D ** -0.5)
    _close(out[:T], ref, slack, "window")
    assert (out[T:] == 5).all()                              # rows behind the last request


@pytest.mark.parametrize("D, act, HQ, HKV, bs", [(128, "bf16", 16, 2, 16), (64, "fp16", 2, 2, 64), (256, "bf16", 16, 1, 528)])
@pytest.mark.usefixtures("crowd")
def test_one_long_request_among_short_ones_is_split_and_joined(D, act, HQ, HKV, bs):
    lengths = [40000, 3, 700, 0, 129]
    cache = _Cache(lengths, HKV, D, bs, act, seed=1)
    g = torch.Generator().manual_seed(2)
    q = _randn(g, len(lengths), HQ, D, dtype=DTYPES[act], scale=2.0)
    gate = _randn(g, len(lengths), HQ, D, dtype=DTYPES[act])
    out = _attend(cache, q, lengths, [1] * 5, gate=gate)
    ref, slack = _attention_reference(q, cache, lengths, [1] * 5, D ** -0.5, gate)
    _close(out, ref, slack, "long")
    assert torch.equal(out, _attend(cache, q, lengths, [1] * 5, gate=gate))


def test_more_runs_than_workgroups():
    lengths = [(37 * i) % 300 for i in range(400)]
    cache = _Cache(lengths, 4, 64, 16, "bf16", seed=4)
    q = _randn(torch.Generator().manual_seed(3), 400, 8, 64, dtype=torch.bfloat16)
    out = _attend(cache, q, lengths, [1] * 400)
    ref, slack = _attention_reference(q, cache, lengths, [1] * 400, 64 ** -0.5)
    _close(out, ref, slack, "many")


@pytest.mark.usefixtures("crowd")
def test_peaked_and_flat_scores_and_other_scales():
    lengths = [1000, 1000, 1000]
    for act in ("bf16", "fp16"):
        cache = _Cache(lengths, 1, 128, 16, act, seed=6)
        g = torch.Generator().manual_seed(8)
        q = _randn(g, 3, 4, 128, dtype=DTYPES[act])
        for scale in (0.0, 1.0, -0.3, 4.0):
            out = _attend(cache, q, lengths, [1] * 3, scale=scale)
            ref, slack = _attention_reference(q, cache, lengths, [1] * 3, scale)
            _close(out, ref, slack, scale)


@pytest.mark.usefixtures("crowd")
def test_requests_that_are_passed_over_leave_their_rows():
    """Windows that are empty, longer than declared or not within q; rows of the block table by index, in any order."""
    lengths, rows = [50, 60, 70, 80, 20], [4, 0, 7, 2, 9]
    cache = _Cache(lengths, 2, 128, 16, "bf16", rows=rows)
    q = _randn(torch.Generator().manual_seed(1), 12, 4, 128, dtype=torch.bfloat16)
    out = torch.full_like(q, 3.0)
    _attend(cache, q, lengths, None, max_query=2, rows=rows, out=out, offsets=[0, 2, 2, 7, 9, 13])
    ref, slack = _attention_reference(q, cache, [50, 60, 70, 80], [2, 0, 5, 2], 128 ** -0.5)
    _close(out[:2], ref[:2], slack[:2], "first")
    _close(out[7:9], ref[7:9], slack[7:9], "fourth")
    assert (out[2:7] == 3).all() and (out[9:] == 3).all()
    out.fill_(3.0)
    _attend(cache, q, lengths, None, max_query=2, rows=rows, out=out, offsets=[2, 0, 2, -2, -1, 1])      # nothing of it makes sense but [0, 2) and one
    assert (out[2:] == 3).all()
    # rows of the table that are none: nothing to see
    out = _attend(cache, q[:5], lengths, [1] * 5, rows=[4, 10, 7, -1, 9])
    ref, slack = _attention_reference(q[:5], cache, lengths, [1] * 5, 128 ** -0.5, visible=lambda n, p: n not in (1, 3))
    _close(out, ref, slack, "rows")


@pytest.mark.usefixtures("crowd")
def test_positions_without_a_block_are_left_out():
    lengths = [300, 90, 40, 1000]
    cache = _Cache(lengths, 2, 64, 16, "fp16", seed=12)
    blocks = cache.k_cache.size(0)
    bad = {(0, 0): -1, (0, 5): blocks, (0, 18): 2 ** 31 - 1, (1, 3): -2 ** 31, (2, 0): blocks, (2, 1): -1, (2, 2): blocks + 5, (3, 40): -1}
    for (n, page), entry in bad.items():
        cache.table[n, page] = entry
    q = _randn(torch.Generator().manual_seed(13), 8, 4, 64, dtype=torch.float16)
    out = _attend(cache, q, lengths, [2, 2, 2, 2])
    ref, slack = _attention_reference(q, cache, lengths, [2] * 4, 64 ** -0.5, visible=lambda n, p: (n, p // 16) not in bad)
    _close(out, ref, slack, "left out")
    assert (out[4:6] == 0).all()
    # lengths past the table: what the table has counts
    cols = cache.table.size(1)
    long = [cols * 16 + 100]
    whole = _Cache([cols * 16], 2, 64, 16, "fp16", seed=14)
    whole.table = whole.table[:, :cols].contiguous()
    out = _attend(whole, q[:1], long, [1])
    ref, slack = _attention_reference(q[:1], whole, [cols * 16], [1], 64 ** -0.5)
    _close(out, ref, slack, "past the table")


@pytest.mark.parametrize("D, act, HQ, HKV, length", [(128, "bf16", 8, 2, 133), (64, "fp16", 4, 4, 640), (256, "bf16", 8, 1, 46), (128, "fp16", 16, 1, 5000)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.usefixtures("crowd")
def test_draft_tokens_that_are_not_finite_do_not_reach_the_ones_before(D, act, HQ, HKV, length, value):
    """The keys and values of draft token 5 of 8: tokens 0 to 4 do not see them and equal a call without them."""
    windows, lengths = [8, 8], [length, length + 3]
    cache = _Cache(lengths, HKV, D, 16, act, seed=21)
    q = _randn(torch.Generator().manual_seed(22), 16, HQ, D, dtype=DTYPES[act])
    clean = _attend(cache, q, lengths, windows)
    at = length - 8 + 5
    block, place = cache.table[0, at // 16].item(), at % 16
    cache.store[block, 1, place, 0, 3] = value               # one channel of a value
    got = _attend(cache, q, lengths, windows)
    G = HQ // HKV
    assert not got[5:8, :G, 3].isfinite().any()
    if not math.isnan(value):
        assert (got[5:8, :G, 3] == value).all()
    got[5:8, :G, 3] = clean[5:8, :G, 3]
    # the tokens that see it add these values at the end of the run: another order of sums, then one rounding
    assert torch.equal(got[8:], clean[8:]) and torch.equal(got[:, G:], clean[:, G:])
    ref, slack = _attention_reference(q, cache, lengths, windows, D ** -0.5)
    _close(got, ref, slack, "value")
    cache.store[block, 0, place, 0] = value                  # the whole key
    got = _attend(cache, q, lengths, windows)
    _close(got[:5], ref[:5], slack[:5], "key")
    assert not got[5:8, :G].isfinite().all(-1).any()
    _close(got[8:], ref[8:], slack[8:], "other request")


@pytest.mark.parametrize("places", [(4,), (13,), (4, 13), (1, 2, 14, 15)])
def test_values_set_aside_in_two_steps_of_one_wavefront(places):
    """Windows that lie in two groups of 32 keys, long requests enough that a wavefront has several groups of a run: values that are
    infinite in the first, the second or both reach the tokens that see them, and every other channel is as without them."""
    D, HKV = 256, 4
    lengths = [1000, 1064, 1032] + [1000 + 7 * i for i in range(27)]           # the windows from 985, 1049 and 1017 on
    windows = [16] * 3 + [1] * 27
    cache = _Cache(lengths, HKV, D, 16, "bf16", seed=71)
    q = _randn(torch.Generator().manual_seed(72), sum(windows), HKV, D, dtype=torch.bfloat16)
    ref, slack = _attention_reference(q, cache, lengths, windows, D ** -0.5)
    for n in range(3):
        for place in places:
            at = lengths[n] - 16 + place
            cache.store[cache.table[n, at // 16].item(), 1, at % 16, :, 5] = math.inf
    got = _attend(cache, q, lengths, windows)
    for n in range(3):
        rows = got[16 * n:16 * n + 16, :, 5]
        assert rows[:places[0]].isfinite().all() and (rows[places[0]:] == math.inf).all()
        rows[places[0]:] = ref[16 * n + places[0]:16 * n + 16, :, 5].to(rows)
    _close(got, ref, slack, "set aside")


@pytest.mark.parametrize("act, length", [("bf16", 70), ("fp16", 1500)])
@pytest.mark.usefixtures("crowd")
def test_values_set_aside_weigh_as_much_as_the_others(act, length):
    """Scores so far apart that the draft tokens' own keys carry most of the weight, with one value among them that is not finite:
    the rows that do not see it, and the other channels of those that do, are what they are without it."""
    D, windows, lengths = 128, [8], [length]
    cache = _Cache(lengths, 1, D, 16, act, seed=41)
    q = _randn(torch.Generator().manual_seed(42), 8, 4, D, dtype=DTYPES[act])
    k = cache.k[0]
    # every query is near the key of its own token
    for j in range(8):
        at = length - 8 + j
        k[at] = (q[j, 0].cpu().float() * 0.7).to(DTYPES[act])
        cache.store[cache.table[0, at // 16].item(), 0, at % 16, 0] = k[at, 0].to(DEV)
    cache.store[cache.table[0, (length - 2) // 16].item(), 1, (length - 2) % 16, 0, 9] = math.inf
    ref, slack = _attention_reference(q, cache, lengths, windows, 0.5)
    got = _attend(cache, q, lengths, windows, scale=0.5)
    assert (got[6:, :, 9] == math.inf).all()
    got[6:, :, 9] = ref[6:, :, 9].to(got)
    _close(got, ref, slack, "set aside")


def test_caches_side_by_side_in_one_buffer_and_strides_of_single_rows():
    """K and V of a token next to each other, one head with a stride of its own, one token whose stride means nothing."""
    from pla.decode.paged import fused_qk_norm_rope, paged_attention_decode
    D, bs = 64, 16
    g = torch.Generator().manual_seed(61)
    both = torch.zeros(4, bs, 1, 2 * D, dtype=torch.bfloat16, device=DEV)
    k_cache, v_cache = both[..., :D], both[..., D:]
    odd = torch.as_strided(both, (4, bs, 1, D), (bs * 2 * D, 2 * D, 3, 1))           # the head stride of one head
    row = _randn(g, 20, 3 * D, dtype=torch.bfloat16)
    q, k, v = (row[:, i * D:(i + 1) * D].view(20, 1, D) for i in range(3))
    slots = torch.arange(20, device=DEV) + bs
    table = _ints([[1, 2]])
    fused_qk_norm_rope(q, k, q_weight=_randn(g, D, dtype=torch.bfloat16), v=v, k_cache=k_cache, v_cache=v_cache, slot_mapping=slots, q_out=q)
    assert torch.equal(both.view(-1, 2 * D)[bs:bs + 20, :D], k[:, 0]) and torch.equal(both.view(-1, 2 * D)[bs:bs + 20, D:], v[:, 0])
    last = torch.as_strided(q, (1, 1, D), (5, 7, 1), q[19:].storage_offset())
    expect = paged_attention_decode(q[19:].contiguous(), k_cache.contiguous(), v_cache.contiguous(), table, _ints([20]))
    assert torch.equal(paged_attention_decode(last, odd, v_cache, table, _ints([20])), expect)
    with pytest.raises(RuntimeError, match="must not share memory"):
        fused_qk_norm_rope(q, k, v=v, k_cache=k_cache, v_cache=both[..., D // 2:D // 2 + D], slot_mapping=slots)


@pytest.mark.usefixtures("crowd")
def test_offsets_past_32_bits():
    """Blocks 2^32 bytes and more apart."""
    D, HKV, pitch = 128, 1, 2 ** 31 + 1024
    store = torch.empty(2 * pitch + 2 * 16 * D + pitch // 2, dtype=torch.bfloat16, device=DEV)
    k_cache = store.as_strided((3, 16, HKV, D), (pitch, D, D, 1))
    v_cache = store.as_strided((3, 16, HKV, D), (pitch, D, D, 1), pitch // 2 // 8 * 8)
    cache = _Cache([40], HKV, D, 16, "bf16", seed=3)
    for p in range(3):
        n = min(16, 40 - 16 * p)
        k_cache[2 - p, :n] = cache.k[0][16 * p:16 * p + n].to(DEV)
        v_cache[2 - p, :n] = cache.v[0][16 * p:16 * p + n].to(DEV)
    cache.k_cache, cache.v_cache, cache.table = k_cache, v_cache, _ints([[2, 1, 0]])
    q = _randn(torch.Generator().manual_seed(4), 1, 4, D, dtype=torch.bfloat16)
    out = _attend(cache, q, [40], [1])
    ref, slack = _attention_reference(q, cache, [40], [1], D ** -0.5)
    _close(out, ref, slack, "far apart")
    # and the write: the same places through slots
    from pla.decode.paged import fused_qk_norm_rope
    k, v = (_randn(torch.Generator().manual_seed(i), 2, HKV, D, dtype=torch.bfloat16) for i in (5, 6))
    fused_qk_norm_rope(q.expand(2, 4, D), k, v=v, k_cache=k_cache, v_cache=v_cache, slot_mapping=_ints([2 * 16 + 15, 0]))
    assert torch.equal(k_cache[2, 15], k[0]) and torch.equal(v_cache[2, 15], v[0]) and torch.equal(k_cache[0, 0], k[1])


@pytest.mark.usefixtures("crowd")
def test_strided_rows_of_q_gate_and_out():
    lengths = [100, 7, 300]
    cache = _Cache(lengths, 2, 128, 16, "bf16", seed=31)
    g = torch.Generator().manual_seed(32)
    mixed = _randn(g, 3, 4, 2 * 128 + 8, dtype=torch.bfloat16)
    q, gate = mixed[..., :128], mixed[..., 128:256]
    out = torch.zeros(4, 3, 128 + 16, dtype=torch.bfloat16, device=DEV).transpose(0, 1)[..., :128]
    got = _attend(cache, q, lengths, [1] * 3, gate=gate, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(out, _attend(cache, q.contiguous(), lengths, [1] * 3, gate=gate.contiguous()))


def test_attention_refuses_shared_memory():
    cache = _Cache([20], 1, 64, 16, "bf16")
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=DEV)
    for out in (q, cache.store.view(-1)[:64].view(1, 1, 64)):
        with pytest.raises(RuntimeError, match="must not share memory"):
            _attend(cache, q, [20], [1], out=out)


# ---- together ----------------------------------------------------------------------------------------------------

class _Serving:
    """One softmax-attention layer of a serving program over a paged cache, beside a plain copy of every request's keys and values."""

    def __init__(self, D=128, HQ=8, HKV=2, act="bf16", reqs=6, capacity=48, max_query=8, bs=16):
        from pla.decode.paged import PagedKVBlocks, PagedKVPlan, rotary_frequencies
        g = torch.Generator().manual_seed(77)
        self.D, self.HQ, self.HKV, self.dtype, self.capacity, self.max_query, self.bs, self.g = D, HQ, HKV, DTYPES[act], capacity, max_query, bs, g
        self.pool = PagedKVBlocks.allocate(60, bs, reqs, 40, DEV)
        self.plan = PagedKVPlan.allocate(reqs, capacity, DEV)
        self.cache = torch.full((60, 2, bs, HKV, D), math.nan, dtype=self.dtype, device=DEV)
        self.inv_freq, self.factor = rotary_frequencies(64, 10000.0, factor=4.0, original_length=256, device=DEV)
        self.q_weight, self.k_weight = _randn(g, D, dtype=self.dtype, scale=0.1), _randn(g, D, dtype=self.dtype, scale=0.1)
        self.rows = torch.zeros(capacity, (2 * HQ + 2 * HKV) * D, dtype=self.dtype, device=DEV)
        self.context, self.query = torch.zeros(reqs, dtype=torch.int32, device=DEV), torch.zeros(reqs, dtype=torch.int32, device=DEV)
        self.out = torch.zeros(capacity, HQ, D, dtype=self.dtype, device=DEV)
        self.kept = [[] for _ in range(reqs)]                # (key, value) rows of each request

    def parts(self):
        D, HQ, HKV = self.D, self.HQ, self.HKV
        qg = self.rows[:, :2 * HQ * D].view(-1, HQ, 2 * D)
        kv = self.rows[:, 2 * HQ * D:].view(-1, 2, HKV, D)
        return qg[..., :D], qg[..., D:], kv[:, 0], kv[:, 1]

    def step(self):
        """The calls of a step, all on the current stream, nothing read back."""
        from pla.decode.paged import fused_qk_norm_rope, paged_attention_decode, paged_kv_plan
        q, gate, k, v = self.parts()
        plan = paged_kv_plan(self.pool, self.context, self.query, token_capacity=self.capacity, out=self.plan)
        turned, _ = fused_qk_norm_rope(q, k, plan.positions, q_weight=self.q_weight, k_weight=self.k_weight, weight_offset=1.0,
                                       inv_freq=self.inv_freq, attention_factor=self.factor, v=v, k_cache=self.cache[:, 0],
                                       v_cache=self.cache[:, 1], slot_mapping=plan.slot_mapping)
        paged_attention_decode(turned, self.cache[:, 0], self.cache[:, 1], self.pool.block_table, plan.seq_lens,
                               query_start_loc=plan.query_start_loc, max_query_len=self.max_query, output_gate=gate, out=self.out)
        return turned

    def load(self, context, query):
        self.context.copy_(_ints(context))
        self.query.copy_(_ints(query))
        self.rows.copy_(_randn(self.g, *self.rows.shape, dtype=self.dtype))

    def check(self, context, query, turned):
        """Against plain lists: what each request kept, its new rows from the reference of the norm, dense attention."""
        q, gate, k, v = self.parts()
        token = 0
        positions, where = [], []
        for n, (c, m) in enumerate(zip(context, query)):
            for j in range(m):
                positions.append(c + j)
                where.append(n)
        T = len(positions)
        how = dict(eps=1e-6, offset=1.0, factor=self.factor, interleaved=False)
        at = torch.tensor(positions)
        ref_q, slack_q = _rope_reference(q[:T], self.q_weight, at, self.inv_freq, **how)
        _close(turned[:T], ref_q, slack_q, "turned q")
        ref_k, slack_k = _rope_reference(k[:T], self.k_weight, at, self.inv_freq, **how)
        slots = self.plan.slot_mapping[:T]
        stored = self.cache[:, 0].reshape(-1, self.HKV, self.D)[slots]
        _close(stored, ref_k, slack_k, "stored k")
        for t in range(T):
            n = where[t]
            del self.kept[n][positions[t]:]
            self.kept[n].append((stored[t].cpu(), v[t].cpu()))
        class Plain:
            pass
        plain = Plain()
        plain.k_cache = self.cache[:, 0]
        empty = torch.zeros(0, self.HKV, self.D, dtype=self.dtype)
        plain.k = [torch.stack([a for a, _ in x]) if x else empty for x in self.kept]
        plain.v = [torch.stack([b for _, b in x]) if x else empty for x in self.kept]
        lengths = [c + m for c, m in zip(context, query)]
        ref, slack = _attention_reference(turned[:T], plain, lengths, query, self.D ** -0.5, gate[:T])
        _close(self.out[:T], ref, slack, "attention")


STEPS = [  # (context, new tokens): prompts, verify windows, roll back, a request ends and another takes its row
    ([0, 0, 0, 0, 0, 0], [8, 3, 1, 8, 0, 5]), ([8, 3, 1, 8, 0, 5], [4, 4, 4, 4, 0, 4]), ([10, 7, 2, 12, 0, 6], [8, 1, 8, 8, 8, 8]),
    ([18, 0, 3, 13, 8, 7], [4, 8, 4, 4, 4, 4]), ([0, 8, 7, 17, 9, 8], [0, 8, 8, 8, 8, 8]), ([0, 16, 15, 18, 10, 16], [7, 1, 1, 8, 1, 1])]


def test_steps_of_a_serving_program():
    s = _Serving()
    for context, query in STEPS:
        s.load(context, query)
        turned = s.step()
        s.check(context, query, turned)


def test_a_captured_step_replays_over_other_lengths():
    """One graph for all steps, eager work and reads between the replays."""
    s = _Serving(D=64, HQ=4, HKV=1, act="fp16")
    s.load([0] * 6, [0] * 6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.step()                                             # nothing to do: lengths of zero
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned = s.step()
    for context, query in STEPS:
        s.load(context, query)
        s.out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        s.check(context, query, turned)
        assert (s.out[sum(query):] == 9).all()


@pytest.mark.parametrize("D, HKV, batch", [(64, 2, 90), (128, 4, 30), (256, 1, 300)])
def test_captured_calls_of_many_runs_replay_over_other_lengths(D, HKV, batch):
    """Wavefronts that have runs of their own: what is cut, and where, follows the lengths at the time of the replay."""
    from pla.decode.paged import paged_attention_decode
    g = torch.Generator().manual_seed(D)
    bs, pages = 32, 12
    cache = _randn(g, batch * pages // 2, 2, bs, HKV, D, dtype=torch.bfloat16)
    table = torch.randint(0, cache.size(0), (batch, pages), generator=g).to(torch.int32).to(DEV)
    q = _randn(g, batch, 4 * HKV, D, dtype=torch.bfloat16)
    lengths, out = _ints([1] * batch), torch.zeros_like(q)
    call = lambda to: paged_attention_decode(q, cache[:, 0], cache[:, 1], table, lengths, out=to)
    call(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for high in (0, 1, 40, 384, 3, 200):
        lengths.copy_(torch.randint(0, high + 1, (batch,), generator=g).to(torch.int32))
        q.copy_(_randn(g, *q.shape, dtype=torch.bfloat16))
        expect = call(torch.empty_like(q))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expect)
        k = cache[:, 0][table.long()].reshape(batch, pages * bs, HKV, D).double()
        v = cache[:, 1][table.long()].reshape(batch, pages * bs, HKV, D).double()
        score = (q.double().view(batch, HKV, 4, 1, D) * k.transpose(1, 2)[:, :, None]).sum(-1) * D ** -0.5
        score = score.masked_fill(torch.arange(pages * bs, device=DEV) >= lengths[:, None, None, None], -math.inf)
        weight = torch.softmax(score, -1).nan_to_num(0.0)
        plain = (weight[..., None] * v.transpose(1, 2)[:, :, None]).sum(-2).view_as(q)
        # weights are rounded by 2^-8 at most, and the outputs; scores in 32 bits are far below that
        slack = 1.1 * 2.0 ** -8 * ((weight[..., None] * (v.transpose(1, 2)[:, :, None] - plain.view(batch, HKV, 4, 1, D)).abs()).sum(-2).view_as(q) + plain.abs()) + 1e-6
        assert ((out.double() - plain).abs() <= slack).all()


def test_two_captured_graphs_and_two_streams_do_not_share_anything():
    lengths = [3000, 50, 900, 0, 131]
    cases = []
    for seed in (1, 2):
        cache = _Cache(lengths, 2, 128, 16, "bf16", seed=seed)
        q = _randn(torch.Generator().manual_seed(seed + 10), 5, 16, 128, dtype=torch.bfloat16)
        out = torch.zeros_like(q)
        expect = _attend(cache, q, lengths, [1] * 5)
        cases.append((cache, q, out, expect, _ints(lengths)))
    from pla.decode.paged import paged_attention_decode

    def call(case):
        cache, q, out, _, lens = case
        paged_attention_decode(q, cache.k_cache, cache.v_cache, cache.table, lens, out=out)
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in cases]
    for case in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(case)
        graphs.append(graph)
    for turn in range(4):
        for case in cases:
            case[2].fill_(-1.0)
        torch.cuda.synchronize()
        for graph, stream, case in zip(graphs, streams, cases):
            with torch.cuda.stream(stream):
                if turn % 2:
                    graph.replay()
                else:
                    call(case)
        torch.cuda.synchronize()
        for case in cases:
            assert torch.equal(case[2], case[3])


def test_the_plan_serves_the_linear_attention_layers_of_the_same_step():
    """query_start_loc of the plan drives a KDA verify, its block table the align-mode commit, beside the softmax layer."""
    from pla.decode.kda_replayssm_vllm import KDAReplayCommitContext, kda_replay_verify
    from pla.decode.paged import PagedKVBlocks, paged_kv_plan
    from pla_amd.workloads import kda_replay_paged
    N, H, Q = 3, 2, 4
    w = kda_replay_paged(N, H, Q, slots=16, seed=5)
    pool = PagedKVBlocks.allocate(16, 16, N, 4, DEV)
    context = _ints([5, 14, 30])
    plan = paged_kv_plan(pool, context, _ints([Q] * N), token_capacity=w.tokens)
    assert torch.equal(plan.query_start_loc, w.offsets)
    expect = kda_replay_verify(**w.verify)
    twin = kda_replay_paged(N, H, Q, slots=16, seed=5)
    got = kda_replay_verify(**dict(twin.verify, query_start_loc=plan.query_start_loc))
    assert torch.equal(got, expect)
    # align mode: the state after the accepted tokens belongs to the block of the last one
    commit = KDAReplayCommitContext.create([twin.layer], Q, N, conv_state_layout="DS")
    source = torch.stack([pool.block_table[n, (c - 1) // 16] for n, c in enumerate((5, 14, 30))])
    accepted = _ints([2, 4, 3])
    made = commit.commit(accepted, source, plan.query_start_loc, block_table=pool.block_table, num_computed_tokens=context,
                         mamba_block_size=16, token_capacity=w.tokens)
    assert made.commit_lens.tolist() == [2, 4, 3]
    assert made.final_state_indices.tolist() == [pool.block_table[n, (c + a - 1) // 16].item() for n, (c, a) in enumerate(((5, 2), (14, 4), (30, 3)))]
    # the next step: what was not accepted falls away
    plan = paged_kv_plan(pool, context + accepted, _ints([1, 0, 1]), token_capacity=w.tokens)
    assert plan.seq_lens.tolist() == [8, 18, 34] and plan.positions[:2].tolist() == [7, 33]


def test_calls_on_another_stream_than_the_tensors_own():
    s = torch.cuda.Stream()
    cache = _Cache([700, 20], 1, 128, 32, "bf16", seed=50)
    q = _randn(torch.Generator().manual_seed(51), 2, 4, 128, dtype=torch.bfloat16)
    expect = _attend(cache, q, [700, 20], [1, 1])
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = [_attend(cache, q, [700, 20], [1, 1]) for _ in range(3)]
    s.synchronize()
    assert all(torch.equal(x, expect) for x in got)


# ---- weights ------------------------------------------------------------------------------------------------------

def _attention_reference_32(q, cache, lengths, windows, scale):
    """As _attention_reference, with the error of weights that are as good as 32-bit arithmetic makes the rest, against outputs that
    values of both signs make small.

    The two parts of a weight are off by 2^-16 of it at most (bf16: eight bits cut off, eight more rounded; fp16 2^-22), in the
    product alone, and by the least fp16, 2^-24 where the largest weight is 2^14; scores, sums and division as there."""
    T, HQ, D = q.shape
    G = HQ // cache.k_cache.size(2)
    part = 2.0 ** -16 if q.dtype == torch.bfloat16 else 2.0 ** -22
    out, slack = torch.zeros(T, HQ, D, dtype=torch.float64), torch.zeros(T, HQ, D, dtype=torch.float64)
    qd, token = q.double().cpu(), 0
    for n, (length, window) in enumerate(zip(lengths, windows)):
        for j in range(window):
            sees = min(max(length - window + j + 1, 0), max(length, 0))
            if sees:
                k, v = cache.k[n][:sees].double().repeat_interleave(G, 1), cache.v[n][:sees].double().repeat_interleave(G, 1)
                terms = qd[token][None] * k
                score = terms.sum(-1) * scale
                wrong = (terms.abs().sum(-1) * abs(scale) * D + 3 * score.abs()) * 2.0 ** -24 + 2.0 ** -22
                w = torch.softmax(score, 0)[:, :, None]
                out[token] = (w * v).sum(0)
                size = (w * v.abs()).sum(0)
                slack[token] = (w * (2 * wrong[:, :, None]) * (v - out[token]).abs()).sum(0) + (part + (sees + 16) * 2.0 ** -24) * size + sees * 2.0 ** -37 * v.abs().amax()
            token += 1
    return out, slack


@pytest.mark.parametrize("D, act, HQ, HKV, max_query", [(64, "bf16", 4, 2, 3), (64, "fp16", 8, 1, 4), (64, "bf16", 8, 1, 8), (128, "bf16", 8, 2, 2),
                                                        (128, "fp16", 7, 1, 3), (128, "fp16", 16, 2, 8), (256, "bf16", 8, 1, 2), (256, "fp16", 4, 1, 8)])
@pytest.mark.usefixtures("crowd")
def test_weights_are_as_good_as_the_sums(D, act, HQ, HKV, max_query):
    """Few keys, whose values partly cancel: an output's own rounding is then small, and a weight in 16 bits would show."""
    rng = random.Random(D + HQ)
    lengths = [1, 2, 3, 4, 5, 8, 15, 16, 17, 33, 40, 64, 100, 130, 300, 700]
    windows = [min(n, rng.randint(1, max_query)) for n in lengths]
    cache = _Cache(lengths, HKV, D, 16, act, seed=D + max_query)
    q = _randn(torch.Generator().manual_seed(HQ), sum(windows), HQ, D, dtype=DTYPES[act])
    out = _attend(cache, q, lengths, windows, max_query=max_query)
    ref, slack = _attention_reference_32(q, cache, lengths, windows, D ** -0.5)
    _close(out, ref, slack, "weights")


@pytest.mark.parametrize("D, act, HQ, HKV", [(64, "fp16", 4, 4), (64, "bf16", 12, 1), (128, "fp16", 8, 2), (128, "bf16", 16, 1), (256, "fp16", 2, 1), (256, "bf16", 8, 1)])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.usefixtures("crowd")
def test_an_infinite_value_counts_however_small_its_weight(D, act, HQ, HKV, sign):
    """Keys that weigh e^-60 and less of the others, in any place of a sequence, whose value is infinite in one channel: every token that
    sees them is infinite there, tokens before them and other channels are what they are."""
    for window, length, places in ((1, 50, (3,)), (1, 900, (600,)), (4, 700, (0, 698)), (4, 7000, (6500, 6998)), (4, 70, (68, 69))):
        cache = _Cache([length, length], HKV, D, 16, act, seed=length)
        q = _randn(torch.Generator().manual_seed(5), 2 * window, HQ, D, dtype=DTYPES[act])
        q[:, :, 0] = 8.0
        clean = _attend(cache, q, [length] * 2, [window] * 2, scale=1.0)
        for at in places:
            block, place = cache.table[0, at // 16].item(), at % 16
            cache.store[block, 0, place, :, 0] = -200.0      # the score falls by more than a thousand
            cache.store[block, 1, place, :, 7] = sign * math.inf
        before = _attend(cache, q, [length] * 2, [window] * 2, scale=1.0)
        for j in range(window):
            sees = any(at < length - window + j + 1 for at in places)
            assert (before[j, :, 7] == sign * math.inf).all() if sees else torch.equal(before[j], clean[j]), (window, length, j)
        before[:, :, 7] = 0
        assert before.isfinite().all()
        assert torch.equal(before[window:, :, 8:], clean[window:, :, 8:])


# ---- plans of every size ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("capacity", [40, 300, 1024, 1025, 1500, 1920, 2048, 2049, 3000])
@pytest.mark.parametrize("batch", [1, 40, 256, 257, 700, 1024, 1025, 2500, 4096, 4097, 8192, 9001])
@pytest.mark.parametrize("mapped", [False, True])
def test_plans_of_every_size(batch, capacity, mapped):
    """Batches and token rows on both sides of each size from which a plan is made in another way (256 and 1024 entries, passes of 4096,
    1024 and 2048 token rows).  Steps whose rows just fit, run out among the last entries and fall back, over a stack that runs out too."""
    rng, bs = random.Random(batch * 4099 + capacity + mapped), 8
    rows = min(8192, batch + 50) if mapped else batch + 3
    longest = 2 * capacity // batch + 3
    cols = -(-(longest + 24) // bs) + 1
    pool, lists = _pool(2 + int(0.9 * batch * (8 + capacity / batch) / bs + 0.6 * batch), bs, rows, cols)
    # more entries than rows that a mapping may name: the last ones name rows of earlier ones
    index = rng.sample(range(rows), min(batch, rows)) + [rng.randrange(rows) for _ in range(batch - rows)] if mapped else None
    context, refused = [rng.randint(0, 9) for _ in range(batch)], 0
    for step, total in enumerate((capacity - 1, capacity + batch // 20 + 3, capacity)):
        query = [0] * batch
        for _ in range(total):
            n = rng.randrange(batch)
            query[n] = min(query[n] + 1, longest)
        if step == 2:
            query[-1] = 0
            query[batch // 2] = -1                           # an entry in the middle that is none, rows of nobody at the end
        used = index
        if mapped and step == 1 and batch > 4:
            used = list(index)
            used[-1], used[-3] = used[0], rows
        plan, lists = _check_plan(pool, lists, context, query, used, capacity)
        refused += sum(s == 0 and c + q > 0 for s, c, q in zip(plan.seq_lens.tolist(), context, query))
        context = [rng.choice((0, max(0, c - 3), min(cols * bs - longest, c + max(q, 0)))) for c, q in zip(context, query)]
    assert refused > 0


# ---- rows of a prompt ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("T, HQ, HKV, D, rot, interleaved, norm, act, stored", [
    (7300, 24, 6, 128, 128, False, True, "bf16", True), (16500, 20, 4, 64, 32, True, True, "fp16", False), (3500, 20, 10, 256, 64, False, True, "bf16", True),
    (2600, 40, 40, 128, 96, False, True, "fp16", True), (6100, 33, 1, 128, 128, True, False, "bf16", False), (4096, 16, 2, 256, 256, False, True, "fp16", True),
    (9001, 9, 3, 128, 128, False, True, "bf16", True)])
def test_norm_rotation_and_store_of_a_prompt(T, HQ, HKV, D, rot, interleaved, norm, act, stored):
    """Wavefronts that have many steps of a token's heads, with weights, stored and unstored, at sizes whose rows stay in the caches and
    at such whose do not.  Every row against 64 bits on the GPU."""
    from pla.decode.paged import fused_qk_norm_rope
    dtype = DTYPES[act]
    g = torch.Generator(device=DEV).manual_seed(T)
    row = torch.empty(T, (HQ + 2 * HKV) * D + 8, dtype=dtype, device=DEV).normal_(generator=g)
    q, k, v = (row[:, a * D:b * D].view(T, b - a, D) for a, b in ((0, HQ), (HQ, HQ + HKV), (HQ + HKV, HQ + 2 * HKV)))
    before = row.clone()
    positions = torch.randint(0, 1 << 20, (T,), generator=g, device=DEV, dtype=torch.int32)
    inv_freq = (10000.0 ** -(torch.arange(0, rot, 2).double() / rot)).float().to(DEV)
    q_weight, k_weight = (torch.empty(D, dtype=dtype, device=DEV).normal_(0, 0.2, generator=g) if norm else None for _ in range(2))
    bs, blocks = 16, -(-T // 16) + 3
    caches = [torch.full((blocks, bs, HKV, D), 7.0, dtype=dtype, device=DEV) for _ in range(2)] if stored else None
    slots = torch.randperm(blocks * bs, generator=g, device=DEV)[:T]
    slots[T - 40:] = -1
    store = dict(v=v, k_cache=caches[0], v_cache=caches[1], slot_mapping=slots) if stored else {}
    k_out = torch.zeros(T, HKV, D, dtype=dtype, device=DEV)
    q_out, _ = fused_qk_norm_rope(q, k, positions, q_weight=q_weight, k_weight=k_weight, weight_offset=1.0, inv_freq=inv_freq,
                                  attention_factor=1.25, interleaved=interleaved, k_out=k_out, **store)
    assert torch.equal(row, before)
    angle = positions.double()[:, None, None] * inv_freq.double()
    cos, sin = angle.cos() * 1.25, angle.sin() * 1.25
    first = torch.arange(0, rot, 2, device=DEV) if interleaved else torch.arange(rot // 2, device=DEV)
    second = first + (1 if interleaved else rot // 2)
    info = torch.finfo(dtype)
    for got, x, weight in ((q_out, q, q_weight), (k_out, k, k_weight)):
        for part in range(0, T, 2000):
            y = x[part:part + 2000].double()
            if weight is not None:
                y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * (weight.double() + 1.0)
            size = y.abs()
            a, b, c, s = y[..., first], y[..., second], cos[part:part + 2000], sin[part:part + 2000]
            y[..., first], y[..., second] = a * c - b * s, b * c + a * s
            size[..., first] = size[..., second] = (a.abs() + b.abs()) * 1.25
            slack = size * 2.0 ** -20                        # as in _rope_reference
            bound = (y.abs() + slack) * (info.eps / 2) + slack + info.tiny * info.eps / 2
            assert ((got[part:part + 2000].double() - y).abs() <= bound).all(), part
    if stored:
        flat, kept = [c.view(-1, HKV, D) for c in caches], slots >= 0
        assert torch.equal(flat[0][slots[kept]], k_out[kept]) and torch.equal(flat[1][slots[kept]], v[kept])
        rest = torch.ones(blocks * bs, dtype=torch.bool, device=DEV)
        rest[slots[kept]] = False
        assert (flat[0][rest] == 7).all() and (flat[1][rest] == 7).all()


# ---- wavefronts alone ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("places", [(4,), (13,), (4, 13), (1, 2, 14, 15)])
@pytest.mark.parametrize("D, HKV, act", [(64, 8, "bf16"), (64, 8, "fp16"), (128, 4, "bf16"), (128, 4, "fp16"), (256, 4, "fp16")])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_values_set_aside_in_two_steps_of_every_form(places, D, HKV, act, value):
    """As above for every head size and type: a wavefront has at least three groups of 32 keys of the long runs."""
    lengths = [1000, 1064, 1032] + [2000 + 7 * i for i in range(37)]
    windows = [16] * 3 + [1] * 37
    cache = _Cache(lengths, HKV, D, 16, act, seed=73)
    q = _randn(torch.Generator().manual_seed(74), sum(windows), HKV, D, dtype=DTYPES[act])
    clean = _attend(cache, q, lengths, windows)
    for n in range(3):
        for place in places:
            at = lengths[n] - 16 + place
            cache.store[cache.table[n, at // 16].item(), 1, at % 16, :, 5] = value
    got = _attend(cache, q, lengths, windows)
    for n in range(3):
        rows = got[16 * n:16 * n + 16, :, 5]
        assert rows[:places[0]].isfinite().all()
        assert rows[places[0]:].isnan().all() if math.isnan(value) else (rows[places[0]:] == value).all()
        rows[places[0]:] = clean[16 * n + places[0]:16 * n + 16, :, 5]
    assert torch.equal(got[48:], clean[48:])
    ref, slack = _attention_reference_32(q[:48], cache, lengths[:3], windows[:3], D ** -0.5)
    _close(got[:48], ref, slack, "set aside")


@pytest.mark.parametrize("D, HKV, batch, window", [(64, 2, 90, 1), (128, 4, 300, 1), (256, 1, 300, 4), (128, 2, 40, 8), (64, 1, 600, 2)])
def test_calls_of_many_runs_side_by_side(D, HKV, batch, window):
    """Two captured graphs and two streams over batches whose wavefronts have runs of their own (and one whose workgroups work together),
    with fewer and with more runs than workgroups: none reads what another leaves."""
    from pla.decode.paged import paged_attention_decode
    bs, pages, cases = 16, 80, []
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed + D)
        cache = _randn(g, 500, 2, bs, HKV, D, dtype=torch.bfloat16)
        table = torch.randint(0, 500, (batch, pages), generator=g).to(torch.int32).to(DEV)
        lengths = torch.randint(window, pages * bs + 1, (batch,), generator=g).to(torch.int32).to(DEV)
        q = _randn(g, batch * window, 2 * HKV, D, dtype=torch.bfloat16)
        offsets = torch.arange(0, batch * window + 1, window, dtype=torch.int32, device=DEV)
        cases.append((q, cache[:, 0], cache[:, 1], table, lengths, offsets, torch.zeros_like(q)))

    def call(q, k, v, table, lengths, offsets, out):
        return paged_attention_decode(q, k, v, table, lengths, query_start_loc=offsets, max_query_len=window, out=out)
    expects = [call(*case[:6], torch.empty_like(case[0])) for case in cases]
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in cases]
    for case in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(*case)
        graphs.append(graph)
    for turn in range(6):
        for case in cases:
            case[-1].fill_(-1.0)
        torch.cuda.synchronize()
        for graph, stream, case in zip(graphs, streams, cases):
            with torch.cuda.stream(stream):
                if turn % 2:
                    graph.replay()
                else:
                    call(*case)
        torch.cuda.synchronize()
        for case, expect in zip(cases, expects):
            assert torch.equal(case[-1], expect), turn


# ---- far positions ------------------------------------------------------------------------------------------------

def _exact_turns(positions, inv_freq):
    """Cosine and sine of position * inv_freq with the product, and its part of a revolution, in 70 digits."""
    from decimal import Decimal, getcontext
    getcontext().prec = 70

    def arctan_of_inverse(n):
        term = total = Decimal(1) / n
        k = 1
        while abs(term) > Decimal(10) ** -68:
            term, k = -term / (n * n), k + 2
            total += term / k
        return total
    turn = 8 * (4 * arctan_of_inverse(5) - arctan_of_inverse(239))
    rest = [[math.fmod(float(Decimal(p) * Decimal(f) % turn), 2 * math.pi) for f in inv_freq.tolist()] for p in positions]
    rest = torch.tensor(rest, dtype=torch.float64)
    return rest.cos(), rest.sin()


@pytest.mark.parametrize("act", ["bf16", "fp16"])
def test_angles_are_as_exact_at_far_positions_as_at_near_ones(act):
    from pla.decode.paged import fused_qk_norm_rope
    D = 128
    far = [3, 2 ** 31 - 1, -2 ** 31, 2 ** 36 + 12345, -2 ** 40 - 1, 2 ** 45 + 7, 2 ** 50 - 3, 2 ** 52 + 1, -2 ** 53 + 1, 2 ** 53 - 1]
    g, _, q, k, _, _ = _rope_case(6, len(far), 4, 2, D, act)
    inv_freq = (1000000.0 ** -(torch.arange(0, D, 2).double() / D)).float().to(DEV)
    q_out, k_out = fused_qk_norm_rope(q, k, torch.tensor(far, dtype=torch.int64, device=DEV), inv_freq=inv_freq)
    cos, sin = (x[:, None, :] for x in _exact_turns(far, inv_freq))
    for got, x in ((q_out, q), (k_out, k)):
        a, b = x.double().cpu().split(D // 2, -1)
        size = (a.abs() + b.abs()) * 2.0 ** -20              # as in _rope_reference
        _close(got, torch.cat([a * cos - b * sin, b * cos + a * sin], -1), torch.cat([size, size], -1), "far")


# ---- shared memory ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("tokens, token_stride, head_stride, ahead", [(5, 432, 248, -72), (4, 480, 408, 800), (2, 408, 296, 184), (2, 464, 280, 400)])
def test_written_rows_among_rows_that_lie_on_each_other_are_refused(tokens, token_stride, head_stride, ahead):
    """q's rows lie on each other, as it may be where they are only read; some place of k_out is one of q's."""
    from pla.decode.paged import fused_qk_norm_rope
    buffer = torch.zeros(8192, dtype=torch.bfloat16, device=DEV)
    q = buffer.as_strided((tokens, 4, 64), (token_stride, head_stride, 1), 1024)
    k_out = buffer.as_strided((tokens, 2, 64), (token_stride, head_stride, 1), 1024 + ahead)
    place = lambda heads, start: {start + t * token_stride + h * head_stride + c for t in range(tokens) for h in range(heads) for c in range(64)}
    assert place(4, 0) & place(2, ahead)
    k = torch.zeros(tokens, 2, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="k_out must not share memory with q"):
        fused_qk_norm_rope(q, k, k_out=k_out)
    # read only, and beside it: what such rows hold is what their copy holds
    apart = torch.zeros(tokens, 2, 64, dtype=torch.bfloat16, device=DEV)
    buffer.normal_()
    got, same = fused_qk_norm_rope(q, k, k_out=apart)
    assert same.data_ptr() == apart.data_ptr() and torch.equal(got, q)
