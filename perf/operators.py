"""The operators of the paged softmax-attention layers that stand between a model's linear-attention layers.

Three operators, each timed as a serving program calls it:

  plan       block tables and slot maps of a serving step, built on the GPU from the requests' lengths
  rope       norms of queries and keys for each head, the position rotation, and the write into the paged cache
  attention  attention of one new token, or of a window of draft tokens, over the paged cache

Draft windows, batch sizes and sequence lengths lie in the ranges of the decode and prefill cases of this framework's
linear-attention layers, with which these operators share their batches.  ``own`` chooses between the framework's entry
points and a plain form of elementary torch operations.  Lengths follow from the case, everything else from the seed.
"""
import math
import random
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


# ---- cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of an ordinary batch: one token each, now and then a request needs a block
        dict(name="plan_decode_b64", op="plan", batch=64, lo=100, hi=6000, window=1, block=16, mapped=False),
        # speculative decoding of a large service: windows of up to eight tokens, batch entries point at request rows
        dict(name="plan_verify_b1500", op="plan", batch=1500, lo=20, hi=4000, window=8, block=32, mapped=True),
        # a step that takes in prompts: 40 960 new tokens, thousands of new blocks
        dict(name="plan_prefill_b40", op="plan", batch=40, lo=0, hi=500, window=1024, block=16, mapped=False),
        # a few concurrent chats: launch and latency count
        dict(name="rope_decode_b8", op="rope", tokens=8, HQ=16, HKV=2, D=128, rot=128, interleaved=False, norm=True, gated=False,
             store=True, block=16, act="bf16"),
        # a verify step of 64 x 4 tokens: large heads of which a quarter turns, q beside its output gate in one row
        dict(name="rope_verify_t256", op="rope", tokens=256, HQ=16, HKV=2, D=256, rot=64, interleaved=False, norm=True, gated=True,
             store=True, block=16, act="bf16"),
        # a long prompt at far positions: interleaved pairs, no norms, dense keys for the prefill's own attention
        dict(name="rope_prefill_t16384", op="rope", tokens=16384, HQ=32, HKV=8, D=128, rot=128, interleaved=True, norm=False,
             gated=False, store=False, block=16, act="fp16"),
        # a few concurrent chats: launch and latency count
        dict(name="attention_chat_b8", op="attention", batch=8, lo=180, hi=700, window=1, ragged=False, HQ=16, HKV=2, D=128, block=16,
             gate=False, act="bf16"),
        # the ordinary decode step of a full batch
        dict(name="attention_decode_b256", op="attention", batch=256, lo=300, hi=4000, window=1, ragged=False, HQ=32, HKV=8, D=128,
             block=64, gate=False, act="bf16"),
        # one request with a very long context: the cache's length itself has to be split
        dict(name="attention_long_b1", op="attention", batch=1, lo=131000, hi=131000, window=1, ragged=False, HQ=16, HKV=2, D=256,
             block=16, gate=True, act="bf16"),
        # verify of four draft tokens, 32 query rows a key-value head, gated output
        dict(name="attention_verify_b64", op="attention", batch=64, lo=1000, hi=16000, window=4, ragged=False, HQ=32, HKV=4, D=128,
             block=16, gate=True, act="bf16"),
        # windows of 0 to 8 tokens over contexts of every length, small heads without sharing
        dict(name="attention_ragged_b37", op="attention", batch=37, lo=1, hi=9000, window=8, ragged=True, HQ=10, HKV=10, D=64,
             block=16, gate=False, act="fp16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


HEADS = ((8, 1), (8, 8), (16, 2), (10, 10), (16, 16), (32, 4), (32, 8), (28, 4), (5, 5), (15, 3))


def draw(rng):
    op = rng.choice(("plan", "rope", "attention"))
    act = rng.choice(("bf16", "bf16", "fp16"))
    block = rng.choice((16, 16, 32, 64, 80, 528))
    if op == "plan":
        batch = _log_int(rng, 1, 1500)
        if rng.random() < 0.3:
            return dict(op=op, batch=min(batch, 40), lo=0, hi=500, window=_log_int(rng, 64, 1024), block=block, mapped=rng.random() < 0.5)
        lo = _log_int(rng, 1, 200)
        return dict(op=op, batch=batch, lo=lo, hi=lo + _log_int(rng, 50, 3800), window=rng.randint(1, 8), block=block,
                    mapped=rng.random() < 0.5)
    HQ, HKV = rng.choice(HEADS)
    D = rng.choice((64, 128, 128, 256))
    if op == "rope":
        rot = rng.choice((0, D, D, D // 2, D // 4))
        return dict(op=op, tokens=_log_int(rng, 1, 16384 * 32 * 128 // (HQ * D) // 2), HQ=HQ, HKV=HKV, D=D, rot=rot,
                    interleaved=rng.random() < 0.5, norm=rot == 0 or rng.random() < 0.7, gated=rng.random() < 0.3,
                    store=rng.random() < 0.6, block=block, act=act)
    window = rng.choice((1, 1, 1, 2, 4, 8, 17, 32))
    # no more keys than the full batch, no more products than the verify step that are listed
    keys = min(256 * 1400 * 8 * 128 // (HKV * D), 64 * 5400 * 4 * 32 * 128 // (window * HQ * D))
    lo = _log_int(rng, 1, min(4000, keys))
    hi = _log_int(rng, lo, min(60000, keys))
    return dict(op=op, batch=_log_int(rng, 1, max(1, min(300, keys // hi))), lo=lo, hi=hi, window=window,
                ragged=window > 1 and rng.random() < 0.5, HQ=HQ, HKV=HKV, D=D, block=block, gate=rng.random() < 0.4, act=act)


def _spread(rng, n, lo, hi):
    """n lengths between lo and hi, even over their logarithm."""
    return [min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1))) - 0.5))) for _ in range(n)]


def _case_rng(c):
    return random.Random(str(sorted((k, v) for k, v in c.items() if k != "name")))


def _plan_lengths(c):
    """Lengths of two steps that follow on each other again and again: (context, new tokens) of every request.  A request in
    eight is over after the first step, the others go on from what was accepted of their window; in the first step of the next
    pass other requests have come in their place."""
    rng = _case_rng(c)
    context = _spread(rng, c["batch"], c["lo"], c["hi"])
    prompts = c["window"] > 32
    first, second = [], []
    for n, length in enumerate(context):
        new = 1 + rng.randrange(c["window"]) if not prompts else c["window"]
        first.append((length, new))
        over = n % 8 == 5
        second.append((0, 0) if over else (length + rng.randint(0, new), 1 if prompts else 1 + rng.randrange(c["window"])))
    return first, second


def _attention_lengths(c):
    """(cached tokens with the window, window) of every request; one of a larger batch has nothing cached."""
    rng = _case_rng(c)
    out = []
    for n, length in enumerate(_spread(rng, c["batch"], c["lo"], c["hi"])):
        window = rng.randint(0 if n else 1, c["window"]) if c["ragged"] else c["window"]
        out.append((max(length, window) if n != 6 or not c["ragged"] else 0, window))
    return out


# ---- inputs -----------------------------------------------------------------------------------------------------

class _Draw:
    """Seeded draws on the GPU."""

    def __init__(self, seed):
        self.device = torch.device("cuda", torch.cuda.current_device())
        self.g = torch.Generator(device=self.device).manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, scale=1.0):
        return torch.empty(*shape, dtype=dtype, device=self.device).normal_(0.0, scale, generator=self.g)

    def permutation(self, n):
        return torch.randperm(n, generator=self.g, device=self.device).to(torch.int32)

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)


def _prepare_plan(c, r):
    first, second = _plan_lengths(c)
    N, bs = c["batch"], c["block"]
    rows = 2 * N + 3 if c["mapped"] else N
    blocks = [max(-(-(a + b) // bs) for a, b in pair) for pair in zip(first, second)]
    cols, total = max(blocks) + 2, sum(blocks) + 8
    row_of = r.permutation(rows)[:N] if c["mapped"] else None
    # the pool as the second step leaves it, block 0 kept aside
    held = [-(-(a + b) // bs) for a, b in second]
    order = 1 + r.permutation(total)
    grid = torch.arange(cols, device=r.device)[None, :]
    held_n = r.ints(held)
    start = held_n.cumsum(0) - held_n
    table = torch.zeros(rows, cols, dtype=torch.int32, device=r.device)
    held_rows = torch.zeros(rows, dtype=torch.int32, device=r.device)
    where = row_of.long() if c["mapped"] else torch.arange(N, device=r.device)
    mine = order[(start[:, None] + grid).clamp(max=total - 1)]
    table[where] = torch.where(grid < held_n[:, None], mine, 0).to(torch.int32)
    held_rows[where] = held_n
    used = sum(held)
    free = torch.zeros(total + 1, dtype=torch.int32, device=r.device)
    free[:total - used] = order[used:]
    steps = []
    for lengths in (first, second):
        tokens = sum(b for _, b in lengths)
        capacity = tokens if tokens < 256 else -(-tokens // 256) * 256           # the padded size of a captured step
        steps.append(SimpleNamespace(context=r.ints([a for a, _ in lengths]), query=r.ints([b for _, b in lengths]), capacity=capacity))
    s = SimpleNamespace(case=c, table=table, held=held_rows, free=free, count=r.ints([total - used]), row_of=row_of, steps=steps)
    if own:
        from pla_amd.decode.paged import PagedKVBlocks
        s.pool = PagedKVBlocks(block_table=s.table, held_blocks=s.held, free_blocks=s.free, free_count=s.count, block_size=bs)
    return s


def _rope_geometry(c):
    width = 2 * c["D"] if c["gated"] else c["D"]
    blocks = -(-c["tokens"] // c["block"]) + 3
    return width, blocks


def _prepare_rope(c, r):
    T, HQ, HKV, D, act = c["tokens"], c["HQ"], c["HKV"], c["D"], DTYPES[c["act"]]
    width, blocks = _rope_geometry(c)
    # one projection row: q (beside its gate where there is one), k, v
    row = r.normal(T, HQ * width + 2 * HKV * D, dtype=act)
    q = row[:, :HQ * width].view(T, HQ, width)[:, :, :D]
    k = row[:, HQ * width:HQ * width + HKV * D].view(T, HKV, D)
    v = row[:, HQ * width + HKV * D:].view(T, HKV, D)
    s = SimpleNamespace(case=c, q=q, k=k, v=v, q_weight=None, k_weight=None, positions=None, inv_freq=None, factor=1.0, k_cache=None,
                        v_cache=None, slots=None)
    if c["norm"]:
        s.q_weight, s.k_weight = r.normal(D, dtype=act, scale=0.1), r.normal(D, dtype=act, scale=0.1)     # about an offset of one
    if c["rot"]:
        s.positions = torch.randint(0, 1 << 20, (T,), generator=r.g, device=r.device, dtype=torch.int32)
        exponent = torch.arange(0, c["rot"], 2, device=r.device, dtype=torch.float64) / c["rot"]
        s.inv_freq, s.factor = (1e6 ** -exponent).to(torch.float32), 1.125
    if c["store"]:
        s.k_cache, s.v_cache = (torch.zeros(blocks, c["block"], HKV, D, dtype=act, device=r.device) for _ in range(2))
        s.slots = torch.randperm(blocks * c["block"], generator=r.g, device=r.device)[:T].contiguous()
        s.slots[T - T // 16:] = -1                           # padding of a captured step
    s.q_out = torch.zeros(T, HQ, D, dtype=act, device=r.device)
    s.k_out = None if c["store"] else torch.zeros(T, HKV, D, dtype=act, device=r.device)
    return s


def _prepare_attention(c, r):
    lengths = _attention_lengths(c)
    HQ, HKV, D, bs, act = c["HQ"], c["HKV"], c["D"], c["block"], DTYPES[c["act"]]
    pages = [-(-a // bs) for a, _ in lengths]
    cols, total = max(pages) + 1, sum(pages) + 1
    # pages of a long-running service: in no order; block 0 kept aside
    order = 1 + r.permutation(total)
    count = r.ints(pages)
    start, grid = count.cumsum(0) - count, torch.arange(cols, device=r.device)[None, :]
    table = torch.where(grid < count[:, None], order[(start[:, None] + grid).clamp(max=total - 1)], 0).to(torch.int32)
    cache = r.normal(total + 1, 2, bs, HKV, D, dtype=act)
    tokens = sum(w for _, w in lengths)
    offsets = [0]
    for _, w in lengths:
        offsets.append(offsets[-1] + w)
    # queries that look at some keys more than at others
    q = r.normal(tokens, HQ, D, dtype=act, scale=1.5)
    return SimpleNamespace(case=c, q=q, k_cache=cache[:, 0], v_cache=cache[:, 1], table=table, seq_lens=r.ints([a for a, _ in lengths]),
                           offsets=None if c["window"] == 1 else r.ints(offsets), scale=D ** -0.5,
                           gate=r.normal(tokens, HQ, D, dtype=act) if c["gate"] else None,
                           out=torch.zeros(tokens, HQ, D, dtype=act, device=r.device))


def prepare(case, seed):
    r = _Draw(seed)
    return {"plan": _prepare_plan, "rope": _prepare_rope, "attention": _prepare_attention}[case["op"]](case, r)


# ---- one pass ---------------------------------------------------------------------------------------------------

def _plain_plan(s, step):
    bs, (rows, cols), device = s.case["block"], s.table.shape, s.table.device
    c, q, N, capacity = step.context.long(), step.query.long(), step.context.numel(), step.capacity
    row = s.row_of.long() if s.row_of is not None else torch.arange(N, device=device)
    rows_used = torch.where((q >= 0) & (q <= capacity), q, 0)
    ends = rows_used.cumsum(0)
    inside = (row >= 0) & (row < rows)
    at = row.clamp(0, rows - 1)
    first = torch.full((rows,), N, device=device).scatter_reduce(0, at, torch.where(inside, torch.arange(N, device=device), N), "amin")
    held = s.held[at].long()
    want = (c + q + bs - 1) // bs
    sound = inside & (first[at] == torch.arange(N, device=device)) & (c >= 0) & (q >= 0) & (q <= capacity) & (want <= cols) & (ends <= capacity)
    want = torch.where(sound, want, held)
    # surplus blocks go back on the stack
    grid = torch.arange(cols, device=device)[None, :]
    surplus = (held - want).clamp(min=0)
    back = (grid >= want[:, None]) & (grid < held[:, None]) & sound[:, None]
    place = s.count.long() + (surplus.cumsum(0) - surplus)[:, None] + grid - want[:, None]
    last = s.free.numel() - 1                                # one entry past the stack takes what is not moved
    s.free.scatter_(0, torch.where(back, place, last).flatten(), torch.where(back, s.table[at], 0).flatten())
    height = s.count.long() + surplus.sum()
    # new blocks come off it
    need = (want - held).clamp(min=0)
    total = need.cumsum(0)
    granted = sound & ((need == 0) | (total <= height))
    take = (grid >= held[:, None]) & (grid < want[:, None]) & granted[:, None]
    source = height - 1 - ((total - need)[:, None] + grid - held[:, None])
    taken = s.free[source.clamp(0, last)]
    mine = torch.where(take, taken, s.table[at])
    s.table[at] = mine
    s.held[at] = torch.where(granted, want, held).to(torch.int32)
    s.count.copy_(height - torch.where(granted, need, 0).sum())
    # token rows
    offsets = torch.cat([torch.zeros(1, dtype=torch.long, device=device), ends]).clamp(max=capacity)
    t = torch.arange(capacity, device=device)
    entry = torch.searchsorted(ends, t, right=True)
    live = entry < N
    entry = entry.clamp(max=N - 1)
    live = live & granted[entry]
    position = torch.where(live, c[entry] + t - (ends - rows_used)[entry], 0)
    block = mine[entry, (position // bs).clamp(max=cols - 1)].long()
    slots = torch.where(live, block * bs + position % bs, -1)
    return offsets.to(torch.int32), torch.where(granted, c + q, 0).to(torch.int32), position.to(torch.int32), slots


def _run_plan(s):
    results = []
    for step in s.steps:
        if own:
            from pla_amd.decode.paged import paged_kv_plan
            p = paged_kv_plan(s.pool, step.context, step.query, s.row_of, token_capacity=step.capacity)
            results += [p.query_start_loc, p.seq_lens, p.positions, p.slot_mapping]
        else:
            results += _plain_plan(s, step)
    return results + [s.table, s.held, s.free[:-1], s.count]


def _plain_heads(s, x, weight):
    """Norm and rotation of one tensor of heads, in 32 bits; angles in 64."""
    c = s.case
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * (weight.float() + 1.0)
    if c["rot"]:
        angle = s.positions.double()[:, None] * s.inv_freq.double()[None, :]
        cos, sin = ((f(angle) * s.factor).float()[:, None, :] for f in (torch.cos, torch.sin))
        turned, rest = y[..., :c["rot"]], y[..., c["rot"]:]
        if c["interleaved"]:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
        else:
            a, b = turned[..., :c["rot"] // 2], turned[..., c["rot"] // 2:]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        y = torch.cat([turned, rest], dim=-1)
    return y.to(x.dtype)


def _run_rope(s):
    c = s.case
    if own:
        from pla_amd.decode.paged import fused_qk_norm_rope
        fused_qk_norm_rope(s.q, s.k, s.positions, q_weight=s.q_weight, k_weight=s.k_weight, eps=EPS, weight_offset=1.0,
                           inv_freq=s.inv_freq, attention_factor=s.factor, interleaved=c["interleaved"], q_out=s.q_out, k_out=s.k_out,
                           v=s.v if c["store"] else None, k_cache=s.k_cache, v_cache=s.v_cache, slot_mapping=s.slots)
    else:
        s.q_out.copy_(_plain_heads(s, s.q, s.q_weight))
        k = _plain_heads(s, s.k, s.k_weight)
        if c["store"]:
            kept = s.slots >= 0
            for cache, x in ((s.k_cache, k), (s.v_cache, s.v)):
                flat = cache.view(-1, c["HKV"], c["D"])
                at = s.slots.clamp(min=0)
                # rows of padding write back what stands at the first stored slot
                at = torch.where(kept, at, at[0])
                flat[at] = torch.where(kept[:, None, None], x, x[0])
        else:
            s.k_out.copy_(k)
    return (s.q_out, s.k_cache, s.v_cache) if c["store"] else (s.q_out, s.k_out)


def _plain_attention(s):
    c = s.case
    HQ, HKV, D, bs = c["HQ"], c["HKV"], c["D"], c["block"]
    G, W = HQ // HKV, c["window"]
    N, cols = s.table.shape
    out = torch.zeros_like(s.q)
    # as many requests at a time as fit 2 GB of widened keys
    group = max(1, int(5e8 / (cols * bs * HKV * max(D, W * G))))
    for n0 in range(0, N, group):
        pages = s.table[n0:n0 + group].long()
        n, L = pages.size(0), cols * bs
        k = s.k_cache[pages].view(n, L, HKV, D).permute(0, 2, 3, 1).float().contiguous()
        v = s.v_cache[pages].view(n, L, HKV, D).permute(0, 2, 1, 3).float().contiguous()
        length = s.seq_lens[n0:n0 + n].long()
        if s.offsets is None:
            begin = torch.arange(n0, n0 + n, device=k.device)
            count = torch.ones_like(begin)
        else:
            begin, end = s.offsets[n0:n0 + n].long(), s.offsets[n0 + 1:n0 + n + 1].long()
            count = end - begin
        j = torch.arange(W, device=k.device)
        real = j[None, :] < count[:, None]                                        # [n, W]
        at = (begin[:, None] + j[None, :]).clamp(max=s.q.size(0) - 1)
        q = s.q[at].float().view(n, W, HKV, G, D).permute(0, 2, 1, 3, 4).reshape(n, HKV, W * G, D)
        score = torch.matmul(q, k) * s.scale                                      # [n, HKV, W G, L]
        limit = (length[:, None] - count[:, None] + j[None, :] + 1)               # keys a token sees
        seen = torch.arange(L, device=k.device)[None, None, :] < limit[:, :, None]
        seen = seen.repeat_interleave(G, dim=1)[:, None]
        score = torch.where(seen, score, -math.inf)
        top = score.amax(-1, keepdim=True)
        weight = torch.where(seen, torch.exp(score - torch.where(top == -math.inf, 0.0, top)), 0.0)
        total = weight.sum(-1, keepdim=True)
        # what stands behind a request's end, or in the pages of another, has no weight and must not count
        v = torch.where((torch.arange(L, device=k.device)[None, :] < length[:, None])[:, None, :, None], v, 0.0)
        o = torch.matmul(weight, v) / torch.where(total == 0, 1.0, total)
        o = o.view(n, HKV, W, G, D).permute(0, 2, 1, 3, 4).reshape(n, W, HQ, D)
        if s.gate is not None:
            o = o / (1.0 + torch.exp(-s.gate[at].float()))
        out.index_put_((torch.where(real, at, begin[:, None].clamp(max=s.q.size(0) - 1)),),
                       torch.where(real[:, :, None, None], o.to(s.q.dtype), 0.0).to(s.q.dtype), accumulate=True)
    s.out.copy_(out)
    return s.out


def _run_attention(s):
    if not own:
        return _plain_attention(s)
    from pla_amd.decode.paged import paged_attention_decode
    return paged_attention_decode(s.q, s.k_cache, s.v_cache, s.table, s.seq_lens, query_start_loc=s.offsets,
                                  max_query_len=s.case["window"], scale=s.scale, output_gate=s.gate, out=s.out)


def run(state):
    return {"plan": _run_plan, "rope": _run_rope, "attention": _run_attention}[state.case["op"]](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "plan":
        first, second = _plan_lengths(c)
        moved, tokens = 0, 0
        for (a, b), (d, e) in zip(first, second):
            moved += 2 * abs(-(-(a + b) // c["block"]) - -(-(d + e) // c["block"]))   # there and back again
            tokens += b + e
        # lengths in, offsets and lengths out, held counts in and out; a moved block is read and written; a token's block is
        # read, its position and slot are written
        return {"bytes": 2 * c["batch"] * (8 + 8 + 8 + (4 if c["mapped"] else 0)) + 8 * moved + 16 * tokens, "flops": 0}
    if c["op"] == "rope":
        heads = c["HQ"] + c["HKV"] * (2 if c["store"] else 1)
        moved = c["tokens"] - (c["tokens"] // 16 if c["store"] else 0)
        read = 2 * c["tokens"] * c["HQ"] * c["D"] * 2 + 2 * moved * (heads - c["HQ"]) * c["D"] * 2
        turned = c["tokens"] * (c["HQ"] + c["HKV"]) * c["D"]
        return {"bytes": read + c["tokens"] * ((4 if c["rot"] else 0) + (8 if c["store"] else 0)), "flops": turned * (3 * bool(c["rot"]) + 4 * c["norm"])}
    lengths = _attention_lengths(c)
    keys = sum(a for a, w in lengths if w)
    tokens = sum(w for _, w in lengths)
    pairs = sum(max(0, a - w + j + 1) for a, w in lengths for j in range(w))
    return {"bytes": keys * c["HKV"] * c["D"] * 4 + tokens * c["HQ"] * c["D"] * (6 if c["gate"] else 4) + 4 * (keys // c["block"] + len(lengths)),
            "flops": 4 * pairs * c["HQ"] * c["D"]}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------

def _exact_plan(s):
    c, bs = s.case, s.case["block"]
    table, held, free = s.table.tolist(), s.held.tolist(), s.free.tolist()
    count = s.count.tolist()[0]
    rows = s.row_of.tolist() if s.row_of is not None else list(range(c["batch"]))
    results = []
    for step in s.steps:
        lengths = list(zip(step.context.tolist(), step.query.tolist()))
        for row, (a, b) in zip(rows, lengths):
            want = -(-(a + b) // bs)
            for page in range(want, held[row]):
                free[count] = table[row][page]
                count += 1
            held[row] = min(held[row], want)
        offsets, seqs, positions, slots = [0], [], [], []
        height, asked = count, 0
        for row, (a, b) in zip(rows, lengths):
            want = -(-(a + b) // bs)
            asked += want - held[row]
            granted = want == held[row] or asked <= height
            if granted:
                while held[row] < want:
                    count -= 1
                    table[row][held[row]] = free[count]
                    held[row] += 1
            for p in range(a, a + b):
                positions.append(p if granted else 0)
                slots.append(table[row][p // bs] * bs + p % bs if granted else -1)
            offsets.append(offsets[-1] + b)
            seqs.append(a + b if granted else 0)
        spare = step.capacity - len(slots)
        results += [offsets, seqs, positions + [0] * spare, slots + [-1] * spare]
    types = 2 * [torch.int32, torch.int32, torch.int32, torch.int64] + 4 * [torch.int32]
    return [torch.tensor(x, dtype=t) for x, t in zip(results + [table, held, free[:-1], [count]], types)]


def _exact_rope(s):
    c = s.case

    def heads(x, weight):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + weight.double())
        if c["rot"]:
            half = c["rot"] // 2
            first = torch.arange(0, c["rot"], 2) if c["interleaved"] else torch.arange(half)
            second = first + (1 if c["interleaved"] else half)
            turn = torch.polar(torch.full((1, half), s.factor, dtype=torch.float64, device=x.device),
                               s.positions.double()[:, None] * s.inv_freq.double())
            z = torch.complex(x[..., first], x[..., second]) * turn[:, None, :]
            x[..., first], x[..., second] = z.real, z.imag
        return x

    q, k = heads(s.q, s.q_weight), heads(s.k, s.k_weight)
    if not c["store"]:
        return q, k
    k_cache, v_cache = s.k_cache.double(), s.v_cache.double()
    stored = int((s.slots >= 0).sum())                       # the others stand at the end
    at = s.slots[:stored]
    k_cache.view(-1, c["HKV"], c["D"])[at] = k[:stored]
    v_cache.view(-1, c["HKV"], c["D"])[at] = s.v[:stored].double()
    return q, k_cache, v_cache


def _exact_attention(s):
    c = s.case
    G, bs = c["HQ"] // c["HKV"], c["block"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=s.q.device)
    token = 0
    for n, (length, window) in enumerate(_attention_lengths(c)):
        if window == 0 or length == 0:
            token += window
            continue
        at = torch.arange(length, device=s.q.device)
        page = s.table[n].long()[at // bs]
        for h in range(c["HKV"]):
            k, v = (x[page, at % bs, h].double() for x in (s.k_cache, s.v_cache))
            for j in range(window):
                sees = length - window + j + 1
                q = s.q[token + j, h * G:(h + 1) * G].double()
                p = torch.softmax(q @ k[:sees].t().contiguous() * s.scale, dim=-1)
                out[token + j, h * G:(h + 1) * G] = p @ v[:sees]
        token += window
    return out if s.gate is None else out * torch.sigmoid(s.gate.double())


def exact(case, seed):
    # about as many products of a matrix with a few rows as take twenty seconds
    if case["op"] == "attention" and case["batch"] * case["HKV"] * case["window"] > 40000:
        return None
    return {"plan": _exact_plan, "rope": _exact_rope, "attention": _exact_attention}[case["op"]](prepare(case, seed))
