"""Paged caches of 8-bit numbers, written and read, and a prefix that all requests of a batch share, against plain implementations in 64 bits."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _offsets(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


# ---- written -----------------------------------------------------------------------------------------------------

def _turned(x, weight, positions, inv_freq, *, eps, offset, factor, interleaved):
    """Norm and rotation in 64 bits."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (weight.double() + offset)
    if inv_freq is not None:
        half = inv_freq.numel()
        first = torch.arange(0, 2 * half, 2) if interleaved else torch.arange(half)
        second = first + (1 if interleaved else half)
        angle = positions.double()[:, None, None] * inv_freq.double()
        a, b = x[..., first], x[..., second]
        x = x.clone()
        x[..., first], x[..., second] = (a * angle.cos() - b * angle.sin()) * factor, (b * angle.cos() + a * angle.sin()) * factor
    return x


def _check_stored(cache, scales, slots, want):
    """Numbers and scales at the tokens' slots.  The 32-bit arithmetic before moves a channel by at most 2^-18 of its head's largest (tens of
    roundings of 2^-24 and angles to 2^-22); a scale by that and two roundings; a number by half a step, 2^-4 of itself or half of the
    smallest, 2^-10, from there."""
    bs, HKV, D = cache.shape[1:]
    kept = (slots >= 0) & (slots < cache.size(0) * bs)
    at = slots[kept]
    got = cache.view(torch.uint8)[at // bs, at % bs].view(E4M3).double()
    scale = scales[at // bs, :, at % bs].double()
    want = want[kept]
    top = want.abs().amax(-1).clamp(min=1e-30)
    torch.testing.assert_close(scale, top / 448, rtol=2 ** -17, atol=0)
    assert got.abs().amax() <= 448
    room = want.abs() * (2 ** -4 + 2 ** -16) + scale[..., None] * 2 ** -10 + top[..., None] * 2 ** -17
    assert ((got * scale[..., None] - want).abs() <= room).all()
    # the largest has the largest number
    assert (got.abs().amax(-1)[top > 1e-20] == 448).all()


@pytest.mark.parametrize("T, HQ, HKV, D, rot, interleaved, norm, act, bs", [
    (1, 1, 1, 64, 64, False, True, "bf16", 16), (8, 16, 2, 128, 128, False, True, "bf16", 16), (37, 10, 10, 64, 0, False, True, "fp16", 64),
    (130, 16, 1, 256, 64, True, True, "fp16", 80), (300, 8, 8, 128, 64, True, False, "bf16", 16), (1500, 32, 8, 128, 128, False, True, "bf16", 528),
    (700, 5, 5, 256, 256, False, False, "fp16", 16), (9000, 8, 3, 128, 32, False, True, "fp16", 32), (2500, 40, 20, 64, 64, False, True, "bf16", 48)])
def test_norm_rotation_and_store_in_8_bits(T, HQ, HKV, D, rot, interleaved, norm, act, bs):
    from pla.decode.paged import fused_qk_norm_rope
    dtype = DTYPES[act]
    row = _randn(T, T, (HQ + 2 * HKV) * D, dtype=dtype)
    q, k, v = (x.view(T, -1, D) for x in row.split([HQ * D, HKV * D, HKV * D], 1))
    k[:, :, 3] *= 20                                         # heads of very different magnitudes
    v[T // 2] *= 1e-3
    v[T // 3, 0] = 0
    wq, wk = (_randn(2, D, dtype=dtype, scale=0.1), _randn(3, D, dtype=dtype, scale=0.1)) if norm else (None, None)
    positions = torch.randint(0, 1 << 20, (T,), device=DEV) if rot else None
    inv_freq = (1e6 ** -(torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().to(DEV) if rot else None
    blocks = -(-T // bs) + 2
    k_cache, v_cache = (torch.full((blocks, bs, HKV, D), 7, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2))
    scales = torch.full((blocks, 2, HKV, -(-bs // 4) * 4 + 4), 5.0, device=DEV)
    k_scales, v_scales = scales[:, 0, :, :bs], scales[:, 1, :, :bs]
    slots = torch.randperm(blocks * bs, device=DEV)[:T]
    slots[T - T // 8:] = -1
    if T > 100:
        slots[4] = blocks * bs
    options = dict(q_weight=wq, k_weight=wk, eps=1e-6, weight_offset=1.0, inv_freq=inv_freq, attention_factor=1.1, interleaved=interleaved)
    k_out = torch.empty_like(k) if T % 2 else None
    q_out, same = fused_qk_norm_rope(q, k, positions, v=v, k_cache=k_cache, v_cache=v_cache, slot_mapping=slots, k_scales=k_scales, v_scales=v_scales,
                                     k_out=k_out, **options)
    assert same is k_out
    want = dict(eps=1e-6, offset=1.0, factor=1.1, interleaved=interleaved)
    _check_stored(k_cache, k_scales, slots, _turned(k, wk, positions, inv_freq, **want))
    _check_stored(v_cache, v_scales, slots, v.double())
    # everything else is as in the 16-bit call, and what is not written stays
    plain_q, plain_k = fused_qk_norm_rope(q, k, positions, **options)
    assert torch.equal(q_out, plain_q) and (k_out is None or torch.equal(k_out, plain_k))
    untouched = torch.ones(blocks * bs, dtype=torch.bool, device=DEV)
    untouched[slots[(slots >= 0) & (slots < blocks * bs)]] = False
    at = untouched.nonzero().flatten()
    for cache, x in ((k_cache, k_scales), (v_cache, v_scales)):
        assert (cache.view(torch.uint8)[at // bs, at % bs] == 7).all() and (x[at // bs, :, at % bs] == 5).all()
    assert (scales[:, :, :, bs:] == 5).all()


def test_keys_alone_and_values_that_are_not_finite():
    from pla.decode.paged import fused_qk_norm_rope
    q, k, v = (_randn(i, 6, 2, 64, dtype=torch.bfloat16) for i in range(3))
    k[1, 0, 5] = math.nan
    k[2, 1, 6] = math.inf
    k[3, 0] = math.nan
    cache = torch.zeros(1, 16, 2, 64, device=DEV).to(E4M3)
    scales = torch.zeros(1, 2, 16, device=DEV)
    slots = torch.arange(6, device=DEV)
    fused_qk_norm_rope(q, k, k_cache=cache, slot_mapping=slots, k_scales=scales)
    stands = cache[0, :6].float() * scales[0, :, :6].t()[..., None]
    bad = torch.zeros(6, 2, 64, dtype=torch.bool, device=DEV)
    bad[1, 0, 5] = bad[2, 1] = bad[3, 0] = True
    assert torch.equal(torch.isnan(stands), bad)
    assert ((stands - k.float()).abs() <= k.float().abs() * (2 ** -4 + 2 ** -10) + scales[0, :, :6].t()[..., None] * 2 ** -10)[~bad].all()


# ---- read --------------------------------------------------------------------------------------------------------

class _Cache8:
    """Caches whose every place outside of the sequences holds NaN, in numbers and scales."""

    def __init__(self, lengths, HKV, D, bs, *, seed=0, heads_first=False):
        pages = [-(-n // bs) for n in lengths]
        total, cols = sum(pages) + 2, max(pages + [1]) + 1
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
        store = torch.full((total, 2, HKV, bs, D) if heads_first else (total, 2, bs, HKV, D), 127, dtype=torch.uint8, device=DEV)
        self.bytes = [store[:, i].transpose(1, 2) if heads_first else store[:, i] for i in range(2)]
        self.scales = [torch.full((total, HKV, bs), math.nan, device=DEV) for _ in range(2)]
        self.table = torch.full((len(lengths), cols), -7, dtype=torch.int32)
        self.values, at = [[], []], 0
        for n, (length, count) in enumerate(zip(lengths, pages)):
            mine = order[at:at + count]
            at += count
            self.table[n, :count] = torch.tensor(mine, dtype=torch.int32)
            p = torch.arange(length, device=DEV)
            block = _ints(mine, torch.int64)[p // bs] if count else p
            for i in range(2):
                code = _randn(seed + 10 * n + i, length, HKV, D, scale=100.0).clamp(-448, 448).to(E4M3)
                scale = torch.rand(length, HKV, device=DEV, generator=torch.Generator(device=DEV).manual_seed(n + i)) * 0.02 + 1e-3
                self.bytes[i][block, p % bs] = code.view(torch.uint8)
                self.scales[i][block, :, p % bs] = scale
                self.values[i].append(code.double() * scale.double()[..., None])
        self.table = self.table.to(DEV)

    @property
    def args(self):
        return dict(k_cache=self.bytes[0].view(E4M3), v_cache=self.bytes[1].view(E4M3), block_table=self.table, k_scales=self.scales[0], v_scales=self.scales[1])


def _rows_reference(q, k, v, scale, parts):
    """(outputs, error) of tokens [m, HQ, D] over k, v [n, HKV, D] in 64 bits; `parts`: relative error of the weights of each key."""
    m, HQ, D = q.shape
    n, HKV = k.shape[:2]
    out, slack = torch.zeros(m, HQ, D, dtype=torch.float64, device=DEV), torch.zeros(m, HQ, D, dtype=torch.float64, device=DEV)
    if m == 0 or n == 0:
        return out, slack
    seen = torch.arange(n, device=DEV)[None, :] <= torch.arange(n - m, n, device=DEV)[:, None]
    some = seen.any(1)
    for h in range(HQ):
        x, y, z = q[:, h].double(), k[:, h * HKV // HQ].double(), v[:, h * HKV // HQ].double()
        score = (x @ y.t().contiguous()) * scale
        # products are exact in 32 bits, sums of D off by D 2^-24 of the sizes, factors, argument and value of the exponential by 2^-24 and 2^-22
        wrong = ((x.abs() @ y.abs().t().contiguous()) * abs(scale) * D + 6 * score.abs().masked_fill(~seen, 0).amax(1, keepdim=True)) * 2.0 ** -24 + 2.0 ** -22
        w = torch.softmax(score.masked_fill(~seen, -1e300), 1) * some[:, None]
        out[:, h] = w @ z
        slack[:, h] = (w * (parts + 2 * wrong + (n + 32) * 2.0 ** -24)) @ z.abs() + n * 2.0 ** -37 * z.abs().amax(0)
    return out, slack


def _close(got, ref, slack, gate=None):
    if gate is not None:
        g = torch.sigmoid(gate.double())
        ref, slack = ref * g, slack * g + (ref * g).abs() * 2.0 ** -20
    eps = torch.finfo(got.dtype).eps / 2
    room = slack + eps * (ref.abs() + slack) + torch.finfo(got.dtype).smallest_normal * eps
    worst = ((got.double() - ref).abs() / room).max().item() if got.numel() else 0.0
    assert worst <= 1, worst


TWO_PARTS = 2.0 ** -15                                       # of bf16: 2^-16, and the error of a factor


@pytest.fixture(params=[0, 160], ids=["together", "alone"])
def crowd(request):
    """Requests without a window behind those of a call: of many runs wavefronts have runs of their own."""
    return request.param


def _decode8(cache, q, lengths, windows, crowd, **more):
    from pla.decode.paged import paged_attention_decode
    offsets = _offsets(windows) + [sum(windows)] * crowd
    rows = list(range(len(lengths))) + [0] * crowd
    return paged_attention_decode(q, seq_lens=_ints(list(lengths) + [9] * crowd), query_start_loc=_ints(offsets), request_indices=_ints(rows),
                                  max_query_len=max(windows), **cache.args, **more)


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 255, 257, 500]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("act", ["bf16", "fp16"])
@pytest.mark.parametrize("HQ, HKV, bs, heads_first, gated", [(1, 1, 16, False, False), (8, 2, 32, True, True), (7, 1, 48, False, False), (40, 2, 16, True, False)])
def test_one_new_token_over_8_bits(D, act, HQ, HKV, bs, heads_first, gated, crowd):
    cache = _Cache8(EDGES, HKV, D, bs, seed=D + HQ, heads_first=heads_first)
    q = _randn(HQ, len(EDGES), HQ, D, dtype=DTYPES[act], scale=2.0)
    gate = _randn(3, len(EDGES), HQ, D, dtype=DTYPES[act]) if gated else None
    out = _decode8(cache, q, EDGES, [1] * len(EDGES), crowd, output_gate=gate)
    for n in range(len(EDGES)):
        _close(out[n:n + 1], *_rows_reference(q[n:n + 1], cache.values[0][n], cache.values[1][n], D ** -0.5, TWO_PARTS), None if gate is None else gate[n:n + 1])
    assert (out[0] == 0).all()


@pytest.mark.parametrize("D, act, HQ, HKV, window", [(64, "fp16", 4, 4, 8), (128, "bf16", 16, 2, 4), (128, "fp16", 6, 2, 32), (256, "bf16", 8, 1, 32), (256, "fp16", 3, 1, 5),
                                                     (64, "bf16", 16, 1, 17), (128, "bf16", 12, 1, 3), (64, "bf16", 8, 1, 4)])
def test_windows_over_8_bits(D, act, HQ, HKV, window, crowd):
    rng = random.Random(D + window)
    windows = [rng.randint(0, window) for _ in range(12)] + [window, 1, window]
    lengths = [0, 1, 2, window, 16, 17, 33, 127, 128, 129, 160, 200, 1300, 2000, 2049]
    cache = _Cache8(lengths, HKV, D, 16, seed=window)
    T = sum(windows)
    q = _randn(7, T + 3, HQ, D, dtype=DTYPES[act], scale=1.5)
    out = torch.full_like(q, 5.0)
    _decode8(cache, q, lengths, windows, crowd, out=out)
    a = 0
    for n, m in enumerate(windows):
        _close(out[a:a + m], *_rows_reference(q[a:a + m], cache.values[0][n], cache.values[1][n], D ** -0.5, TWO_PARTS))
        a += m
    assert (out[T:] == 5).all()


@pytest.mark.parametrize("D, act, HQ, HKV, bs", [(128, "bf16", 16, 2, 16), (64, "fp16", 2, 2, 64), (256, "bf16", 16, 1, 528)])
def test_a_long_request_over_8_bits_is_split_and_joined(D, act, HQ, HKV, bs, crowd):
    lengths = [9000, 5, 40000, 130, 700]
    cache = _Cache8(lengths, HKV, D, bs, seed=1)
    q = _randn(7, 5, HQ, D, dtype=DTYPES[act], scale=1.5)
    out = _decode8(cache, q, lengths, [1] * 5, crowd)
    for n in range(5):
        _close(out[n:n + 1], *_rows_reference(q[n:n + 1], cache.values[0][n], cache.values[1][n], D ** -0.5, TWO_PARTS))


@pytest.mark.parametrize("D, act, HQ, HKV", [(64, "bf16", 4, 4), (128, "fp16", 8, 2), (256, "bf16", 4, 1)])
@pytest.mark.parametrize("what", ["key", "value", "key scale", "value scale"])
def test_later_tokens_that_are_nan_do_not_reach_the_ones_before(D, act, HQ, HKV, what, crowd):
    lengths, windows = [70, 300], [4, 6]
    cache = _Cache8(lengths, HKV, D, 16, seed=4)
    q = _randn(7, 10, HQ, D, dtype=DTYPES[act], scale=1.5)
    sane = _decode8(cache, q, lengths, windows, crowd)
    for n, p in ((0, 68), (1, 297)):                         # the last two tokens of the first window, the last three of the second
        block, place = cache.table[n, p // 16].item(), p % 16
        i = 0 if what.startswith("key") else 1
        if what.endswith("scale"):
            cache.scales[i][block, :, place] = math.nan
        else:
            cache.bytes[i][block, place, :, 11] = 127
    got = _decode8(cache, q, lengths, windows, crowd)
    reached = [False, False, True, True] + [False, False, False, True, True, True]
    for row, nan in enumerate(reached):
        if not nan:
            torch.testing.assert_close(got[row].float(), sane[row].float(), rtol=2 * torch.finfo(q.dtype).eps, atol=1e-6)
        elif what == "value":
            assert torch.isnan(got[row, :, 11]).all() and torch.isfinite(got[row, :, :11]).all() and torch.isfinite(got[row, :, 12:]).all()
        else:
            assert torch.isnan(got[row]).all()


def test_what_is_written_is_read():
    """Plan, store and attention of a few steps over one cache, 8 bits next to 16."""
    from pla.decode.paged import PagedKVBlocks, fused_qk_norm_rope, paged_attention_decode, paged_kv_plan, rotary_frequencies
    N, HQ, HKV, D, bs = 5, 8, 2, 128, 16
    pool = PagedKVBlocks.allocate(200, bs, N, 40, DEV)
    inv_freq, factor = rotary_frequencies(64, device=DEV)
    w = _randn(1, D, dtype=torch.bfloat16, scale=0.1)
    c8 = [torch.zeros(200, bs, HKV, D, device=DEV).to(E4M3) for _ in range(2)]
    s8 = [torch.zeros(200, HKV, bs, device=DEV) for _ in range(2)]
    c16 = [torch.zeros(200, bs, HKV, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    context = [0] * N
    for step, new in enumerate(([32, 7, 1, 20, 31], [1] * N, [4, 2, 0, 1, 3], [1] * N)):
        T = sum(new)
        plan = paged_kv_plan(pool, _ints(context), _ints(new), token_capacity=T + 2)
        q, k, v = _randn(step, T + 2, HQ, D, dtype=torch.bfloat16), _randn(step + 9, T + 2, HKV, D, dtype=torch.bfloat16), _randn(step + 5, T + 2, HKV, D, dtype=torch.bfloat16)
        turn = dict(q_weight=w, k_weight=w, weight_offset=1.0, inv_freq=inv_freq, attention_factor=factor, v=v, slot_mapping=plan.slot_mapping)
        q8, _ = fused_qk_norm_rope(q, k, plan.positions, k_cache=c8[0], v_cache=c8[1], k_scales=s8[0], v_scales=s8[1], **turn)
        q16, _ = fused_qk_norm_rope(q, k, plan.positions, k_cache=c16[0], v_cache=c16[1], **turn)
        assert torch.equal(q8, q16)
        see = dict(query_start_loc=plan.query_start_loc, max_query_len=32)
        a = paged_attention_decode(q8, c8[0], c8[1], pool.block_table, plan.seq_lens, k_scales=s8[0], v_scales=s8[1], **see)[:T].float()
        b = paged_attention_decode(q16, c16[0], c16[1], pool.block_table, plan.seq_lens, **see)[:T].float()
        # numbers of 8 bits are off by up to 2^-4 each: by half of that on the whole
        assert (a - b).norm() <= 2 ** -4 * b.norm()
        context = [c + n for c, n in zip(context, new)]


def test_captured_stores_and_reads_of_8_bits():
    """Two graphs of a step (store, then attention) on two streams, replayed over other slots and lengths."""
    from pla.decode.paged import fused_qk_norm_rope, paged_attention_decode
    N, HQ, HKV, D, bs, pages = 6, 8, 2, 128, 16, 80
    table = torch.randperm(N * pages, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(torch.int32).view(N, pages)
    steps = []
    for g in range(2):
        caches = [torch.randint(0, 120, (N * pages, bs, HKV, D), dtype=torch.uint8, device=DEV, generator=torch.Generator(device=DEV).manual_seed(g)).view(E4M3) for _ in range(2)]
        scales = [torch.rand(N * pages, HKV, bs, device=DEV) * 0.01 for _ in range(2)]
        q, k, v = _randn(g, N, HQ, D, dtype=torch.bfloat16), _randn(g + 4, N, HKV, D, dtype=torch.bfloat16), _randn(g + 8, N, HKV, D, dtype=torch.bfloat16)
        slots, lens, out = torch.full((N,), -1, dtype=torch.int64, device=DEV), torch.zeros(N, dtype=torch.int32, device=DEV), torch.zeros_like(q)

        def call(caches, scales, out, q=q, k=k, v=v, slots=slots, lens=lens):
            turned, _ = fused_qk_norm_rope(q, k, v=v, k_cache=caches[0], v_cache=caches[1], slot_mapping=slots, k_scales=scales[0], v_scales=scales[1])
            return paged_attention_decode(turned, caches[0], caches[1], table, lens, k_scales=scales[0], v_scales=scales[1], out=out)
        call(caches, scales, out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(caches, scales, out)
        steps.append((graph, torch.cuda.Stream(), caches, scales, slots, lens, out, call))
    for lengths in ([1, 2, 16, 17, 1200, 0], [1280, 1280, 3, 40, 900, 77], [0, 0, 0, 0, 0, 0], [33, 1000, 1000, 1, 7, 1279]):
        expected = []
        for graph, stream, caches, scales, slots, lens, out, call in steps:
            last = [(n, x - 1) for n, x in enumerate(lengths)]
            slots.copy_(torch.tensor([table[n, p // bs].item() * bs + p % bs if p >= 0 else -1 for n, p in last], device=DEV))
            lens.copy_(_ints(lengths))
            out.fill_(9.0)
            mine = [c.view(torch.uint8).clone().view(E4M3) for c in caches], [x.clone() for x in scales]
            expected.append((mine, call(*mine, torch.zeros_like(out))))
        torch.cuda.synchronize()
        for graph, stream, *_ in steps:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, caches, scales, _, _, out, _), (mine, ref) in zip(steps, expected):
            assert torch.equal(out, ref) and (out[[n for n, x in enumerate(lengths) if x == 0]] == 0).all()
            for a, b in zip(caches + scales, mine[0] + mine[1]):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_8_bits_past_32_bits():
    """The last blocks of a cache of more than 2^32 numbers against the same tokens in a small one, bit for bit."""
    from pla.decode.paged import fused_qk_norm_rope, paged_attention_decode
    N, HQ, HKV, D, bs, pages, far = 3, 16, 8, 128, 16, 30, 264_000
    q, k, v = (_randn(i, N * 16 * pages, h, D, dtype=torch.bfloat16) for i, h in ((1, HQ), (2, HKV), (3, HKV)))
    results = []
    for blocks, base in ((N * pages, 0), (far, far - N * pages)):
        caches = [torch.empty(blocks, bs, HKV, D, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2)]
        scales = [torch.empty(blocks, HKV, bs, device=DEV) for _ in range(2)]
        fused_qk_norm_rope(q, k, v=v, k_cache=caches[0], v_cache=caches[1], slot_mapping=torch.arange(N * 16 * pages, device=DEV) + base * bs, k_scales=scales[0], v_scales=scales[1])
        table = (torch.arange(N * pages, dtype=torch.int32, device=DEV) + base).view(N, pages)
        results.append([paged_attention_decode(q[:N * m], caches[0], caches[1], table, _ints([480, 77, 300]), query_start_loc=_ints([0, m, 2 * m, 3 * m]), max_query_len=m,
                                               k_scales=scales[0], v_scales=scales[1]) for m in (1, 4, 32)])
    assert far * bs * HKV * D > 2 ** 32
    for a, b in zip(*results):
        assert torch.equal(a, b) and a.isfinite().all()


def test_shared_memory_of_scales_is_refused():
    from pla.decode.paged import fused_qk_norm_rope, paged_attention_decode
    q, k, v = (_randn(i, 4, 2, 64, dtype=torch.bfloat16) for i in range(3))
    kc, vc = (torch.zeros(2, 16, 2, 64, device=DEV).to(E4M3) for _ in range(2))
    s = torch.zeros(2, 2, 16, device=DEV)
    args = dict(v=v, k_cache=kc, v_cache=vc, slot_mapping=torch.arange(4, device=DEV))
    with pytest.raises(RuntimeError, match="v_scales must not share memory with k_scales"):
        fused_qk_norm_rope(q, k, k_scales=s, v_scales=s, **args)
    with pytest.raises(RuntimeError, match="k_scales must not share memory with itself"):
        fused_qk_norm_rope(q, k, k_scales=s[:1].expand(2, 2, 16), v_scales=s, **args)
    out = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="out must not share memory with v_scales"):
        paged_attention_decode(q, kc, vc, _ints([[0]] * 4), _ints([1] * 4), k_scales=s, v_scales=out.view(torch.float32).view(-1)[:64].view(2, 2, 16), out=out)


# ---- shared prefixes ---------------------------------------------------------------------------------------------

def _cache16(lengths, HKV, D, bs, act, seed=0):
    """Caches of 16 bits with every other place NaN, their table, and the sequences' keys and values."""
    pages = [-(-n // bs) for n in lengths]
    total, cols = sum(pages) + 2, max(pages + [1]) + 1
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    caches = [torch.full((total, bs, HKV, D), math.nan, dtype=DTYPES[act], device=DEV) for _ in range(2)]
    table, kept, at = torch.full((len(lengths), cols), -7, dtype=torch.int32), [[], []], 0
    for n, (length, count) in enumerate(zip(lengths, pages)):
        mine = order[at:at + count]
        at += count
        table[n, :count] = torch.tensor(mine, dtype=torch.int32)
        p = torch.arange(length, device=DEV)
        for i in range(2):
            x = _randn(seed + 10 * n + i, length, HKV, D, dtype=DTYPES[act])
            if count:
                caches[i][_ints(mine, torch.int64)[p // bs], p % bs] = x
            kept[i].append(x)
    return caches, table.to(DEV), kept


def _check_prefix(q, got, kept, lengths, windows, prefix, scale, gate=None, n_prefix=None):
    """The last sequence of `kept` is the prefix.  Its weights are rounded once to q's type, the others' in two parts."""
    u = torch.finfo(q.dtype).eps / 2
    pk, pv = kept[0][-1][:prefix], kept[1][-1][:prefix]
    a = 0
    for n, (length, m) in enumerate(zip(lengths, windows)):
        if length >= m:
            k, v = torch.cat([pk, kept[0][n][:length]]), torch.cat([pv, kept[1][n][:length]])
            parts = torch.cat([torch.full((prefix,), u * (1 + 2 * u), dtype=torch.float64, device=DEV), torch.full((length,), TWO_PARTS, dtype=torch.float64, device=DEV)])
            _close(got[a:a + m], *_rows_reference(q[a:a + m], k, v, scale, parts), None if gate is None else gate[a:a + m])
        a += m


@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 500, 4001])
@pytest.mark.parametrize("D, act, HQ, HKV, bs, window, gated", [(128, "bf16", 8, 2, 16, 1, False), (64, "fp16", 4, 4, 64, 4, True), (256, "bf16", 8, 1, 48, 3, True),
                                                                (128, "fp16", 7, 1, 528, 32, False), (64, "bf16", 16, 2, 16, 1, True), (256, "fp16", 2, 2, 16, 1, False)])
def test_windows_over_a_shared_prefix(prefix, D, act, HQ, HKV, bs, window, gated, crowd):
    from pla.decode.paged import paged_attention_decode
    rng = random.Random(prefix + D)
    lengths = [window, 500, 40, 129, 2000, window + 1, 64, 33]
    windows = [window] * len(lengths) if window == 1 else [window] + [rng.randint(0, window) for _ in lengths[1:]]
    lengths = [max(a, w) for a, w in zip(lengths, windows)]
    caches, table, kept = _cache16(lengths + [prefix], HKV, D, bs, act, seed=D)
    pages = -(-prefix // bs)
    T = sum(windows)
    q = _randn(5, T + 2, HQ, D, dtype=DTYPES[act], scale=1.5)
    gate = _randn(6, T + 2, HQ, D, dtype=DTYPES[act]) if gated else None
    out = torch.full_like(q, 5.0)
    paged_attention_decode(q, caches[0], caches[1], table[:-1], _ints(lengths + [9] * crowd), query_start_loc=_ints(_offsets(windows) + [T] * crowd),
                           request_indices=_ints(list(range(len(lengths))) + [0] * crowd), max_query_len=window, output_gate=gate, out=out,
                           prefix_blocks=table[-1, :pages].contiguous(), prefix_len=_ints([prefix], torch.int64))
    _check_prefix(q, out, kept, lengths, windows, prefix, D ** -0.5, gate)
    assert (out[T:] == 5).all()


def test_large_batches_over_a_long_prefix():
    from pla.decode.paged import paged_attention_decode
    for N, HQ, HKV, D, act, prefix, window in ((300, 8, 2, 64, "bf16", 9000, 1), (70, 32, 8, 128, "bf16", 3000, 4), (3, 16, 1, 256, "fp16", 20000, 1), (1, 4, 4, 128, "fp16", 30000, 1)):
        lengths = [window + 13 * n % 300 for n in range(N)]
        caches, table, kept = _cache16(lengths + [prefix], HKV, D, 16, act, seed=N)
        q = _randn(5, N * window, HQ, D, dtype=DTYPES[act], scale=1.5)
        got = paged_attention_decode(q, caches[0], caches[1], table[:-1], _ints(lengths), query_start_loc=_ints(_offsets([window] * N)), max_query_len=window,
                                     prefix_blocks=table[-1, :-(-prefix // 16)].contiguous(), prefix_len=_ints([prefix]))
        _check_prefix(q, got, kept, lengths, [window] * N, prefix, D ** -0.5)


def test_prefix_lengths_blocks_and_rows_out_of_range():
    from pla.decode.paged import paged_attention_decode
    lengths, prefix = [50, 0, 20, 30], 200
    caches, table, kept = _cache16(lengths + [prefix], 2, 128, 16, "bf16")
    q = _randn(5, 4, 4, 128, dtype=torch.bfloat16)
    pages = table[-1, :13].contiguous()

    def call(n=_ints([prefix]), blocks=pages, **more):
        return paged_attention_decode(q, caches[0], caches[1], table[:-1], _ints(lengths), prefix_blocks=blocks, prefix_len=n, **more)
    got = call()
    assert (got[1] == 0).all()                               # a refused request has no part in the prefix
    _check_prefix(q, got, kept, lengths, [1] * 4, prefix, 128 ** -0.5)
    for n in (0, -5, -2 ** 40):
        plain = paged_attention_decode(q, caches[0], caches[1], table[:-1], _ints(lengths))
        assert torch.equal(call(_ints([n], torch.int64)), plain)
    assert torch.equal(call(_ints([0]), pages[:0]), plain) and torch.equal(call(_ints([77]), pages[:0]), plain)
    caches[0][pages[12].long(), 8:], caches[1][pages[12].long(), 8:] = 0.25, 0.5
    whole = [torch.cat([x[-1], torch.full((8, 2, 128), y, dtype=torch.bfloat16, device=DEV)]) for x, y in zip(kept, (0.25, 0.5))]
    _check_prefix(q, call(_ints([2 ** 40], torch.int64)), [kept[0][:-1] + whole[:1], kept[1][:-1] + whole[1:]], lengths, [1] * 4, 208, 128 ** -0.5)
    bad = pages.clone()
    bad[3], bad[12] = -1, caches[0].size(0)
    left = [torch.cat([x[-1][:48], x[-1][64:192]]) for x in kept]
    _check_prefix(q, call(blocks=bad), [kept[0][:-1] + left[:1], kept[1][:-1] + left[1:]], lengths, [1] * 4, 176, 128 ** -0.5)
    _check_prefix(q, call(scale=-0.2), kept, lengths, [1] * 4, prefix, -0.2)


def test_values_of_a_prefix_that_are_not_finite_reach_every_row_that_sees_it():
    from pla.decode.paged import paged_attention_decode
    lengths, prefix = [50, 0, 20], 200
    for value in (math.inf, -math.inf, math.nan):
        caches, table, kept = _cache16(lengths + [prefix], 1, 64, 16, "fp16")
        block, place = table[-1, 6].long(), 4
        caches[1][block, place, 0, 9] = value
        q = _randn(5, 3, 4, 64, dtype=torch.float16, scale=8.0)
        got = paged_attention_decode(q, caches[0], caches[1], table[:-1], _ints(lengths), prefix_blocks=table[-1, :13].contiguous(), prefix_len=_ints([prefix]))
        seen = got[[0, 2], :, 9]
        assert (torch.isnan(seen) if math.isnan(value) else seen == value).all()
        assert (got[1] == 0).all() and torch.isfinite(got[..., :9]).all() and torch.isfinite(got[..., 10:]).all()


def test_a_captured_step_replays_over_other_prefixes():
    from pla.decode.paged import paged_attention_decode
    lengths = [70, 9, 300]
    caches, table, kept = _cache16(lengths + [5000], 2, 128, 16, "bf16")
    q, out = _randn(5, 3, 8, 128, dtype=torch.bfloat16), torch.zeros(3, 8, 128, dtype=torch.bfloat16, device=DEV)
    seq, n, pages = _ints(lengths), _ints([5000]), table[-1, :313].contiguous()
    call = lambda o: paged_attention_decode(q, caches[0], caches[1], table[:-1], seq, prefix_blocks=pages, prefix_len=n, out=o)
    call(out)
    graphs = []
    for _ in range(2):                                       # two graphs, each with a workspace of its own
        o, graph = torch.zeros_like(out), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(o)
        graphs.append((graph, o, torch.cuda.Stream()))
    for prefix, own in ((5000, lengths), (0, [1, 0, 40]), (3, [70, 9, 0]), (1111, lengths)):
        n.copy_(_ints([prefix]))
        seq.copy_(_ints(own))
        for graph, o, stream in graphs:
            o.fill_(9.0)
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        eager = call(torch.zeros_like(out))
        for _, o, _ in graphs:
            assert torch.equal(o, eager)
        _check_prefix(q, eager, kept, own, [1] * 3, prefix, 128 ** -0.5)


def test_a_prompt_then_its_requests():
    """A text is taken in by the prompt operator and becomes the prefix of requests; their attention is that of prompts which begin with it."""
    from pla.decode.paged import paged_attention_decode
    from pla.prefill.attention import packed_attention_fwd
    HQ, HKV, D, prefix, own = 8, 2, 128, 700, [5, 40, 1]
    caches, table, kept = _cache16(own + [prefix], HKV, D, 16, "bf16")
    q = _randn(5, sum(own), HQ, D, dtype=torch.bfloat16)
    k, v = (torch.cat([y for n in range(3) for y in (x[-1], x[n])]) for x in kept)
    whole = packed_attention_fwd(q, k, v, _ints(_offsets(own)), cu_seqlens_k=_ints(_offsets(prefix + n for n in own)))
    last = torch.tensor(_offsets(own)[1:], device=DEV) - 1
    got = paged_attention_decode(q[last], caches[0], caches[1], table[:-1], _ints(own), prefix_blocks=table[-1, :44].contiguous(), prefix_len=_ints([prefix]))
    torch.testing.assert_close(got.float(), whole[last].float(), atol=2 ** -7, rtol=2 ** -6)
