"""Causal attention of prompts, over dense keys and over a paged cache, against a plain implementation in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"


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


def _reference(q, k, v, scale, gate=None, there=None):
    """(outputs, size of the error that the kernel's arithmetic may have) of one sequence in 64 bits; q [m, HQ, D], k, v [n, HKV, D].

    A weight that is rounded by a relative u, but summed before it is, moves a result by at most u sum w |v|; an error e of a score
    by e sum w |v - o|, at most 2 e sum w |v|.  Scores: products are exact in 32 bits, their sum of D terms is off by at most D 2^-24 of
    the sum of the sizes, factor and argument of the exponential by 2^-24 of the score each (and of the running maximum, which is one of
    them), its value by 2^-22.  Sums over n keys in 32 bits, rescaled now and then: at most (n + 16) 2^-24 sum w |v|; one division, one
    product with the gate.  Weights in fp16 are scaled by 2^7 about a maximum that is at most 2^8 too small: below 2^-39 of the largest
    they are dropped."""
    m, HQ, D = q.shape
    n, HKV = k.shape[:2]
    u = torch.finfo(q.dtype).eps / 2
    out, slack = torch.zeros(m, HQ, D, dtype=torch.float64, device=DEV), torch.zeros(m, HQ, D, dtype=torch.float64, device=DEV)
    if m == 0 or n == 0:
        return out, slack
    seen = torch.arange(n, device=DEV)[None, :] <= torch.arange(n - m, n, device=DEV)[:, None]
    if there is not None:
        seen = seen & there[None, :]
    some = seen.any(1)
    for h in range(HQ):
        x, y, z = q[:, h].double(), k[:, h * HKV // HQ].double(), v[:, h * HKV // HQ].double()
        score = (x @ y.t().contiguous()) * scale
        wrong = ((x.abs() @ y.abs().t().contiguous()) * abs(scale) * D + 4 * score.abs().masked_fill(~seen, 0).amax(1, keepdim=True)) * 2.0 ** -24 + 2.0 ** -22
        w = torch.softmax(score.masked_fill(~seen, -1e300), 1) * some[:, None]
        o = w @ z
        size = (w * (u * (1 + 2 * u) + 2 * wrong)) @ z.abs() + (n + 16) * 2.0 ** -24 * (w @ z.abs())
        out[:, h] = o
        slack[:, h] = size + n * 2.0 ** -38 * z.abs().amax(0)
    if gate is not None:
        g = torch.sigmoid(gate.double())
        out, slack = out * g, slack * g + (out * g).abs() * 2.0 ** -20
    return out, slack


def _close(got, ref, slack):
    """Within the arithmetic's error and one rounding of the output (half a step, or half of the smallest number)."""
    eps = torch.finfo(got.dtype).eps / 2
    room = slack + eps * (ref.abs() + slack) + torch.finfo(got.dtype).smallest_normal * eps
    worst = ((got.double() - ref).abs() / room).max().item() if got.numel() else 0.0
    assert worst <= 1, worst


def _check_packed(lens, HQ, HKV, D, act, *, keys=None, gated=False, seed=0, scale=None, q_scale=1.5, wide=torch.int32, strided=False):
    from pla.prefill.attention import packed_attention_fwd
    dtype, T = DTYPES[act], sum(lens)
    key_lens = lens if keys is None else keys
    K = sum(key_lens)
    if strided:
        row = _randn(seed, max(T, K), (HQ + 2 * HKV) * D + 8, dtype=dtype)
        q = (row[:T, :HQ * D].view(T, HQ, D) * q_scale).to(dtype)
        k, v = (row[:K, i * D:(i + HKV) * D].view(K, HKV, D) for i in (HQ, HQ + HKV))
        out = torch.full((HQ, T, D + 8), 3.0, dtype=dtype, device=DEV).transpose(0, 1)[..., :D]
    else:
        q, k, v = _randn(seed, T, HQ, D, dtype=dtype, scale=q_scale), _randn(seed + 1, K, HKV, D, dtype=dtype), _randn(seed + 2, K, HKV, D, dtype=dtype)
        out = None
    gate = _randn(seed + 3, T, HQ, D, dtype=dtype, scale=2.0) if gated else None
    got = packed_attention_fwd(q, k, v, _ints(_offsets(lens), wide), cu_seqlens_k=None if keys is None else _ints(_offsets(keys), wide), scale=scale,
                               output_gate=gate, out=out)
    assert out is None or got is out
    a = b = 0
    for m, n in zip(lens, key_lens):
        ref, slack = _reference(q[a:a + m], k[b:b + n], v[b:b + n], D ** -0.5 if scale is None else scale, None if gate is None else gate[a:a + m])
        _close(got[a:a + m], ref, slack)
        a, b = a + m, b + n
    return q, k, v, got


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("act", ["bf16", "fp16"])
@pytest.mark.parametrize("HQ, HKV, gated, strided", [(1, 1, False, False), (8, 2, True, True), (7, 1, False, False), (40, 1, False, True), (10, 10, True, False)])
def test_short_prompts_of_every_length(D, act, HQ, HKV, gated, strided):
    _check_packed([0, 1, 2, 31, 0, 32, 33, 63, 64, 65, 127, 130, 257, 1, 0], HQ, HKV, D, act, gated=gated, strided=strided, seed=D + HQ)


@pytest.mark.parametrize("lens, HQ, HKV, D, act", [
    ([2500], 16, 2, 128, "bf16"), ([1], 16, 2, 64, "fp16"), ([1999, 3, 1000], 32, 8, 128, "fp16"), ([1537], 10, 10, 64, "bf16"), ([901, 2048], 8, 1, 256, "bf16"),
    ([40] * 150, 4, 4, 128, "bf16"), ([3, 0, 70, 1] * 90, 4, 1, 64, "fp16"), ([2] * 2100, 2, 1, 64, "bf16"), ([9, 0] * 150 + [1500], 8, 8, 128, "bf16"), ([777], 15, 3, 256, "fp16"), ([2100], 32, 32, 64, "fp16")])
def test_longer_prompts(lens, HQ, HKV, D, act):
    _check_packed(lens, HQ, HKV, D, act, seed=sum(lens), wide=torch.int64)


@pytest.mark.parametrize("D, act, HQ, HKV", [(128, "bf16", 8, 2), (64, "fp16", 5, 5), (256, "bf16", 4, 1)])
def test_earlier_keys_and_fewer_keys_than_tokens(D, act, HQ, HKV):
    _, _, _, got = _check_packed([5, 33, 1, 70, 9, 0, 4], HQ, HKV, D, act, keys=[900, 64, 5000, 70, 3, 77, 0], seed=D)
    assert (got[109:115] == 0).all() and (got[118:] == 0).all()           # tokens before the first key


@pytest.mark.parametrize("tokens, keys, HQ, HKV, D, act, gated", [
    (3, 20000, 16, 2, 128, "bf16", True), (1, 9000, 4, 1, 64, "fp16", False), (40, 16001, 8, 1, 256, "bf16", True), (200, 12345, 8, 4, 128, "fp16", False)])
def test_few_rows_over_many_keys_are_split_and_joined(tokens, keys, HQ, HKV, D, act, gated):
    from pla_amd import _lib
    assert _lib.load().pla_prompt_attention_workspace_bytes(1, tokens, HQ, HKV, D, keys) > 0
    _check_packed([tokens], HQ, HKV, D, act, keys=[keys], gated=gated, seed=keys)
    _check_packed([tokens, 1, tokens], HQ, HKV, D, act, keys=[keys, 70, 300], seed=keys)


@pytest.mark.parametrize("HQ, HKV, D, act", [(130, 1, 64, "bf16"), (300, 1, 128, "fp16"), (258, 2, 256, "bf16")])
def test_more_query_heads_than_rows_of_a_block(HQ, HKV, D, act):
    _check_packed([1, 70, 0, 3], HQ, HKV, D, act, gated=True, seed=HQ)
    _check_packed([2, 1], HQ, HKV, D, act, keys=[3000, 1], seed=HQ)


def test_nothing_to_do_and_no_keys_at_all():
    from pla.prefill.attention import packed_attention_fwd, paged_attention_prefill
    q, none = _randn(1, 5, 4, 128, dtype=torch.bfloat16), torch.empty(0, 2, 128, dtype=torch.bfloat16, device=DEV)
    assert (packed_attention_fwd(q, none, none, _ints([0, 2, 5]), cu_seqlens_k=_ints([0, 0, 0])) == 0).all()
    out = torch.full_like(q, 3.0)
    assert packed_attention_fwd(q, none, none, _ints([0]), cu_seqlens_k=_ints([0]), out=out) is out and (out == 3).all()
    assert packed_attention_fwd(q[:0], none, none, _ints([0, 0])).shape == (0, 4, 128)
    cache = _randn(2, 3, 16, 2, 128, dtype=torch.bfloat16)
    got = paged_attention_prefill(q, cache, cache, torch.zeros(2, 0, dtype=torch.int32, device=DEV), _ints([7, 3]), _ints([0, 2, 5]))
    assert (got == 0).all()                                               # no page of the table
    table = _ints([[0, 1], [2, 2]])
    paged_attention_prefill(q, cache, cache, table, _ints([]), _ints([0]), out=out)
    assert (out == 3).all()
    k = cache.view(48, 2, 128)
    got = paged_attention_prefill(q, cache, cache, table, _ints([20, 30, 18]), _ints([0, 2, 3, 5]), request_indices=_ints([0, 1, 0]))   # one row of the table twice
    keys = torch.cat([k[:20], k[32:], k[32:46], k[:18]])
    for (a, b), x in zip(((0, 2), (2, 3), (3, 5)), keys.split([20, 30, 18])):
        _close(got[a:b], *_reference(q[a:b], x, x, 128 ** -0.5))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-20, 3.0])
@pytest.mark.parametrize("act, D", [("bf16", 128), ("fp16", 64)])
def test_other_scales(scale, act, D):
    _check_packed([300, 5], 4, 2, D, act, scale=scale, seed=3)


def test_scores_that_rise_along_the_keys():
    """Every tile raises the maximum, some by more than a step that is not followed."""
    from pla.prefill.attention import packed_attention_fwd
    for act, D in (("bf16", 128), ("fp16", 64), ("fp16", 256)):
        T = 700
        q, k, v = _randn(1, T, 2, D, dtype=DTYPES[act]), _randn(2, T, 1, D, dtype=DTYPES[act]), _randn(3, T, 1, D, dtype=DTYPES[act])
        q[..., 0] = 4.0
        k[..., 0] = (torch.arange(T, device=DEV) * D ** 0.5 / 60).to(k.dtype)[:, None]
        got = packed_attention_fwd(q, k, v, _ints([0, T]))
        _close(got, *_reference(q, k, v, D ** -0.5))


@pytest.mark.parametrize("D, act", [(64, "bf16"), (128, "bf16"), (256, "bf16"), (128, "fp16")])
@pytest.mark.parametrize("tokens, keys", [(300, 300), (3, 9000)])
def test_the_largest_values(D, act, tokens, keys):
    """Values up to half of the type's largest, under weights and sums that pass FP32 with them where they are not scaled."""
    from pla.prefill.attention import packed_attention_fwd
    dtype = DTYPES[act]
    q, k, v = _randn(1, tokens, 4, D, dtype=dtype), _randn(2, keys, 2, D, dtype=dtype), (torch.tanh(_randn(3, keys, 2, D)) * torch.finfo(dtype).max / 2).to(dtype)
    q[..., 0] = 4.0
    k[..., 0] = (torch.arange(keys, device=DEV) % 300 * D ** 0.5 / 200).to(k.dtype)[:, None]
    k[keys // 3] = float("nan") if tokens == keys else 1.0                # an infinite sum next to a token that is not finite
    got = packed_attention_fwd(q, k, v, _ints([0, tokens]), cu_seqlens_k=_ints([0, keys]))
    first = keys // 3 if tokens == keys else tokens                       # rows before the token
    ref, slack = _reference(q[:first], k[:keys - tokens + first], v[:keys - tokens + first], D ** -0.5)
    _close(got[:first], ref, slack)
    assert got[first:].isnan().all()


def test_rows_of_no_sequence_and_sequences_that_are_passed_over():
    from pla.prefill.attention import packed_attention_fwd
    q, k, v = _randn(1, 50, 4, 128, dtype=torch.bfloat16), _randn(2, 50, 2, 128, dtype=torch.bfloat16), _randn(3, 50, 2, 128, dtype=torch.bfloat16)
    for bad in ([5, 20, 10, 51], [5, 20, -3, 20], [5, 20, 20, 1 << 40], [5, 20, 1 << 33, 3]):
        out = torch.full_like(q, 5.0)
        packed_attention_fwd(q, k, v, _ints(bad, torch.int64), out=out)
        _close(out[5:20], *_reference(q[5:20], k[5:20], v[5:20], 128 ** -0.5))
        others = [out[:5], out[20:]]
        assert all((x == 5).all() for x in others), bad
    out = torch.full_like(q, 5.0)
    packed_attention_fwd(q, k, v, _ints([0, 9, 20]), cu_seqlens_k=_ints([0, 40, 51]), out=out)
    assert (out[9:] == 5).all() and (out[:9] != 5).any()
    assert packed_attention_fwd(q[:0], k[:0], v[:0], _ints([0, 0])).shape == (0, 4, 128)
    assert (packed_attention_fwd(q, k[:0], v[:0], _ints([0, 20, 50]), cu_seqlens_k=_ints([0, 0, 0])) == 0).all()         # no keys at all
    packed_attention_fwd(q, k, v, _ints([0]), out=out)
    assert (out[9:] == 5).all()


@pytest.mark.parametrize("T, N", [(50, 40), (3000, 30), (600, 1500)])
def test_sequences_that_share_rows_stay_within_bounds(T, N):
    """Not a call to make, but one that ends: offsets go forth and back, so that sequences come to more row blocks than T and N allow."""
    from pla.prefill.attention import packed_attention_fwd
    q, k, v = _randn(1, T, 8, 64, dtype=torch.bfloat16), _randn(2, 9000, 2, 64, dtype=torch.bfloat16), _randn(3, 9000, 2, 64, dtype=torch.bfloat16)
    offsets, keys = [], []
    for n in range(N + 1):
        offsets.append(0 if n % 2 == 0 else T)
        keys.append(0 if n % 2 == 0 else 9000)
    out = torch.full_like(q, 5.0)
    packed_attention_fwd(q, k, v, _ints(offsets), cu_seqlens_k=_ints(keys), out=out)
    torch.cuda.synchronize()
    # the sequence (it is always the same one) that stands first has been taken
    _close(out[-1:], *_reference(q[-1:], k, v, 64 ** -0.5))


def _formula(q, k, v, scale):
    """The definition row by row in 64 bits, over what a row sees: infinite and NaN values as it has them, weights never zero."""
    m, HQ, D = q.shape
    n, HKV = k.shape[:2]
    out = torch.zeros(m, HQ, D, dtype=torch.float64, device=DEV)
    for j in range(m):
        sees = n - m + j + 1
        for h in range(HQ):
            score = (k[:sees, h * HKV // HQ].double() @ q[j, h].double()) * scale
            w = torch.softmax(score, 0).clamp(min=1e-300)
            out[j, h] = (w[:, None] * v[:sees, h * HKV // HQ].double()).sum(0)
    return out


@pytest.mark.parametrize("D, act, HQ, HKV", [(128, "bf16", 4, 2), (64, "fp16", 2, 2), (256, "bf16", 2, 1), (128, "fp16", 8, 1)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_tokens_that_are_not_finite_do_not_reach_the_ones_before(D, act, HQ, HKV, value):
    from pla.prefill.attention import packed_attention_fwd
    T = 150
    for tokens in ([0], [70], [149], [64, 65], [3, 100]):
        q, k, v = _randn(1, T, HQ, D, dtype=DTYPES[act]), _randn(2, T, HKV, D, dtype=DTYPES[act]), _randn(3, T, HKV, D, dtype=DTYPES[act])
        sane = packed_attention_fwd(q, k, v, _ints([0, T]))
        for i, t in enumerate(tokens):
            v[t, :, 5 + i] = value if i == 0 else -value
            v[t, 0, 40] = value if i == 0 else -value
        got = packed_attention_fwd(q, k, v, _ints([0, T]))
        ref = _formula(q, k, v, D ** -0.5)
        fine = torch.isfinite(ref)
        assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isposinf(got), torch.isposinf(ref))
        assert torch.equal(got[fine], sane[fine])
        # keys
        v[tokens] = 0.5
        k[tokens[-1]] = value
        got = packed_attention_fwd(q, k, v, _ints([0, T]))
        ref, slack = _reference(q[:tokens[-1]], k[:tokens[-1]], v[:tokens[-1]], D ** -0.5)
        _close(got[:tokens[-1]], ref, slack)


def test_an_infinite_value_counts_however_small_its_weight():
    from pla.prefill.attention import packed_attention_fwd
    q, k, v = _randn(1, 200, 2, 128, dtype=torch.bfloat16, scale=40.0), _randn(2, 200, 1, 128, dtype=torch.bfloat16, scale=4.0), _randn(3, 200, 1, 128, dtype=torch.bfloat16)
    v[10, 0, 7] = math.inf
    v[20, 0, 8] = -math.inf
    got = packed_attention_fwd(q, k, v, _ints([0, 200]))
    assert torch.isposinf(got[10:, :, 7]).all() and torch.isneginf(got[20:, :, 8]).all()
    assert torch.isfinite(got[:10]).all() and torch.isfinite(got[:, :, 9:]).all() and torch.isfinite(got[:, :, :7]).all()


# ---- paged -------------------------------------------------------------------------------------------------------

def _paged(lengths, HKV, D, bs, act, *, seed=0, heads_first=False, junk=math.nan):
    """Caches, table and the sequences' own keys and values; every other place holds ``junk``."""
    pages = [-(-n // bs) for n in lengths]
    total, cols = sum(pages) + 2, max(pages + [1]) + 1
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    store = torch.full((total, 2, HKV, bs, D) if heads_first else (total, 2, bs, HKV, D), junk, dtype=DTYPES[act], device=DEV)
    k_cache, v_cache = (store[:, i].transpose(1, 2) if heads_first else store[:, i] for i in range(2))
    table = torch.full((len(lengths), cols), -7, dtype=torch.int32)
    ks, vs, at = [], [], 0
    for n, (length, count) in enumerate(zip(lengths, pages)):
        mine = order[at:at + count]
        at += count
        table[n, :count] = torch.tensor(mine, dtype=torch.int32)
        k, v = (_randn(seed + 10 * n + i, length, HKV, D, dtype=DTYPES[act]) for i in range(2))
        ks.append(k)
        vs.append(v)
        p = torch.arange(length, device=DEV)
        block = _ints(mine, torch.int64)[p // bs] if count else p
        k_cache[block, p % bs], v_cache[block, p % bs] = k, v
    return k_cache, v_cache, table.to(DEV), ks, vs


@pytest.mark.parametrize("D, act, HQ, HKV, bs, heads_first, gated", [
    (128, "bf16", 8, 2, 16, False, True), (64, "fp16", 10, 10, 64, True, False), (256, "bf16", 16, 2, 48, False, False), (128, "fp16", 7, 1, 528, True, True),
    (64, "bf16", 16, 1, 32, False, False)])
def test_windows_of_any_length_over_a_paged_cache(D, act, HQ, HKV, bs, heads_first, gated):
    from pla.prefill.attention import paged_attention_prefill
    windows = [0, 1, 33, 64, 200, 5, 300, 17]
    lengths = [10, 900, 33, 65, 201, 4, 1300, 529]
    k_cache, v_cache, table, ks, vs = _paged(lengths, HKV, D, bs, act, seed=D, heads_first=heads_first)
    T = sum(windows)
    q = _randn(5, T + 3, HQ, D, dtype=DTYPES[act], scale=1.5)
    gate = _randn(6, T + 3, HQ, D, dtype=DTYPES[act]) if gated else None
    order = [3, 0, 7, 1, 2, 6, 5, 4]
    out = torch.full_like(q, 5.0)
    paged_attention_prefill(q, k_cache, v_cache, table, _ints([lengths[i] for i in order]), _ints(_offsets(windows[i] for i in order), torch.int64),
                            request_indices=_ints(order), output_gate=gate, out=out)
    a = 0
    for i in order:
        m = windows[i]
        ref, slack = _reference(q[a:a + m], ks[i], vs[i], D ** -0.5, None if gate is None else gate[a:a + m])
        _close(out[a:a + m], ref, slack)
        a += m
    assert (out[T:] == 5).all()


def test_agrees_with_the_decode_operator_on_its_windows():
    from pla.decode.paged import paged_attention_decode
    from pla.prefill.attention import paged_attention_prefill
    lengths, windows = [500, 77, 32], [8, 1, 32]
    k_cache, v_cache, table, _, _ = _paged(lengths, 2, 128, 16, "bf16")
    q = _randn(5, 41, 8, 128, dtype=torch.bfloat16)
    args = (q, k_cache, v_cache, table, _ints(lengths))
    a = paged_attention_prefill(*args, _ints(_offsets(windows)))
    b = paged_attention_decode(*args, query_start_loc=_ints(_offsets(windows)), max_query_len=32)
    torch.testing.assert_close(a.float(), b.float(), atol=2 ** -6, rtol=2 ** -6)


def test_positions_without_a_block_are_left_out():
    from pla.prefill.attention import paged_attention_prefill
    lengths, windows = [300, 100, 64, 50], [100, 60, 64, 50]
    k_cache, v_cache, table, ks, vs = _paged(lengths, 2, 64, 16, "bf16")
    bad = [(0, 0), (0, 11), (0, 18), (1, 6), (2, 0), (2, 1), (2, 2), (2, 3)]
    for n, page in bad:
        table[n, page] = k_cache.size(0) if page % 2 else -1
    q = _randn(5, sum(windows), 4, 64, dtype=torch.bfloat16)
    got = paged_attention_prefill(q, k_cache, v_cache, table, _ints(lengths), _ints(_offsets(windows)))
    a = 0
    for n, m in enumerate(windows):
        there = torch.tensor([(n, p // 16) not in bad for p in range(lengths[n])], device=DEV)
        _close(got[a:a + m], *_reference(q[a:a + m], ks[n], vs[n], 64 ** -0.5, there=there))
        a += m
    # a length past the table, a row that is none of it, nothing cached
    k_cache, v_cache, table, ks, vs = _paged([64, 64], 2, 64, 16, "bf16")
    got = paged_attention_prefill(q[:5], k_cache, v_cache, table[:1, :4], _ints([68]), _ints([0, 5]))
    _close(got, *_reference(q[:5], torch.cat([ks[0], ks[0][:4]]), torch.cat([vs[0], vs[0][:4]]), 64 ** -0.5, there=torch.arange(68, device=DEV) < 64))
    for lengths, rows in (([50], [9]), ([50], [-1]), ([0], [0]), ([-4], [0])):
        got = paged_attention_prefill(q[:50], k_cache, v_cache, table, _ints(lengths), _ints([0, 50]), request_indices=_ints(rows))
        assert (got == 0).all()


@pytest.mark.parametrize("D, act", [(128, "bf16"), (64, "fp16"), (256, "fp16")])
def test_offsets_past_32_bits(D, act):
    from pla.prefill.attention import packed_attention_fwd, paged_attention_prefill
    bs, HKV = 16, 2
    stride = 2 ** 31 // 40                                   # elements of a block, in a cache whose far blocks pass 2^31 elements and 2^32 bytes
    stride -= stride % 8
    store = torch.empty(60 * stride, dtype=DTYPES[act], device=DEV)
    k_cache = store.as_strided((60, bs, HKV, D), (stride, HKV * D, D, 1))
    v_cache = store.as_strided((60, bs, HKV, D), (stride, HKV * D, D, 1), bs * HKV * D)
    pages = _ints([59, 0, 57, 41, 58], torch.int32)
    k, v = _randn(1, 80, HKV, D, dtype=DTYPES[act]), _randn(2, 80, HKV, D, dtype=DTYPES[act])
    k_cache[pages.long()], v_cache[pages.long()] = k.view(5, bs, HKV, D), v.view(5, bs, HKV, D)
    q = _randn(3, 70, 4, D, dtype=DTYPES[act])
    got = paged_attention_prefill(q, k_cache, v_cache, pages[None], _ints([80]), _ints([0, 70]))
    _close(got, *_reference(q, k, v, D ** -0.5))
    # dense rows of a wide buffer
    wide = store.as_strided((190, HKV, D), ((1 << 24) - 8, D, 1))
    wide[40:110], wide[120:190] = k[:70], v[:70]
    got = packed_attention_fwd(q, wide[40:110], wide[120:190], _ints([0, 70]))
    _close(got, *_reference(q, k[:70], v[:70], D ** -0.5))


# ---- as a program uses them --------------------------------------------------------------------------------------

def test_captured_calls_replay_over_other_lengths():
    from pla.prefill.attention import packed_attention_fwd, paged_attention_prefill
    T, HQ, HKV, D = 400, 8, 2, 128
    q, k, v = _randn(1, T, HQ, D, dtype=torch.bfloat16), _randn(2, T, HKV, D, dtype=torch.bfloat16), _randn(3, T, HKV, D, dtype=torch.bfloat16)
    k_cache, v_cache, table, ks, vs = _paged([5000, 700], HKV, D, 16, "bf16")
    cu, lens = _ints([0, 100, 400]), _ints([5000, 700])
    out, paged_out = torch.zeros_like(q), torch.zeros_like(q)
    packed_attention_fwd(q, k, v, cu, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        packed_attention_fwd(q, k, v, cu, out=out)
        paged_attention_prefill(q, k_cache, v_cache, table, lens, cu, out=paged_out)
    for split, lengths in ((100, (5000, 700)), (1, (300, 650)), (400, (4999, 9)), (250, (260, 700))):
        cu.copy_(_ints([0, split, 400]))
        lens.copy_(_ints(lengths))
        out.fill_(7.0)
        paged_out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        a = 0
        for n, m in enumerate((split, 400 - split)):
            _close(out[a:a + m], *_reference(q[a:a + m], k[a:a + m], v[a:a + m], D ** -0.5))
            _close(paged_out[a:a + m], *_reference(q[a:a + m], ks[n][:lengths[n]], vs[n][:lengths[n]], D ** -0.5))
            a += m
        assert torch.equal(out, packed_attention_fwd(q, k, v, cu)) and torch.equal(paged_out, paged_attention_prefill(q, k_cache, v_cache, table, lens, cu))


def test_two_captured_graphs_and_two_streams_do_not_share_anything():
    from pla.prefill.attention import packed_attention_fwd
    sets = []
    for i in range(2):
        q, k, v = _randn(i, 30, 8, 128, dtype=torch.bfloat16), _randn(i + 5, 9000, 2, 128, dtype=torch.bfloat16), _randn(i + 9, 9000, 2, 128, dtype=torch.bfloat16)
        cu, ck = _ints([0, 30]), _ints([0, 9000])
        want, out = packed_attention_fwd(q, k, v, cu, cu_seqlens_k=ck), torch.zeros_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            packed_attention_fwd(q, k, v, cu, cu_seqlens_k=ck, out=out)
        sets.append((graph, out, want, torch.cuda.Stream(), (q, k, v, cu, ck)))
    for _ in range(5):
        for graph, out, _, stream, _ in sets:
            out.zero_()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _, _ in sets:
            assert torch.equal(out, want)


def test_shared_memory_is_refused():
    from pla.prefill.attention import packed_attention_fwd, paged_attention_prefill
    row = torch.zeros(20, 8, 64, dtype=torch.bfloat16, device=DEV)
    q, k, v, cu = row[:, :4], row[:, 4:6], row[:, 6:], _ints([0, 20])
    for out in (q, row[:, 2:6], row[:, 4:]):
        with pytest.raises(RuntimeError, match="must not share memory"):
            packed_attention_fwd(q, k, v, cu, out=out)
    with pytest.raises(RuntimeError, match="must not share memory with itself"):
        packed_attention_fwd(q, k, v, cu, out=torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV).expand(20, 4, 64))
    cache = torch.zeros(3, 2, 16, 2, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="must not share memory with k_cache"):
        paged_attention_prefill(q.contiguous(), cache[:, 0], cache[:, 1], _ints([[1, 2]]), _ints([20]), cu, out=cache.view(-1, 4, 64)[:20])
