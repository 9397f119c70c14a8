"""Shared prefixes and own keys whose scores or values are not finite, or are as large as the type, against plain forms in 64 bits."""
import math

import pytest
import torch

from test_paged_cache8_and_prefix_gpu import DEV, DTYPES, _cache16, _close, _ints, _offsets, _randn, _rows_reference, crowd  # noqa: F401

pytestmark = pytest.mark.gpu


def _call(q, caches, table, lengths, prefix, crowd, windows=None, **more):
    """The last row of the table is the prefix."""
    from pla.decode.paged import paged_attention_decode
    windows = [1] * len(lengths) if windows is None else windows
    return paged_attention_decode(q, caches[0], caches[1], table[:-1], _ints(list(lengths) + [9] * crowd),
                                  query_start_loc=_ints(_offsets(windows) + [sum(windows)] * crowd), request_indices=_ints(list(range(len(lengths))) + [0] * crowd),
                                  max_query_len=max(windows), prefix_blocks=table[-1, :-(-prefix // caches[0].size(1))].contiguous(),
                                  prefix_len=_ints([prefix]), **more)


def _place(table, n, position, bs=16):
    return table[n, position // bs].long(), position % bs


SHAPES = [(128, "bf16", 8, 2), (64, "fp16", 4, 4), (256, "bf16", 8, 1), (128, "fp16", 7, 1), (64, "bf16", 16, 1)]


@pytest.mark.parametrize("D, act, HQ, HKV", SHAPES)
@pytest.mark.parametrize("prefix", [1, 200, 9000])
def test_keys_of_a_prefix_that_are_all_nan(D, act, HQ, HKV, prefix, crowd):
    lengths = [1, 50, 0, 7000]
    caches, table, _ = _cache16(lengths + [prefix], HKV, D, 16, act, seed=D)
    pages = table[-1, :-(-prefix // 16)].long()
    caches[0][pages] = math.nan
    q = _randn(5, 4, HQ, D, dtype=DTYPES[act], scale=1.5)
    got = _call(q, caches, table, lengths, prefix, crowd)
    assert torch.isnan(got[[0, 1, 3]]).all() and (got[2] == 0).all()
    if HKV > 1:                                              # of one key-value head alone
        caches, table, _ = _cache16(lengths + [prefix], HKV, D, 16, act, seed=D)
        caches[0][pages, :, 1] = math.nan
        got = _call(q, caches, table, lengths, prefix, crowd).view(4, HKV, HQ // HKV, D)
        assert torch.isnan(got[[0, 1, 3], 1]).all() and torch.isfinite(got[:, 0]).all() and torch.isfinite(got[:, 2:]).all()


@pytest.mark.parametrize("D, act, HQ, HKV", SHAPES)
@pytest.mark.parametrize("prefix", [1, 200, 9000])
def test_own_keys_whose_scores_are_all_minus_infinity(D, act, HQ, HKV, prefix, crowd):
    """Such a row sees keys of its own, all of weight zero: it is the attention over the prefix."""
    lengths, windows = [1, 40, 7000, 60, 20, 2, 300], [1, 3, 2, 1, 1, 4, 4]
    caches, table, kept = _cache16(lengths + [prefix], HKV, D, 16, act, seed=D)
    for n, length in enumerate(lengths):
        for page in range(-(-length // 16)):
            caches[0][table[n, page].long(), :, :, 0] = -math.inf
    block, place = _place(table, 6, 299)
    caches[0][block, place, :, 0] = 0.5                      # the last token of the last request sees another one
    table[3, 1:3] = caches[0].size(0)                        # some pages are missing,
    table[4, :2] = -1                                        # all pages are
    q = _randn(5, sum(windows), HQ, D, dtype=DTYPES[act], scale=1.5)
    q[..., 0] = 4.0
    got = _call(q, caches, table, lengths, prefix, crowd, windows)
    u = torch.finfo(q.dtype).eps / 2
    parts = torch.full((prefix,), u * (1 + 2 * u), dtype=torch.float64, device=DEV)
    first = _offsets(windows)
    zeros = [first[4], first[5], first[5] + 1]               # no pages; tokens before the first of their own
    for row in range(sum(windows) - 1):
        if row in zeros:
            assert (got[row] == 0).all(), row
        else:
            _close(got[row:row + 1], *_rows_reference(q[row:row + 1], kept[0][-1], kept[1][-1], D ** -0.5, parts))
    k, v = (torch.cat([kept[i][-1], caches[i][block, place][None]]) for i in range(2))
    parts = torch.cat([parts, torch.full((1,), 2.0 ** -15, dtype=torch.float64, device=DEV)])
    _close(got[-1:], *_rows_reference(q[-1:], k, v, D ** -0.5, parts))
    # without a prefix in sight as before: zeros
    assert (_call(q, caches, table, lengths, 0, crowd, windows)[:-1] == 0).all()


@pytest.mark.parametrize("D, HQ, HKV", [(128, 8, 2), (64, 4, 4), (256, 8, 1)])
@pytest.mark.parametrize("prefix, own, value", [(2, 1, 1.5e38), (500, 300, 6e35), (500, 300, -6e35), (9000, 7000, 2.5e34)])
def test_sums_of_prefix_and_own_keys_that_pass_32_bits_together(D, HQ, HKV, prefix, own, value, crowd):
    caches, table, _ = _cache16([own, prefix], HKV, D, 16, "bf16")
    for n, length in enumerate((own, prefix)):
        for page in range(-(-length // 16)):
            caches[1][table[n, page].long(), :, :, :D // 2] = value
            caches[1][table[n, page].long(), :, :, D // 2:] = 0.375
    q = torch.zeros(1, HQ, D, dtype=torch.bfloat16, device=DEV)
    got = _call(q, caches, table, [own], prefix, crowd).double()
    # equal weights of equal values: sums of n products, a division, one rounding
    want = torch.tensor(value, dtype=torch.bfloat16).item()
    assert ((got[..., :D // 2] - want).abs() <= abs(want) * (2 ** -8 + (prefix + own + 32) * 2 ** -24)).all()
    assert ((got[..., D // 2:] - 0.375).abs() <= 0.375 * (2 ** -8 + (prefix + own + 32) * 2 ** -24)).all()


@pytest.mark.parametrize("D, HQ, HKV", [(128, 8, 2), (64, 4, 4), (256, 8, 1)])
@pytest.mark.parametrize("prefix, own", [(3, 5), (700, 300), (9000, 7000)])
@pytest.mark.parametrize("far", ["prefix", "own"])
def test_large_values_under_weights_of_nothing(D, HQ, HKV, prefix, own, far, crowd):
    """Values of 1e38 under weights of exp(-300) are nothing beside ones of 1, infinite ones are infinite all the same."""
    caches, table, kept = _cache16([own, prefix], HKV, D, 16, "bf16", seed=3)
    q = _randn(5, 1, HQ, D, dtype=torch.bfloat16)
    q[..., 0] = 4.0
    n, length = (1, prefix) if far == "prefix" else (0, own)
    near = 1 - n
    pages = [table[i, :-(-x // 16)].long() for i, x in enumerate((own, prefix))]
    caches[0][pages[near], :, :, 0] = 75.0 * D ** 0.5        # 300 more than the others' scores
    caches[0][pages[n], :, :, 0] = 0.0
    kept[0][near][..., 0] = 75.0 * D ** 0.5
    sane = kept[1][near]
    if far == "prefix":
        caches[1][pages[n], :, :, 5] = 1e38
    else:                                                    # (own keys' sums are 32 bits wide, several such values pass them)
        block, place = _place(table, n, length // 2)
        caches[1][block, place, :, 5] = 1e38
    got = _call(q, caches, table, [own], prefix, crowd)
    u = 2.0 ** -8 * (1 + 2 ** -7)
    parts = torch.full((sane.size(0),), u, dtype=torch.float64, device=DEV)
    _close(got, *_rows_reference(q, kept[0][near], sane, D ** -0.5, parts))
    block, place = _place(table, n, length - 1)
    caches[1][block, place, :, 7] = -math.inf
    got = _call(q, caches, table, [own], prefix, crowd)
    assert (got[..., 7] == -math.inf).all() and torch.isfinite(got[..., :7]).all() and torch.isfinite(got[..., 8:]).all()


@pytest.mark.parametrize("D, act, HQ, HKV", SHAPES)
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_rows_of_no_request_may_hold_anything(D, act, HQ, HKV, value, crowd):
    lengths, windows, prefix = [50, 300, 1, 9], [2, 3, 1, 0], 4001
    caches, table, _ = _cache16(lengths + [prefix], HKV, D, 16, act, seed=D)
    q = _randn(5, 40, HQ, D, dtype=DTYPES[act], scale=1.5)
    sane = _call(q[:6], caches, table, lengths, prefix, crowd, windows)
    q[6:] = value
    out = torch.full_like(q, 5.0)
    _call(q, caches, table, lengths, prefix, crowd, windows, out=out)
    assert (out[6:] == 5).all()
    torch.testing.assert_close(out[:6].float(), sane.float(), atol=2 ** -7, rtol=2 ** -6)       # other pieces, so other roundings
