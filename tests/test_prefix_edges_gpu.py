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
