"""Workspace of prompts whose keys are too few for the pieces that the chip could take."""
import pytest

from pla_amd import _lib


@pytest.mark.parametrize("batch, tokens, HQ, HKV, D, keys", [(12, 1200, 16, 2, 128, 1200), (1, 1, 4, 1, 64, 1025), (5, 600, 16, 2, 128, 1088), (20, 1500, 8, 8, 256, 1500)])
def test_no_more_than_the_keys_can_be_cut_into(batch, tokens, HQ, HKV, D, keys):
    rows = tokens * (HQ // HKV)
    blocks = min(rows // 128 + batch, rows)
    items = blocks + blocks * ((-(-keys // 64) - 1) // 8)     # a piece has at least eight tiles of 64 keys
    slots = items * HKV * min(rows, 128)
    most = slots * (4 * D + 8) + items * 48                   # outputs, maxima and sums; the list
    size = _lib.load().pla_prompt_attention_workspace_bytes(batch, tokens, HQ, HKV, D, keys)
    assert 0 < size <= most + 3 * 256


def test_more_keys_never_take_less():
    size = _lib.load().pla_prompt_attention_workspace_bytes
    sizes = [size(12, 1200, 16, 2, 128, keys) for keys in (1200, 2000, 30000, 2 ** 30, 2 ** 31, 2 ** 32 + 70, 2 ** 40)]
    assert sizes == sorted(sizes) and sizes[0] < sizes[1]
