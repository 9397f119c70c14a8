"""Prompts cut into as many pieces as their keys allow, at the lengths where one more begins."""
import pytest

from test_prompt_attention_gpu import _check_packed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D, act, HQ, HKV", [(128, "bf16", 16, 2), (64, "fp16", 4, 1), (256, "bf16", 8, 8)])
@pytest.mark.parametrize("keys", [1024, 1025, 1088, 1089, 1536, 1537, 1600, 1601, 2561])
def test_every_piece_has_room(D, act, HQ, HKV, keys):
    for tokens in (1, 17, 130):
        _check_packed([tokens], HQ, HKV, D, act, keys=[keys], seed=keys)
    _check_packed([1, 0, 30, 1], HQ, HKV, D, act, keys=[keys, 5, 513, 577], seed=keys)
    _check_packed([1] * 40 + [keys - 39], HQ, HKV, D, act, seed=keys)
