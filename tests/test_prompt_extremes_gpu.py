"""Prompts whose values or scores are about as large as their type, against plain forms in 64 bits."""
import math

import pytest
import torch

from test_prompt_attention_gpu import DEV, DTYPES, _close, _ints, _randn, _reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("tokens, keys, value", [(3, 9000, 5e35), (3, 9000, -5e35), (40, 30000, 4e35), (1, 3000, 6e35)])
def test_pieces_whose_sums_pass_32_bits_together(D, tokens, keys, value):
    from pla.prefill.attention import packed_attention_fwd
    q, k, v = (torch.zeros(tokens if h == 4 else keys, h, D, dtype=torch.bfloat16, device=DEV) for h in (4, 2, 2))
    k.normal_()
    v[..., :D // 2], v[..., D // 2:] = value, 0.375
    got = packed_attention_fwd(q, k, v, _ints([0, tokens]), cu_seqlens_k=_ints([0, keys])).double()
    # equal weights of equal values: sums of n products, a division, one rounding
    for x, want in ((got[..., :D // 2], v[0, 0, 0].item()), (got[..., D // 2:], 0.375)):
        assert ((x - want).abs() <= abs(want) * (2 ** -8 + (keys + 32) * 2 ** -24)).all()


@pytest.mark.parametrize("D, act", [(64, "bf16"), (128, "bf16"), (256, "bf16"), (128, "fp16")])
@pytest.mark.parametrize("tokens, keys", [(300, 300), (3, 9000)])
def test_large_values_under_weights_of_nothing(D, act, tokens, keys):
    """Values of 1e38 (fp16: 60 000) under weights of exp(-300) are nothing beside ones of 1, infinite ones are infinite all the same."""
    from pla.prefill.attention import packed_attention_fwd
    dtype, first = DTYPES[act], 64 if tokens == keys else 700
    q, k, v = _randn(1, tokens, 4, D, dtype=dtype), _randn(2, keys, 2, D, dtype=dtype), _randn(3, keys, 2, D, dtype=dtype)
    q[..., 0] = 4.0
    k[:first, :, 0], k[first:, :, 0] = 0.0, 75.0 * D ** 0.5
    call = lambda: packed_attention_fwd(q, k, v, _ints([0, tokens]), cu_seqlens_k=_ints([0, keys]))
    v[:first, :, 5] = 1e38 if act == "bf16" else 6e4
    rows = slice(first, tokens) if tokens == keys else slice(0, tokens)               # that see near keys
    n = tokens - rows.start
    _close(call()[rows], *_reference(q[rows], k[first:], v[first:], D ** -0.5))
    v[9, :, 7] = -math.inf
    got = call()
    assert (got[rows, :, 7] == -math.inf).all() and torch.isfinite(got[rows, :, :7]).all() and torch.isfinite(got[rows, :, 8:]).all() and n > 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("tokens, keys", [(300, 300), (3, 9000)])
def test_a_scale_of_zero_makes_all_finite_scores_equal(D, tokens, keys):
    from pla.prefill.attention import packed_attention_fwd
    q, k, v = _randn(1, tokens, 4, D, dtype=torch.bfloat16), _randn(2, keys, 2, D, dtype=torch.bfloat16), _randn(3, keys, 2, D, dtype=torch.bfloat16)
    q[..., 0] = 1e19
    k[::3, :, 0], k[1::3, :, 0] = 1.5e19, -1.5e19
    got = packed_attention_fwd(q, k, v, _ints([0, tokens]), cu_seqlens_k=_ints([0, keys]), scale=0.0)
    zero = torch.zeros_like(q)
    _close(got, *_reference(zero, k * 0, v, 1.0))
