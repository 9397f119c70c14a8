"""Sanity mode leaves calls with a prefix that are not of their form to the compiled checks."""
import pytest
import torch

from test_paged_cache8_and_prefix_cpu import _INTS, _prefix_args

from pla_amd.decode.paged import paged_attention_decode


def test_a_cache_of_empty_blocks_is_refused_by_the_compiled_checks(monkeypatch):
    cache = torch.zeros(5, 0, 2, 128, dtype=torch.bfloat16)
    for mode in ("0", "1"):
        monkeypatch.setenv("PLA_SANITY_CHECK", mode)
        with pytest.raises(RuntimeError, match="must hold at least one block"):
            paged_attention_decode(**_prefix_args(k_cache=cache, v_cache=cache, prefix_len=torch.zeros(1, **_INTS)))
