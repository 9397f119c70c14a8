"""Attention over prompts: what is refused before any launch, host arithmetic, values that sanity mode names."""
import pytest
import torch

from pla_amd.prefill.attention import packed_attention_fwd, paged_attention_prefill

BF16 = torch.bfloat16
_INTS = dict(dtype=torch.int32)


def _packed_args(**change):
    args = dict(q=torch.zeros(6, 4, 128, dtype=BF16), k=torch.zeros(6, 2, 128, dtype=BF16), v=torch.zeros(6, 2, 128, dtype=BF16),
                cu_seqlens=torch.tensor([0, 2, 6], **_INTS))
    args.update(change)
    return args


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros(6, 4, 96, dtype=BF16)), "head_dim must be 64, 128 or 256"),
    (dict(q=torch.zeros(6, 512, dtype=BF16)), "must be \\[tokens, heads, head_dim\\]"),
    (dict(q=torch.zeros(6, 4, 128)), "q must be bf16 or fp16"),
    (dict(q=torch.zeros(6, 3, 128, dtype=BF16)), "multiple of key-value heads"),
    (dict(k=torch.zeros(6, 0, 128, dtype=BF16)), "multiple of key-value heads"),
    (dict(k=torch.zeros(6, 2, 128, dtype=torch.float16)), "k must be"),
    (dict(v=torch.zeros(6, 4, 128, dtype=BF16)), "v must be"),
    (dict(v=torch.zeros(5, 2, 128, dtype=BF16)), "v must be"),
    (dict(k=torch.zeros(6, 2, 256, dtype=BF16)[..., ::2]), "dense channels"),
    (dict(v=torch.zeros(6 * 256 + 4, dtype=BF16)[4:].view(6, 2, 128)), "16-byte aligned"),
    (dict(k=torch.zeros(5, 2, 128, dtype=BF16), v=torch.zeros(5, 2, 128, dtype=BF16)), "a key for every token"),
    (dict(k=torch.empty(6, 2, 128, dtype=BF16, device="meta").as_strided((6, 2, 128), (1 << 24, 128, 1))), "below 2\\^24"),
    (dict(cu_seqlens=torch.zeros(0, **_INTS)), "at least one entry"),
    (dict(cu_seqlens=torch.zeros(3)), "cu_seqlens must be an int32 or int64 vector"),
    (dict(cu_seqlens_k=torch.zeros(2, **_INTS)), "cu_seqlens_k must have 3 entries"),
    (dict(q=torch.empty(1 << 28, 8, 64, dtype=BF16, device="meta"), k=torch.empty(1 << 28, 1, 64, dtype=BF16, device="meta"),
          v=torch.empty(1 << 28, 1, 64, dtype=BF16, device="meta")), "too many rows"),
    (dict(scale=float("nan")), "scale must be finite"),
    (dict(scale=1e39), "scale must be finite"),
    (dict(output_gate=torch.zeros(6, 4, 64, dtype=BF16)), "output_gate must be"),
    (dict(out=torch.zeros(5, 4, 128, dtype=BF16)), "out must be"),
    (dict(cu_seqlens=torch.zeros(3, device="meta", **_INTS)), "cu_seqlens must be on the device of q"),
    (dict(), "q must be a CUDA tensor"),
])
def test_packed_attention_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        packed_attention_fwd(**_packed_args(**change))


def _paged_args(**change):
    cache = torch.zeros(5, 2, 16, 2, 128, dtype=BF16)
    args = dict(q=torch.zeros(60, 4, 128, dtype=BF16), k_cache=cache[:, 0], v_cache=cache[:, 1], block_table=torch.zeros(3, 4, **_INTS),
                seq_lens=torch.zeros(3, **_INTS), query_start_loc=torch.tensor([0, 20, 40, 60], **_INTS))
    args.update(change)
    return args


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros(6, 4, 80, dtype=BF16)), "head_dim must be"),
    (dict(q=torch.zeros(6, 4, 128)), "q must be bf16 or fp16"),
    (dict(q=torch.zeros(6, 3, 128, dtype=BF16)), "multiple of key-value heads"),
    (dict(q=torch.zeros(6, 4, 128, dtype=torch.float16)), "k_cache must be"),
    (dict(k_cache=torch.zeros(5, 16, 2, 128, dtype=BF16)), "same shape and strides"),
    (dict(k_cache=torch.zeros(5, 24, 2, 128, dtype=BF16), v_cache=torch.zeros(5, 24, 2, 128, dtype=BF16)), "multiple of 16"),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int64)), "block_table must be int32"),
    (dict(block_table=torch.zeros(2, 4, **_INTS)), "more requests than rows"),
    (dict(block_table=torch.empty(3, 2 ** 26 + 1, device="meta", **_INTS)), "at most 2\\^30 positions"),
    (dict(seq_lens=torch.zeros(3)), "seq_lens must be an int32 or int64 vector"),
    (dict(query_start_loc=torch.zeros(3, **_INTS)), "query_start_loc must have 4 entries"),
    (dict(request_indices=torch.zeros(2, **_INTS)), "request_indices must have 3 entries"),
    (dict(scale=float("inf")), "scale must be finite"),
    (dict(output_gate=torch.zeros(60, 4, 64, dtype=BF16)), "output_gate must be"),
    (dict(out=torch.zeros(60, 4, 128, dtype=torch.float16)), "out must be"),
    (dict(seq_lens=torch.zeros(3, device="meta", **_INTS)), "seq_lens must be on the device of q"),
    (dict(), "q must be a CUDA tensor"),
])
def test_paged_prefill_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        paged_attention_prefill(**_paged_args(**change))


def test_native_entry_points_reject_bad_arguments():
    from pla_amd import _lib
    lib = _lib.load()

    def refused(name, args, message):
        assert getattr(lib, name)(*args) != 0 and message in lib.pla_last_error(), lib.pla_last_error()

    packed = [None, 0, 0, None, 0, 0, None, 0, 0, None, 0, None, 0, None, 0, 0, None, 0, 0, 0.1, 3, 30, 30, 4, 2, 128, _lib.BF16, None, 0, None]
    refused("pla_prompt_attention_launch", packed, b"null tensor pointer")
    refused("pla_prompt_attention_launch", packed[:25] + [96] + packed[26:], b"head_dim")
    refused("pla_prompt_attention_launch", packed[:24] + [3] + packed[25:], b"multiple of key-value heads")
    refused("pla_prompt_attention_launch", packed[:26] + [_lib.F32] + packed[27:], b"bf16 or fp16")
    refused("pla_prompt_attention_launch", packed[:22] + [2 ** 31] + packed[23:], b"too many keys")
    refused("pla_prompt_attention_launch", packed[:20] + [2 ** 24] + packed[21:], b"too many sequences")
    paged = [None, 0, 0, None, None, 0, 0, 0, 5, 16, None, 4, 3, 4, None, 0, None, 0, None, 0, None, 0, 0, None, 0, 0, 0.1, 3, 30, 4, 2, 128, _lib.BF16,
             None, 0, None]
    refused("pla_paged_prompt_attention_launch", paged, b"null tensor pointer")
    refused("pla_paged_prompt_attention_launch", paged[:9] + [24] + paged[10:], b"multiple of 16")
    refused("pla_paged_prompt_attention_launch", paged[:27] + [4] + paged[28:], b"more requests")


def test_workspace_is_host_arithmetic():
    from pla_amd import _lib
    size = _lib.load().pla_prompt_attention_workspace_bytes
    assert size(1, 1 << 15, 16, 2, 128, 1 << 15) == 0                     # enough rows: no pieces
    assert size(0, 100, 16, 2, 128, 100) == 0 and size(3, 0, 16, 2, 128, 100) == 0
    assert size(1, 40, 16, 2, 96, 1 << 15) == -1 and size(1, 40, 16, 3, 128, 1 << 15) == -1 and size(1, 40, 16, 2, 128, -1) == -1
    few = size(1, 40, 16, 2, 128, 1 << 15)
    assert few > 0 and few % 256 == 0


def test_sanity_mode_names_values_that_would_be_passed_over(monkeypatch):
    ints = lambda *x: torch.tensor(x, **_INTS)
    monkeypatch.setenv("PLA_SANITY_CHECK", "1")
    for cu, cu_k, message in ((ints(1, 2, 6), None, "cu_seqlens must start at 0"), (ints(0, 4, 2), None, "not decrease"), (ints(0, 4, 7), None, "stay within"),
                              (ints(0, 2, 6), ints(0, 3, 7), "cu_seqlens_k must"), (ints(0, 2, 6), ints(0, 1, 6), "fewer keys than tokens")):
        with pytest.raises(RuntimeError, match=r"PLA_SANITY_CHECK \[packed_attention_fwd\]: .*" + message):
            packed_attention_fwd(**_packed_args(cu_seqlens=cu, cu_seqlens_k=cu_k))
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):      # what is sound goes on to the compiled checks
        packed_attention_fwd(**_packed_args())
    with pytest.raises(RuntimeError, match="cu_seqlens_k must have 3 entries"):
        packed_attention_fwd(**_packed_args(cu_seqlens_k=ints(0, 2)))
    with pytest.raises(RuntimeError, match=r"PLA_SANITY_CHECK \[paged_attention_prefill\]: .*stay within q"):
        paged_attention_prefill(**_paged_args(query_start_loc=ints(0, 20, 40, 61)))
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        paged_attention_prefill(**_paged_args())


def test_the_namespace_is_the_same_module_under_both_names():
    import pla.prefill.attention
    import pla_amd.prefill.attention
    assert pla.prefill.attention is pla_amd.prefill.attention
    assert set(pla.prefill.attention.__all__) == {"packed_attention_fwd", "paged_attention_prefill"}
