"""Caches of 8-bit numbers and shared prefixes: what is refused before any launch, and host arithmetic."""
import pytest
import torch

from pla_amd.decode.paged import fused_qk_norm_rope, paged_attention_decode

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
_INTS = dict(dtype=torch.int32)


def _e4m3(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(E4M3)


def _store_args(**change):
    T, HQ, HKV, D = 5, 4, 2, 64
    args = dict(q=torch.zeros(T, HQ, D, dtype=BF16), k=torch.zeros(T, HKV, D, dtype=BF16), v=torch.zeros(T, HKV, D, dtype=BF16), k_cache=_e4m3(3, 16, HKV, D),
                v_cache=_e4m3(3, 16, HKV, D), slot_mapping=torch.zeros(T, dtype=torch.int64), k_scales=torch.zeros(3, HKV, 16), v_scales=torch.zeros(3, HKV, 16))
    args.update(change)
    return args


@pytest.mark.parametrize("change, message", [
    (dict(k_scales=None, v_scales=None), "k_cache must be BFloat16"),
    (dict(k_cache=torch.zeros(3, 16, 2, 64, dtype=BF16)), "k_cache must be Float8_e4m3fn"),
    (dict(v_cache=torch.zeros(3, 16, 2, 64, dtype=torch.uint8)), "v_cache must be Float8_e4m3fn"),
    (dict(k_scales=None), "v_scales come with v and k_scales"),
    (dict(v_scales=None), "v_scales come with v and k_scales"),
    (dict(v=None, v_cache=None), "v_scales come with v and k_scales"),
    (dict(k_cache=None, slot_mapping=None, v=None, v_cache=None, v_scales=None), "k_scales come with k_cache"),
    (dict(k_scales=torch.zeros(3, 16, 2)), "k_scales must be"),
    (dict(v_scales=torch.zeros(3, 2, 15)), "v_scales must be"),
    (dict(k_scales=torch.zeros(3, 2, 16, dtype=BF16)), "must be float32"),
    (dict(k_scales=torch.zeros(3, 2, 32)[..., ::2]), "dense places"),
    (dict(k_scales=torch.zeros(3, 2, 18)[..., :16]), "16-byte aligned heads"),
    (dict(v_scales=torch.zeros(97)[1:].view(3, 2, 16)), "16-byte aligned heads"),
    (dict(k_cache=_e4m3(3, 16, 2, 72)[..., :64]), "16-byte aligned rows"),
    (dict(k_scales=torch.zeros(3, 2, 16, device="meta")), "k_scales must be on the device of q"),
    (dict(), "q must be a CUDA tensor"),
])
def test_store_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        fused_qk_norm_rope(**_store_args(**change))


def _read_args(**change):
    T, HQ, HKV, D = 6, 4, 2, 128
    args = dict(q=torch.zeros(T, HQ, D, dtype=BF16), k_cache=_e4m3(5, 16, HKV, D), v_cache=_e4m3(5, 16, HKV, D), block_table=torch.zeros(3, 4, **_INTS),
                seq_lens=torch.zeros(3, **_INTS), query_start_loc=torch.tensor([0, 2, 4, 6], **_INTS), max_query_len=2,
                k_scales=torch.zeros(5, HKV, 16), v_scales=torch.zeros(5, HKV, 16))
    args.update(change)
    return args


@pytest.mark.parametrize("change, message", [
    (dict(k_scales=None), "come together"),
    (dict(k_scales=None, v_scales=None), "k_cache must be BFloat16"),
    (dict(k_cache=torch.zeros(5, 16, 2, 128, dtype=BF16), v_cache=torch.zeros(5, 16, 2, 128, dtype=BF16)), "k_cache must be Float8_e4m3fn"),
    (dict(k_scales=torch.zeros(5, 16, 2)), "k_scales must be"),
    (dict(v_scales=torch.zeros(5, 2, 16, dtype=torch.float64)), "must be float32"),
    (dict(v_scales=torch.zeros(5, 2, 20)[..., :16]), "same strides"),
    (dict(prefix_blocks=torch.zeros(2, **_INTS), prefix_len=torch.zeros(1, **_INTS)), "a cache of q's type"),
    (dict(v_scales=torch.zeros(5, 2, 16, device="meta")), "v_scales must be on the device of q"),
    (dict(), "q must be a CUDA tensor"),
])
def test_attention_over_8_bits_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        paged_attention_decode(**_read_args(**change))


def _prefix_args(**change):
    cache = torch.zeros(5, 2, 16, 2, 128, dtype=BF16)
    args = dict(q=torch.zeros(3, 4, 128, dtype=BF16), k_cache=cache[:, 0], v_cache=cache[:, 1], block_table=torch.zeros(3, 4, **_INTS),
                seq_lens=torch.zeros(3, **_INTS), prefix_blocks=torch.zeros(2, **_INTS), prefix_len=torch.zeros(1, **_INTS))
    args.update(change)
    return args


@pytest.mark.parametrize("change, message", [
    (dict(prefix_len=None), "come together"),
    (dict(prefix_blocks=None), "come together"),
    (dict(prefix_blocks=torch.zeros(2, dtype=torch.int64)), "prefix_blocks must be"),
    (dict(prefix_blocks=torch.zeros(1, 2, **_INTS)), "prefix_blocks must be"),
    (dict(prefix_blocks=torch.zeros(4, **_INTS)[::2]), "prefix_blocks must be"),
    (dict(prefix_blocks=torch.empty(2 ** 26 + 1, device="meta", **_INTS)), "at most 2\\^30 positions"),
    (dict(prefix_len=torch.zeros(2, **_INTS)), "prefix_len must have 1 entries"),
    (dict(prefix_len=torch.zeros(1)), "prefix_len must be an int32 or int64 vector"),
    (dict(prefix_len=torch.zeros((), **_INTS)), "prefix_len must be an int32 or int64 vector"),
    (dict(prefix_len=torch.zeros(1, device="meta", **_INTS)), "prefix_len must be on the device of q"),
    (dict(), "q must be a CUDA tensor"),
])
def test_attention_over_a_prefix_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        paged_attention_decode(**_prefix_args(**change))


def test_native_entry_points_reject_bad_arguments():
    from pla_amd import _lib
    lib = _lib.load()

    def refused(name, args, message):
        assert getattr(lib, name)(*args) != 0 and message in lib.pla_last_error(), lib.pla_last_error()

    rope = [None, None, None, None, None, 0, None, None, 0, 1e-6, 0.0, None, 0, 1.0, 0, None, None, None, None, None, None, None, None, 0, 0, 16, 4, 2, 1, 128,
            _lib.BF16, None]
    refused("pla_qk_norm_rope_fp8_launch", rope, b"null tensor pointer")
    tail = [None, 4, 3, 4, None, 0, None, 0, None, 0, None, 0, 0, None, 0, 0, 0.1, 3, 3, 1, 4, 2, 128, _lib.BF16, None, 0, None]
    refused("pla_paged_attention_fp8_launch", [None, 0, 0, None, None, 0, 0, 0, 5, 16, None, None, 0, 0] + tail, b"null tensor pointer")
    refused("pla_paged_attention_prefix_launch", [None, 0, 0, None, None, 0, 0, 0, 5, 16, None, 0, None, 0] + tail, b"null tensor pointer")


def test_workspace_of_a_prefix_is_host_arithmetic():
    from pla_amd import _lib
    size, plain = _lib.load().pla_paged_attention_prefix_workspace_bytes, _lib.load().pla_paged_attention_workspace_bytes
    assert size(0, 5, 4, 2, 128, 1, 64, 64) == 0 and size(3, 0, 4, 2, 128, 1, 64, 64) == 0
    assert size(3, 3, 4, 2, 96, 1, 64, 64) == -1 and size(3, 3, 4, 2, 128, 33, 64, 64) == -1 and size(3, 3, 4, 2, 128, 1, 64, -1) == -1
    # one piece is kept even of a prefix of no pages
    assert size(3, 3, 4, 2, 128, 1, 4096, 0) >= plain(3, 4, 2, 128, 1, 4096) + 3 * 4 * (128 * 4 + 8)
    assert size(64, 64, 32, 8, 128, 1, 4096, 1 << 16) == size(64, 64, 32, 8, 128, 1, 4096, 16)          # the length stands on the device


def test_sanity_mode_names_a_prefix_that_would_be_cut_or_left_out(monkeypatch):
    ints = lambda *x: torch.tensor(x, **_INTS)
    monkeypatch.setenv("PLA_SANITY_CHECK", "1")
    for blocks, length, message in ((ints(1, 2), ints(33), "passes prefix_blocks"), (ints(1, 2), ints(-1), "negative"), (ints(1, 5), ints(17), "not in the cache"),
                                    (ints(-1, 2), ints(1), "not in the cache")):
        with pytest.raises(RuntimeError, match=r"PLA_SANITY_CHECK \[paged_attention_decode\]: .*" + message):
            paged_attention_decode(**_prefix_args(prefix_blocks=blocks, prefix_len=length))
    for blocks, length in ((ints(1, 5), ints(16)), (ints(1, 2), ints(0)), (ints(), ints(0))):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            paged_attention_decode(**_prefix_args(prefix_blocks=blocks, prefix_len=length))
    with pytest.raises(RuntimeError, match="prefix_len must have 1 entries"):
        paged_attention_decode(**_prefix_args(prefix_len=ints(1, 2)))
