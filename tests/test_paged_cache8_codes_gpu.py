"""What a cache of 8-bit numbers holds of heads that no arithmetic comes before: scales and numbers to the last bit."""
import pytest
import torch

from test_paged_cache8_and_prefix_gpu import DEV, DTYPES, E4M3, _randn

pytestmark = pytest.mark.gpu


def _stored(x):
    """The definition, each step rounded once: scale = max(largest magnitude, 1e-30) / 448 in 32 bits, numbers = x / scale in 32 bits, to nearest."""
    x = x.float().cpu()
    scale = x.abs().amax(-1).clamp(min=1e-30) / 448
    return (x / scale[..., None]).to(E4M3).float(), scale


@pytest.mark.parametrize("T, HKV, D, act", [(7, 2, 64, "bf16"), (4096, 8, 128, "bf16"), (4096, 8, 128, "fp16"), (3000, 3, 256, "bf16"), (9000, 4, 64, "fp16")])
def test_numbers_and_scales_are_the_quotients(T, HKV, D, act):
    from pla.decode.paged import fused_qk_norm_rope
    q, k, v = (_randn(i, T, HKV, D, dtype=DTYPES[act]) for i in range(3))
    for x, seed in ((k, 4), (v, 5)):
        # largest magnitudes of which 448 parts are short numbers: the quotients of others meet the middle between two numbers
        tops = torch.tensor([3.0625, 3.5, 4.375, 7.0, 2.625, 5.25, 3.28125, 6.125], device=DEV)
        x.clamp_(-2.5, 2.5)
        x[:, :, D // 3] = tops[torch.randint(0, 8, (T, HKV), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))].to(x.dtype)
        x[T // 2:] = _randn(seed + 6, T - T // 2, HKV, D, dtype=DTYPES[act])          # and largest magnitudes as they come
        x[2] *= 1e-3
        x[3, 0] = 0
        x[4, 1, 1:] = 0
        x[5, 0, :8] = torch.tensor([3.0625, -1.3671875, 1.3671875, 0.0013, -1e-5, 3e-6, 2e-7, 0], device=DEV).to(x.dtype)
        x[5, 0, 8:] = 0
    blocks = -(-T // 16)
    k_cache, v_cache = (torch.zeros(blocks, 16, HKV, D, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2))
    k_scales, v_scales = (torch.zeros(blocks, HKV, 16, device=DEV) for _ in range(2))
    fused_qk_norm_rope(q, k, v=v, k_cache=k_cache, v_cache=v_cache, slot_mapping=torch.arange(T, device=DEV), k_scales=k_scales, v_scales=v_scales)
    for x, cache, scales in ((v, v_cache, v_scales), (k, k_cache, k_scales)):
        numbers, scale = _stored(x)
        got = cache.view(-1, HKV, D)[:T].float().cpu()
        assert torch.equal(scales.transpose(1, 2).reshape(-1, HKV)[:T].cpu(), scale)
        assert torch.equal(got, numbers), (got != numbers).sum().item()


def test_heads_with_infinities_hold_zeros_and_nan():
    from pla.decode.paged import fused_qk_norm_rope
    q, k, v = (_randn(i, 3, 2, 128, dtype=torch.bfloat16) for i in range(3))
    v[1, 0, 7], v[1, 0, 9] = float("inf"), float("-inf")
    cache, scales = torch.zeros(2, 1, 16, 2, 128, device=DEV).to(E4M3), torch.zeros(2, 1, 2, 16, device=DEV)
    fused_qk_norm_rope(q, k, v=v, k_cache=cache[0], v_cache=cache[1], slot_mapping=torch.arange(3, device=DEV), k_scales=scales[0], v_scales=scales[1])
    numbers, scale = _stored(v)
    assert torch.equal(scales[1, 0, :, :3].t().cpu(), scale)
    torch.testing.assert_close(cache[1, 0, :3].float().cpu(), numbers, rtol=0, atol=0, equal_nan=True)
