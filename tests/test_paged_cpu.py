"""Host side of the paged attention operators (no GPU): how the work is dealt out, refused calls, frequencies, value checks."""
import ctypes
import math
import random

import pytest
import torch

from pla.decode.paged import (PagedKVBlocks, PagedKVPlan, fused_qk_norm_rope, paged_attention_decode, paged_kv_plan,
                              rotary_frequencies)

BF16 = torch.bfloat16


# ---- schedule ---------------------------------------------------------------------------------------------------

def _segments(windows, lengths, HQ, HKV, D, max_query, positions, tokens=None):
    """Every worker's segments of a batch, as the kernel takes them."""
    from pla_amd import _lib
    lib = _lib.load()
    offsets = [0]
    for w in windows:
        offsets.append(offsets[-1] + w)
    tokens = offsets[-1] if tokens is None else tokens
    n = len(windows)
    c_off, c_len = (ctypes.c_int32 * (n + 1))(*offsets), (ctypes.c_int32 * n)(*lengths)
    room = 4096
    buf = (ctypes.c_int64 * (7 * room))()
    out = []
    for worker in range(4 * 256 + 1):
        found = lib.pla_paged_attention_segments(c_off, c_len, n, tokens, HQ, HKV, D, max_query, positions, worker, buf, room)
        assert 0 <= found <= room
        if found == 0:
            break
        out.append([tuple(buf[7 * i:7 * i + 7]) for i in range(found)])
    return out


def _rows_of_a_block(D, max_query, group):
    return 16 if max_query * group <= 16 else 32 if max_query * group <= 32 or D == 256 else 64


def _keys_of_a_tile(D, rows, alone):
    return 32 if alone else 256 if D == 64 and rows == 16 else 128


@pytest.mark.parametrize("seed", range(30))
def test_every_tile_of_every_run_is_taken_once_and_its_pieces_are_found(seed):
    rng = random.Random(seed)
    HKV, group, D = rng.choice((1, 2, 3, 8)), rng.choice((1, 4, 7, 16)), rng.choice((64, 128, 256))
    max_query = rng.choice((1, 1, 4, 8, 32))
    n = rng.choice((1, 1, 2, 7, 65, 300))
    positions = rng.choice((32, 128, 130, 5000, 131072))
    windows = [rng.randint(0, max_query) for _ in range(n)]
    windows[rng.randrange(n)] = max_query
    lengths = [rng.choice((0, -3, 1, 127, 128, 129, positions, positions + 500, rng.randint(0, positions))) for _ in range(n)]
    got = _segments(windows, lengths, HKV * group, HKV, D, max_query, positions)
    rows = _rows_of_a_block(D, max_query, group)
    workers, waves = 256 if D == 256 else 512, 8 if D == 64 else 4
    alone = rows == 16 and n * HKV >= workers * waves // 32 and not (positions <= 32 * waves and n * HKV <= workers)
    tile_keys = _keys_of_a_tile(D, rows, alone)
    expected = {}
    for i, (w, length) in enumerate(zip(windows, lengths)):
        tiles = max(1, -(-min(max(length, 0), positions) // tile_keys)) + alone        # one on top of each
        for h in range(HKV):
            for b in range(-(-w * group // rows)):
                expected[i, h, b] = tiles
    total = sum(expected.values())
    taken, slots = {}, {}
    for worker, segments in enumerate(got):
        for r, h, b, tile, tiles, slot, pieces in segments:
            assert tiles >= 1
            for t in range(tile, tile + tiles):
                assert (r, h, b, t) not in taken
                taken[r, h, b, t] = worker
            whole = tile == 0 and tiles == expected[r, h, b]
            assert (slot == -1) == whole
            if not whole:
                assert slot == 2 * worker + (1 if tile == 0 else 0) and slot not in slots
                slots[slot] = (r, h, b, tile, tiles)
    assert set(taken) == {(*run, t) for run, tiles in expected.items() for t in range(tiles)}
    # stretches are as equal as whole tiles are
    sizes = [sum(s[4] for s in segments) for segments in got]
    assert max(sizes) - min(sizes) <= 1 and len(got) <= total
    # the joining workgroup's arithmetic: piece 0 in slot 2 w + 1, piece i in slot 2 (w + i)
    for worker, segments in enumerate(got):
        for r, h, b, tile, tiles, slot, pieces in segments:
            if tile != 0:
                assert pieces == 0
                continue
            if slot == -1:
                assert pieces == 1
                continue
            assert pieces >= 2
            found = [slots[2 * worker + 1 if i == 0 else 2 * (worker + i)] for i in range(pieces)]
            assert all(f[:3] == (r, h, b) for f in found)
            at = 0
            for f in found:
                assert f[3] == at
                at += f[4]
            assert at == expected[r, h, b]


def test_requests_that_are_passed_over_take_no_work():
    # empty, too long, outside of the token rows; the others keep theirs
    got = _segments([0, 5, 2, 3], [400, 400, 400, 400], 2, 1, 128, 4, 1024, tokens=9)
    assert {s[0] for segments in got for s in segments} == {2}
    assert _segments([0, 0], [5, 6], 2, 1, 64, 4, 1024, tokens=3) == []


def test_workspace_is_host_arithmetic():
    from pla_amd import _lib
    size = _lib.load().pla_paged_attention_workspace_bytes
    assert size(8, 16, 2, 128, 1, 128) == 0                  # one tile a run: nothing is ever cut
    assert size(0, 16, 2, 128, 1, 4096) == 0
    one, many = size(1, 16, 2, 128, 1, 4096), size(64, 16, 2, 128, 1, 4096)
    assert 0 < one < many and one % 256 == 0 and many == size(1000, 16, 2, 128, 1, 4096)      # bounded by the chip
    for bad in ((1, 16, 3, 128, 1, 99), (1, 16, 2, 96, 1, 99), (1, 16, 2, 128, 33, 99), (1, 16, 2, 128, 0, 99), (-1, 16, 2, 128, 1, 99),
                (1, 16, 2, 128, 1, 2 ** 30 + 1), (1, 2 ** 26, 1, 128, 32, 99)):
        assert size(*bad) == -1


def test_places_of_pages_good_and_bad(tmp_path):
    """The kernel's own arithmetic from position to page to place in the cache, compiled for the host: entries that are no block of
    the cache lie nowhere, whatever they are, and the division by the block size is exact."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    source, library = tmp_path / "places.cpp", tmp_path / "places.so"
    source.write_text('#include "%s"\n' % os.path.join(root, "pla_amd", "csrc", "paged_schedule.h") + """
        extern "C" long long place(int entry, int at, int blocks, long long block, long long token) {
          return pla::paged_place(entry, at, blocks, block, token);
        }
        extern "C" int page(int n, int d) { return pla::paged_quotient(pla::paged_divisor(d), n); }
    """)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(library), str(source)], check=True)
    lib = ctypes.CDLL(str(library))
    lib.place.restype = ctypes.c_longlong
    lib.place.argtypes = [ctypes.c_int] * 3 + [ctypes.c_longlong] * 2
    far = 2 ** 33 + 8
    assert [lib.place(e, 5, 7, far, 128) for e in (0, 3, 6)] == [640, 3 * far + 640, 6 * far + 640]
    for bad in (-1, 7, 8, 2 ** 31 - 1, -2 ** 31):
        assert lib.place(bad, 5, 7, far, 128) == -1
    rng = random.Random(1)
    for d in list(range(1, 70)) + [528, 784, 1000, 4096, 65520, 2 ** 30 - 1, 2 ** 30]:
        edges = [k * d + e for k in (0, 1, 2, 1000, (2 ** 31 - 1) // d) for e in (-1, 0, 1)]
        for n in edges + [2 ** 31 - 1] + [rng.randrange(2 ** 31) for _ in range(200)]:
            if 0 <= n < 2 ** 31:
                assert lib.page(n, d) == n // d, (n, d)


# ---- refusals ---------------------------------------------------------------------------------------------------

def _rope_args(**change):
    T, HQ, HKV, D = 5, 4, 2, 64
    row = torch.zeros(T, (HQ + 2 * HKV) * D, dtype=BF16)
    q, k, v = row[:, :HQ * D].view(T, HQ, D), row[:, HQ * D:(HQ + HKV) * D].view(T, HKV, D), row[:, (HQ + HKV) * D:].view(T, HKV, D)
    args = dict(q=q, k=k, positions=torch.zeros(T, dtype=torch.int32), q_weight=torch.zeros(D, dtype=BF16), k_weight=torch.zeros(D, dtype=BF16),
                inv_freq=torch.ones(16), v=v, k_cache=torch.zeros(3, 16, HKV, D, dtype=BF16), v_cache=torch.zeros(3, 16, HKV, D, dtype=BF16),
                slot_mapping=torch.zeros(T, dtype=torch.int64))
    args.update(change)
    return args


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros(5, 4, 96, dtype=BF16)), "head_dim must be 64, 128 or 256"),
    (dict(q=torch.zeros(5, 4, 64)), "q must be bf16 or fp16"),
    (dict(q=torch.zeros(4, 4, 64, dtype=BF16)), "k must be"),
    (dict(k=torch.zeros(5, 2, 64, dtype=torch.float16)), "k must be"),
    (dict(q=torch.zeros(5, 4, 64 * 2, dtype=BF16)[:, :, ::2]), "dense channels"),
    (dict(q=torch.zeros(5 * 4 * 64 + 4, dtype=BF16)[4:].view(5, 4, 64)), "16-byte aligned"),
    (dict(positions=None), "a rotation needs positions"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), "positions must have 5 entries"),
    (dict(positions=torch.zeros(5)), "positions must be an int32 or int64 vector"),
    (dict(inv_freq=torch.ones(4)), "multiple of 16"),
    (dict(inv_freq=torch.ones(40)), "multiple of 16 up to head_dim"),
    (dict(inv_freq=torch.ones(16, dtype=torch.float64)), "inv_freq must be a contiguous float32"),
    (dict(q_weight=torch.zeros(32, dtype=BF16)), "q_weight must be"),
    (dict(k_weight=torch.zeros(64)), "of one type"),
    (dict(slot_mapping=None), "come together"),
    (dict(k_cache=None, slot_mapping=None), "v comes with v_cache"),
    (dict(v=None), "v comes with v_cache"),
    (dict(v_cache=torch.zeros(4, 16, 2, 64, dtype=BF16)), "same blocks"),
    (dict(k_cache=torch.zeros(0, 16, 2, 64, dtype=BF16)), "at least one block"),
    (dict(k_cache=torch.zeros(3, 16, 2, 128, dtype=BF16)), "k_cache must be"),
    (dict(eps=-1.0), "eps not negative"),
    (dict(eps=float("nan")), "must be finite"),
    (dict(attention_factor=float("inf")), "must be finite"),
    (dict(weight_offset=1e300), "must be finite"),           # not in float32
    (dict(q_out=torch.zeros(5, 3, 64, dtype=BF16)), "q_out must be"),
    (dict(slot_mapping=torch.zeros(5, dtype=torch.int64, device="meta")), "slot_mapping must be on the device of q"),
    (dict(), "q must be a CUDA tensor"),
])
def test_norm_and_rotation_refuse(change, message):
    with pytest.raises(RuntimeError, match=message):
        fused_qk_norm_rope(**_rope_args(**change))


def _attention_args(**change):
    T, HQ, HKV, D = 6, 4, 2, 128
    cache = torch.zeros(5, 2, 16, HKV, D, dtype=BF16)
    args = dict(q=torch.zeros(T, HQ, D, dtype=BF16), k_cache=cache[:, 0], v_cache=cache[:, 1], block_table=torch.zeros(3, 4, dtype=torch.int32),
                seq_lens=torch.zeros(3, dtype=torch.int32), query_start_loc=torch.tensor([0, 2, 4, 6], dtype=torch.int32), max_query_len=2)
    args.update(change)
    return args


@pytest.mark.parametrize("change, message", [
    (dict(q=torch.zeros(6, 4, 80, dtype=BF16)), "head_dim must be"),
    (dict(q=torch.zeros(6, 4, 128)), "q must be bf16 or fp16"),
    (dict(q=torch.zeros(6, 3, 128, dtype=BF16)), "multiple of key-value heads"),
    (dict(q=torch.zeros(6, 4, 128, dtype=torch.float16)), "k_cache must be"),
    (dict(k_cache=torch.zeros(5, 16, 2, 128, dtype=BF16)), "same shape and strides"),
    (dict(k_cache=torch.zeros(5, 24, 2, 128, dtype=BF16), v_cache=torch.zeros(5, 24, 2, 128, dtype=BF16)), "multiple of 16"),
    (dict(k_cache=torch.zeros(5, 16, 2, 256, dtype=BF16)[..., ::2], v_cache=torch.zeros(5, 16, 2, 256, dtype=BF16)[..., ::2]), "dense channels"),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int64)), "block_table must be int32"),
    (dict(block_table=torch.zeros(3, 8, dtype=torch.int32)[:, ::2]), "dense rows"),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int32)), "more requests than rows"),
    (dict(block_table=torch.empty(3, 2 ** 26 + 1, dtype=torch.int32, device="meta")), "at most 2\\^30 positions"),
    (dict(seq_lens=torch.zeros(3)), "seq_lens must be an int32 or int64 vector"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int32)), "query_start_loc must have 3 entries"),
    (dict(query_start_loc=None), "every request has one token row"),
    (dict(max_query_len=0), "between 1 and 32"),
    (dict(max_query_len=33), "between 1 and 32"),
    (dict(request_indices=torch.zeros(2, dtype=torch.int32)), "request_indices must have 3 entries"),
    (dict(scale=float("nan")), "scale must be finite"),
    (dict(scale=1e39), "scale must be finite"),              # not in float32
    (dict(output_gate=torch.zeros(6, 4, 64, dtype=BF16)), "output_gate must be"),
    (dict(out=torch.zeros(5, 4, 128, dtype=BF16)), "out must be"),
    (dict(out=torch.zeros(6, 4, 128, dtype=torch.float16)), "out must be"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32, device="meta")), "seq_lens must be on the device of q"),
    (dict(), "q must be a CUDA tensor"),
])
def test_attention_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        paged_attention_decode(**_attention_args(**change))


def _blocks(**change):
    made = PagedKVBlocks.allocate(20, 16, 4, 5, "cpu")
    fields = dict(block_table=made.block_table, held_blocks=made.held_blocks, free_blocks=made.free_blocks, free_count=made.free_count, block_size=16)
    fields.update(change)
    return PagedKVBlocks(**fields)


_INTS = dict(dtype=torch.int32)


@pytest.mark.parametrize("blocks, args, message", [
    (dict(block_table=torch.zeros(4, 5)), {}, "block_table must be int32"),
    (dict(held_blocks=torch.zeros(3, **_INTS)), {}, "held_blocks must have 4 entries"),
    (dict(free_blocks=torch.zeros(20, dtype=torch.int64)), {}, "free_blocks must be"),
    (dict(free_count=torch.zeros(2, **_INTS)), {}, "free_count must have 1"),
    (dict(block_size=0), {}, "block_size must be positive"),
    (dict(block_size=2 ** 28), {}, "at most 2\\^30"),
    ({}, dict(context_lens=torch.zeros(2)), "context_lens must be an int32"),
    ({}, dict(query_lens=torch.zeros(4, **_INTS)), "query_lens must have 3 entries"),
    ({}, dict(context_lens=torch.zeros(5, **_INTS), query_lens=torch.zeros(5, **_INTS)), "more batch entries than rows"),
    ({}, dict(request_indices=torch.zeros(2, **_INTS)), "request_indices must have 3"),
    ({}, dict(token_capacity=-1), "token_capacity must be"),
    ({}, dict(token_capacity=2 ** 30 + 1), "token_capacity must be"),
    ({}, dict(out=PagedKVPlan.allocate(3, 7, "cpu")), "positions must have 8 entries"),
    ({}, dict(out=PagedKVPlan.allocate(2, 8, "cpu")), "query_start_loc must have 4 entries"),
    ({}, dict(query_lens=torch.zeros(3, device="meta", **_INTS)), "query_lens must be on the device"),
    ({}, {}, "block_table must be a CUDA tensor"),
])
def test_plan_refuses(blocks, args, message):
    call = dict(context_lens=torch.zeros(3, **_INTS), query_lens=torch.zeros(3, **_INTS), token_capacity=8)
    call.update(args)
    with pytest.raises(RuntimeError, match=message):
        paged_kv_plan(_blocks(**blocks), **call)


def test_native_entry_points_reject_bad_arguments():
    from pla_amd import _lib
    lib = _lib.load()

    def refused(name, args, message):
        assert getattr(lib, name)(*args) != 0 and message in lib.pla_last_error(), lib.pla_last_error()

    plan = [None, 0, None, 0, None, 0, None, 4, 3, 4, None, None, None, 8, 3, 16, 10, None, None, None, None, None]
    refused("pla_paged_kv_plan_launch", plan, b"null tensor pointer")
    refused("pla_paged_kv_plan_launch", plan[:14] + [4] + plan[15:], b"more batch entries")
    refused("pla_paged_kv_plan_launch", plan[:15] + [0] + plan[16:], b"block_size")
    refused("pla_paged_kv_plan_launch", plan[:4] + [8, 0, None, 4, 8193] + plan[9:], b"at most 8192 rows")
    rope = [None, None, None, None, None, 0, None, None, 0, 1e-6, 0.0, None, 0, 1.0, 0, None, None, None, None, None, 0, 0, 16, 4, 2, 1, 128,
            _lib.BF16, None]
    refused("pla_qk_norm_rope_launch", rope, b"null tensor pointer")
    refused("pla_qk_norm_rope_launch", rope[:12] + [24] + rope[13:], b"multiple of 16")
    refused("pla_qk_norm_rope_launch", rope[:26] + [96] + rope[27:], b"head_dim")
    refused("pla_qk_norm_rope_launch", rope[:27] + [_lib.F32] + rope[28:], b"bf16 or fp16")
    attn = [None, 0, 0, None, None, 0, 0, 0, 5, 16, None, 4, 3, 4, None, 0, None, 0, None, 0, None, 0, 0, None, 0, 0, 0.1, 3, 3, 1, 4, 2, 128,
            _lib.BF16, None, 0, None]
    refused("pla_paged_attention_launch", attn, b"null tensor pointer")
    refused("pla_paged_attention_launch", attn[:9] + [24] + attn[10:], b"multiple of 16")
    refused("pla_paged_attention_launch", attn[:27] + [4] + attn[28:], b"more requests than token rows")
    refused("pla_paged_attention_launch", attn[:29] + [33] + attn[30:], b"max_query_len")
    refused("pla_paged_attention_launch", attn[:31] + [3] + attn[32:], b"multiple of key-value heads")


# ---- values ------------------------------------------------------------------------------------------------------

def test_frequencies():
    inv, factor = rotary_frequencies(64, 1e6)
    assert factor == 1.0 and inv.dtype == torch.float32 and inv.shape == (32,)
    assert inv[0] == 1.0 and abs(inv[31].item() * 1e6 ** (62 / 64) - 1) < 1e-6
    scaled, factor = rotary_frequencies(64, 1e6, factor=8.0, original_length=4096)
    assert abs(factor - (0.1 * math.log(8.0) + 1)) < 1e-12
    turns = inv.double() * 4096 / (2 * math.pi)
    ratio = (scaled / inv).double()
    # many turns: as they were; hardly any: an eighth; between them no frequency rises
    assert torch.allclose(ratio[turns > 40], torch.ones(1, dtype=torch.float64), atol=1e-6)
    assert torch.allclose(ratio[turns < 0.6], torch.full((1,), 0.125, dtype=torch.float64), atol=1e-6)
    assert (ratio[1:] <= ratio[:-1] + 1e-6).all()
    for bad in (dict(rotary_dim=63), dict(rotary_dim=64, base=1.0), dict(rotary_dim=64, factor=0.5), dict(rotary_dim=64, factor=4.0),
                dict(rotary_dim=64, factor=4.0, original_length=100, beta_fast=1.0, beta_slow=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_block_pool_allocation():
    pool = PagedKVBlocks.allocate(10, 16, 3, 4, "cpu")
    assert pool.free_blocks.tolist() == list(range(9, 0, -1)) and pool.free_count.item() == 9
    assert pool.block_table.shape == (3, 4) and pool.held_blocks.tolist() == [0, 0, 0]
    assert PagedKVBlocks.allocate(4, 16, 1, 1, "cpu", first_block=0).free_blocks.tolist() == [3, 2, 1, 0]
    for bad in ((3, 16, 1, 1, "cpu", 4), (4, 0, 1, 1, "cpu"), (4, 16, -1, 1, "cpu"), (4, 2 ** 28, 1, 5, "cpu")):
        with pytest.raises(ValueError):
            PagedKVBlocks.allocate(*bad)


def test_sanity_mode_names_values_that_would_be_passed_over(monkeypatch):
    from pla_amd.decode.paged import _sanity
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)
    pool = PagedKVBlocks.allocate(10, 16, 3, 4, "cpu")
    _sanity.check_plan(pool, ints(3, 5), ints(1, 1), ints(2, 0))
    for context, query, rows, message in ((ints(-1), ints(1), None, "negative"), (ints(60), ints(5), None, "pass its row"),
                                          (ints(1, 1), ints(1, 1), ints(2, 2), "different rows"), (ints(1), ints(1), ints(3), "different rows")):
        with pytest.raises(RuntimeError, match=r"PLA_SANITY_CHECK \[paged_kv_plan\]: .*" + message):
            _sanity.check_plan(pool, context, query, rows)
    pool.held_blocks[1] = 1
    pool.block_table[1, 0] = 4
    with pytest.raises(RuntimeError, match="held twice"):
        _sanity.check_plan(pool, ints(1), ints(1), None)
    cache = torch.zeros(3, 16, 1, 64)
    _sanity.check_slots(ints(-1, -1, 5, 47), cache)
    for slots, message in ((ints(5, 5), "name one slot"), (ints(48), "past the cache")):
        with pytest.raises(RuntimeError, match=message):
            _sanity.check_slots(slots, cache)
    q, table = torch.zeros(4, 1, 64), ints(1, 2, 0, 0).view(2, 2)
    _sanity.check_attention(q, cache, table, ints(20, 3), ints(0, 2, 4), None, 2)
    for lengths, offsets, rows, message in ((ints(20, 33), ints(0, 2, 4), None, "passes the block table"), (ints(2, 3), ints(0, 3, 4), None, "longer"),
                                            (ints(2, 3), ints(0, 2, 5), None, "stay within q"), (ints(2, 3), ints(0, 2, 4), ints(0, 2), "rows of"),
                                            (ints(2, 3), ints(1, 2, 4), None, "start at 0")):
        with pytest.raises(RuntimeError, match=message):
            _sanity.check_attention(q, cache, table, lengths, offsets, rows, 2)
    table[0, 1] = 3
    with pytest.raises(RuntimeError, match="not in the cache"):
        _sanity.check_attention(q, cache, table, ints(20, 3), ints(0, 2, 4), None, 2)
    monkeypatch.setenv("PLA_SANITY_CHECK", "1")                         # the entry points ask
    with pytest.raises(RuntimeError, match="negative"):
        paged_kv_plan(PagedKVBlocks.allocate(10, 16, 3, 4, "cpu"), ints(-1), ints(1), token_capacity=4)


def test_the_namespace_is_the_same_module_under_both_names():
    import pla.decode.paged
    import pla_amd.decode.paged
    assert pla.decode.paged is pla_amd.decode.paged
    assert set(pla.decode.paged.__all__) == {"PagedKVBlocks", "PagedKVPlan", "paged_kv_plan", "rotary_frequencies", "fused_qk_norm_rope",
                                             "paged_attention_decode"}


@pytest.mark.parametrize("HKV, D, positions", [(128, 128, 536870864), (1000, 128, 68719440), (2 ** 30, 64, 16)])
def test_a_request_of_more_units_than_32_bits_count_is_refused(HKV, D, positions):
    """A run takes one unit more than it has tiles of 32 keys where wavefronts work alone; the largest number of positions that fits is
    dealt out, and one block more is refused."""
    from pla_amd import _lib
    lib = _lib.load()
    size = lib.pla_paged_attention_workspace_bytes
    units = lambda p: (-(-max(p, 1) // 32) + 1) * HKV
    assert units(positions) > 2 ** 31 - 1 and size(1, HKV, HKV, D, 1, positions) == -1
    assert b"too many heads" in lib.pla_last_error()
    fits = positions - 16
    if units(fits) > 2 ** 31 - 1:
        return
    assert size(1, HKV, HKV, D, 1, fits) > 0
    offsets, lengths, buf = (ctypes.c_int32 * 2)(0, 1), (ctypes.c_int32 * 1)(fits), (ctypes.c_int64 * (7 * 4096))()
    taken = 0
    for worker in range(1025):
        found = lib.pla_paged_attention_segments(offsets, lengths, 1, 1, HKV, HKV, D, 1, fits, worker, buf, 4096)
        assert 0 <= found <= 4096
        taken += sum(buf[7 * i + 4] for i in range(found))
    assert taken == units(fits)


def test_sanity_mode_names_token_rows_that_pass_the_capacity(monkeypatch):
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)
    monkeypatch.setenv("PLA_SANITY_CHECK", "1")
    for query, capacity in ((ints(4, 5), 8), (ints(0, 9), 8), (ints(1, 0), 0)):
        with pytest.raises(RuntimeError, match=r"PLA_SANITY_CHECK \[paged_kv_plan\]: .*token rows pass token_capacity"):
            paged_kv_plan(PagedKVBlocks.allocate(10, 16, 3, 4, "cpu"), ints(1, 2), query, token_capacity=capacity)
    # a batch that fits goes on to the compiled checks, and so does one that asks for more blocks than are free
    for context, query in ((ints(1, 2), ints(4, 4)), (ints(50, 50, 50), ints(4, 4, 0))):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            paged_kv_plan(PagedKVBlocks.allocate(5, 16, 3, 4, "cpu"), context, query, token_capacity=8)


@pytest.mark.parametrize("call, message", [
    (lambda: paged_kv_plan(_blocks(block_size=0), torch.zeros(3, **_INTS), torch.zeros(3, **_INTS), token_capacity=8), "block_size must be positive"),
    (lambda: paged_kv_plan(_blocks(free_count=torch.zeros(2, **_INTS)), torch.zeros(3, **_INTS), torch.zeros(3, **_INTS), token_capacity=8), "free_count must have 1"),
    (lambda: paged_kv_plan(_blocks(block_table=torch.zeros(4, **_INTS)), torch.zeros(3, **_INTS), torch.zeros(3, **_INTS), token_capacity=8), "block_table must be int32"),
    (lambda: paged_kv_plan(_blocks(), torch.zeros(3, 1, **_INTS), torch.zeros(3, **_INTS), token_capacity=8), "context_lens must be an int32"),
    (lambda: paged_kv_plan(_blocks(), torch.zeros(3, **_INTS), torch.zeros(3, device="meta", **_INTS), token_capacity=8), "query_lens must be on the device"),
    (lambda: fused_qk_norm_rope(**_rope_args(slot_mapping=torch.zeros(5, dtype=torch.int64, device="meta"))), "slot_mapping must be on the device of q"),
    (lambda: fused_qk_norm_rope(**_rope_args(slot_mapping=torch.zeros(5, 1, dtype=torch.int64))), "slot_mapping must be an int32 or int64 vector"),
    (lambda: paged_attention_decode(**_attention_args(seq_lens=torch.zeros(3))), "seq_lens must be an int32 or int64 vector"),
    (lambda: paged_attention_decode(**_attention_args(query_start_loc=torch.zeros(0, **_INTS))), "query_start_loc must have 4 entries"),
    (lambda: paged_attention_decode(**_attention_args(block_table=torch.zeros(3, 4, 1, **_INTS))), "block_table must be int32"),
    (lambda: paged_attention_decode(**_attention_args(seq_lens=torch.zeros(3, device="meta", **_INTS))), "seq_lens must be on the device of q"),
])
def test_sanity_mode_leaves_what_is_not_of_its_form_to_the_compiled_checks(call, message, monkeypatch):
    monkeypatch.setenv("PLA_SANITY_CHECK", "1")
    with pytest.raises(RuntimeError, match=message):
        call()


@pytest.mark.parametrize("original_length, beta_slow", [(1, 1.0), (6, 1.0), (25, 4.0), (7, 1.0), (4096, 1.0)])
def test_frequencies_that_hardly_turn_within_the_original_length_are_divided(original_length, beta_slow):
    """All that turn at most beta_slow times, also where that is every one of them."""
    inv, _ = rotary_frequencies(64, 10000.0)
    scaled, _ = rotary_frequencies(64, 10000.0, factor=4.0, original_length=original_length, beta_slow=beta_slow)
    turns, ratio = inv.double() * original_length / (2 * math.pi), (scaled / inv).double()
    few, many = turns <= beta_slow * (1 - 1e-6), turns >= 32.0 * (1 + 1e-6)
    assert few.any() and torch.allclose(ratio[few], torch.full((1,), 0.25, dtype=torch.float64), atol=1e-6)
    assert torch.allclose(ratio[many], torch.ones(1, dtype=torch.float64), atol=1e-6)
