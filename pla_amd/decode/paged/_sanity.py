"""Checks of values under ``PLA_SANITY_CHECK=1``: what the operators would pass over or leave out without a word.

Every rejection raises ``RuntimeError("PLA_SANITY_CHECK [op]: ...")`` before anything is launched.  The checks read device memory
and are skipped while a stream is being captured.  A plan's entry that the free blocks do not suffice for is no mistake: its sequence
length of 0 is the answer that a scheduler waits for.
"""

import torch


def _fail(op, msg):
    raise RuntimeError(f"PLA_SANITY_CHECK [{op}]: {msg}")


def _capturing():
    return torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()


def _formed(table, *vectors):
    """Whether a call's tables and vectors have values to look at; what is not of its form the compiled layer refuses."""
    return ((table is None or (table.dim() == 2 and not table.is_meta)) and
            all(v is None or (v.dim() == 1 and v.dtype in (torch.int32, torch.int64) and not v.is_meta) for v in vectors))


def check_plan(blocks, context_lens, query_lens, request_indices, token_capacity=None):
    if _capturing() or not _formed(blocks.block_table, blocks.held_blocks, blocks.free_blocks, blocks.free_count, context_lens, query_lens,
                                   request_indices) or blocks.block_size < 1 or blocks.free_count.numel() != 1:
        return
    op, (rows, cols) = "paged_kv_plan", blocks.block_table.shape
    context, query = context_lens.tolist(), query_lens.tolist()
    if any(x < 0 for x in context + query):
        _fail(op, "lengths must not be negative")
    if token_capacity is not None and sum(query) > token_capacity:
        _fail(op, "the batch's token rows pass token_capacity")
    if any(-(-(c + q) // blocks.block_size) > cols for c, q in zip(context, query)):
        _fail(op, "a request's positions pass its row of the block table")
    if request_indices is not None:
        index = request_indices.tolist()
        if len(set(index)) != len(index) or any(not 0 <= x < rows for x in index):
            _fail(op, "request_indices must be different rows of the block table")
    height, held = blocks.free_count.item(), blocks.held_blocks.tolist()
    if not 0 <= height <= blocks.free_blocks.numel() or any(not 0 <= h <= cols for h in held):
        _fail(op, "free_count and held_blocks must lie within their tables")
    owned = blocks.free_blocks[:height].tolist()
    for row, h in zip(blocks.block_table.tolist(), held):
        owned += row[:h]
    if len(set(owned)) != len(owned):
        _fail(op, "a block is held twice")


def check_slots(slot_mapping, k_cache):
    if slot_mapping is None or k_cache is None or _capturing() or not _formed(None, slot_mapping) or k_cache.dim() < 2:
        return
    slots = [x for x in slot_mapping.tolist() if x >= 0]
    if any(x >= k_cache.size(0) * k_cache.size(1) for x in slots):
        _fail("fused_qk_norm_rope", "a slot is past the cache")
    if len(set(slots)) != len(slots):
        _fail("fused_qk_norm_rope", "two tokens name one slot")


def check_attention(q, k_cache, block_table, seq_lens, query_start_loc, request_indices, max_query_len, op="paged_attention_decode"):
    if (_capturing() or not _formed(block_table, seq_lens, query_start_loc, request_indices) or k_cache.dim() < 2 or q.dim() < 1 or
            k_cache.size(1) < 1 or (query_start_loc is not None and query_start_loc.numel() != seq_lens.numel() + 1)):
        return
    rows, cols = block_table.shape
    blocks, block_size = k_cache.shape[:2]
    lengths = seq_lens.tolist()
    offsets = list(range(len(lengths) + 1)) if query_start_loc is None else query_start_loc.tolist()
    index = list(range(len(lengths))) if request_indices is None else request_indices.tolist()
    if offsets[0] != 0 or any(b < a for a, b in zip(offsets, offsets[1:])) or offsets[-1] > q.size(0):
        _fail(op, "query_start_loc must start at 0, not decrease and stay within q")
    if max_query_len is not None and any(b - a > max_query_len for a, b in zip(offsets, offsets[1:])):
        _fail(op, "a window is longer than max_query_len")
    if any(not 0 <= x < rows for x in index):
        _fail(op, "request_indices must be rows of the block table")
    table = block_table.tolist()
    for row, length in zip(index, lengths):
        if not 0 <= length <= cols * block_size:
            _fail(op, "a sequence length is negative or passes the block table")
        if any(not 0 <= b < blocks for b in table[row][:-(-length // block_size)]):
            _fail(op, "a block of the table is not in the cache")


def check_prefix(k_cache, prefix_blocks, prefix_len):
    if (prefix_blocks is None or prefix_len is None or _capturing() or not _formed(None, prefix_blocks, prefix_len) or prefix_len.numel() != 1 or
            k_cache.dim() < 2 or k_cache.size(1) < 1):
        return
    op, length, block_size = "paged_attention_decode", prefix_len.item(), k_cache.size(1)
    if not 0 <= length <= prefix_blocks.numel() * block_size:
        _fail(op, "prefix_len is negative or passes prefix_blocks")
    if any(not 0 <= b < k_cache.size(0) for b in prefix_blocks[:-(-length // block_size)].tolist()):
        _fail(op, "a block of the prefix is not in the cache")


def check_packed(q, k, cu_seqlens, cu_seqlens_k):
    if _capturing() or not _formed(None, cu_seqlens, cu_seqlens_k) or q.dim() < 1 or k.dim() < 1 or cu_seqlens.numel() < 1:
        return
    op = "packed_attention_fwd"
    offsets = cu_seqlens.tolist()
    key_offsets = offsets if cu_seqlens_k is None else cu_seqlens_k.tolist()
    if len(key_offsets) != len(offsets):
        return
    for name, x, rows in (("cu_seqlens", offsets, q.size(0)), ("cu_seqlens_k", key_offsets, k.size(0))):
        if x[0] != 0 or any(b < a for a, b in zip(x, x[1:])) or x[-1] > rows:
            _fail(op, f"{name} must start at 0, not decrease and stay within its tensor")
    if any(d - c < b - a for a, b, c, d in zip(offsets, offsets[1:], key_offsets, key_offsets[1:])):
        _fail(op, "a sequence has fewer keys than tokens")
