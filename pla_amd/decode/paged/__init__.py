"""Paged softmax attention next to the linear-attention layers (``pla.decode.paged``).

Many of the models that the rest of this package serves put softmax-attention layers between their linear-attention layers.  Both see the
same serving step: the same requests, windows of draft tokens and ``query_start_loc``.  This namespace holds what such a step
needs besides the linear-attention operators; it has no counterpart in the reference.

``paged_kv_plan``           block tables, slot map, positions and offsets of a step, from the requests' lengths, on the GPU.  Its
                            ``query_start_loc`` is the one ``kda_replay_verify`` takes, its block table the one that
                            ``KDAReplayCommitContext.commit`` takes in align mode.
``fused_qk_norm_rope``      norms of queries and keys for each head, position rotation and write into the paged cache, of 16 or 8 bits.
``rotary_frequencies``      the rotation's frequencies, plain or scaled for long contexts.
``paged_attention_decode``  attention of one new token, or of a window of up to 32 draft tokens, over the paged cache, and over a prefix
                            that all requests share.

Longer windows, prompts and parts of them: ``pla.prefill.attention.paged_attention_prefill``.

All checks live in the compiled layer (``pla.decode.paged._C``), raise RuntimeError and come before any launch.  Nothing is read
back from the device, so every call can be captured in a graph.  ``PLA_SANITY_CHECK=1`` adds checks of values (they read device
memory and are skipped under capture).
"""

import math
import os
from dataclasses import dataclass
from typing import Optional

import torch

from ... import _lib

__all__ = ["PagedKVBlocks", "PagedKVPlan", "paged_kv_plan", "rotary_frequencies", "fused_qk_norm_rope", "paged_attention_decode"]

_native = None


def _compiled():
    global _native
    if _native is None:
        _lib.load()                              # a missing library is reported as such
        import importlib
        try:
            _native = importlib.import_module("._C", __name__)
        except ModuleNotFoundError as exc:
            if exc.name is None or not exc.name.endswith("_C"):
                raise
            raise ImportError("pla.decode.paged._C is not built: run `python -m pla_amd.build`") from None
    return _native


def _sanity_enabled():
    return os.environ.get("PLA_SANITY_CHECK", "0") == "1"


@dataclass(frozen=True)
class PagedKVBlocks:
    """Which blocks of a paged cache belong to which request: block_table [requests, blocks a request] int32, of whose rows the
    first held_blocks [requests] int32 entries count, and the other blocks as a stack, free_blocks [capacity] int32 of height
    free_count [1] int32, with places for all blocks (one that comes back to a full stack is nobody's from then on).
    ``paged_kv_plan`` updates all four in place."""
    block_table: torch.Tensor
    held_blocks: torch.Tensor
    free_blocks: torch.Tensor
    free_count: torch.Tensor
    block_size: int

    @classmethod
    def allocate(cls, num_blocks, block_size, max_num_reqs, max_blocks_per_req, device, first_block=1):
        """All blocks from ``first_block`` on free, to be handed out in ascending order.  Block 0 is by default nobody's: table
        entries past a request's blocks are 0, and the linear-attention caches take it as the null block."""
        if not 0 <= first_block <= num_blocks or num_blocks > 2 ** 30:
            raise ValueError("allocate requires 0 <= first_block <= num_blocks <= 2**30")
        if block_size < 1 or max_num_reqs < 0 or max_blocks_per_req < 0 or max_blocks_per_req * block_size > 2 ** 30:
            raise ValueError("allocate requires block_size >= 1, counts >= 0 and at most 2**30 positions a request")
        ints = dict(dtype=torch.int32, device=device)
        return cls(block_table=torch.zeros(max_num_reqs, max_blocks_per_req, **ints), held_blocks=torch.zeros(max_num_reqs, **ints),
                   free_blocks=torch.arange(num_blocks - 1, first_block - 1, -1, **ints),
                   free_count=torch.full((1,), num_blocks - first_block, **ints), block_size=int(block_size))


@dataclass(frozen=True)
class PagedKVPlan:
    """A step's query_start_loc [N+1] int32, seq_lens [N] int32, positions [token_capacity] int32 and slot_mapping
    [token_capacity] int64."""
    query_start_loc: torch.Tensor
    seq_lens: torch.Tensor
    positions: torch.Tensor
    slot_mapping: torch.Tensor

    @classmethod
    def allocate(cls, num_reqs, token_capacity, device):
        ints = dict(dtype=torch.int32, device=device)
        return cls(torch.zeros(num_reqs + 1, **ints), torch.zeros(num_reqs, **ints), torch.zeros(token_capacity, **ints),
                   torch.full((token_capacity,), -1, dtype=torch.int64, device=device))


def paged_kv_plan(blocks, context_lens, query_lens, request_indices=None, *, token_capacity, out=None):
    """Plans a step in which entry n of the batch brings ``query_lens[n]`` new tokens to ``context_lens[n]`` cached ones.

    Its row of the block table is ``request_indices[n]`` (at most 8192 rows then), or n.  Blocks that the row holds beyond the
    sum of the two go back on the free stack first - after a verify the context is what was accepted, a finished request has
    0 and 0 - then missing ones come off it.  An entry gets all it misses or nothing: it is granted if the running sum of what
    entries ask for, up to and with its own, is on the stack.  An entry is refused as well if a length is negative, if its
    positions pass the row, if an earlier entry has the same row, if its row does not exist, or if its token rows pass
    ``token_capacity``.  A refused entry keeps its blocks and has sequence length 0 (attention gives zeros), position 0 and slot
    -1 (nothing is stored).  Rows behind the batch get position 0 and slot -1.

    context_lens, query_lens, request_indices: int32 or int64 [N].  ``token_capacity``: rows of the step's tensors.  Returns a
    PagedKVPlan, ``out`` if one is given; neither it nor ``blocks`` may share memory with an input.
    """
    if _sanity_enabled():
        from ._sanity import check_plan
        check_plan(blocks, context_lens, query_lens, request_indices, token_capacity)
    outs = (None,) * 4 if out is None else (out.query_start_loc, out.seq_lens, out.positions, out.slot_mapping)
    made = _compiled().paged_kv_plan(blocks.block_table, blocks.held_blocks, blocks.free_blocks, blocks.free_count, blocks.block_size,
                                     context_lens, query_lens, request_indices, token_capacity, *outs)
    return PagedKVPlan(*made) if out is None else out


def rotary_frequencies(rotary_dim, base=10000.0, *, factor=1.0, original_length=None, beta_fast=32.0, beta_slow=1.0, device=None):
    """(inv_freq [rotary_dim / 2] float32, attention_factor) of a rotation.

    Plain (``factor`` 1): base^(-2 i / rotary_dim), and 1.  For contexts ``factor`` times as long as the ``original_length`` that a
    model was trained on, as in YaRN (Peng et al., 2023): frequencies that turn at least ``beta_fast`` times within the original
    length stay, those that turn at most ``beta_slow`` times are divided by the factor, a linear ramp over i in between, and the
    attention factor is 0.1 ln(factor) + 1.
    """
    if rotary_dim < 2 or rotary_dim % 2 or base <= 1 or factor < 1:
        raise ValueError("rotary_frequencies requires an even rotary_dim, base > 1 and factor >= 1")
    inv_freq = float(base) ** -(torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    if factor == 1:
        return inv_freq.to(torch.float32).to(device), 1.0
    if original_length is None or original_length < 1 or not beta_fast > beta_slow > 0:
        raise ValueError("a scaled rotation requires original_length >= 1 and beta_fast > beta_slow > 0")

    def index_of(turns):                         # i whose frequency turns that often within the original length
        return rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
    low, high = max(math.floor(index_of(beta_fast)), 0), min(math.ceil(index_of(beta_slow)), rotary_dim - 1)
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
    ramp[i >= index_of(beta_slow)] = 1           # also where that is below the first
    inv_freq = inv_freq * (1 - ramp) + inv_freq / factor * ramp
    return inv_freq.to(torch.float32).to(device), 0.1 * math.log(factor) + 1.0


def fused_qk_norm_rope(q, k, positions=None, *, q_weight=None, k_weight=None, eps=1e-6, weight_offset=0.0, inv_freq=None,
                       attention_factor=1.0, interleaved=False, q_out=None, k_out=None, v=None, k_cache=None, v_cache=None,
                       slot_mapping: Optional[torch.Tensor] = None, k_scales=None, v_scales=None):
    """Norms the heads of q [T, HQ, D] and k [T, HKV, D], turns them by their positions, stores k and v [T, HKV, D].

    bf16 or fp16, D 64, 128 or 256; rows are views with any 16-byte aligned token and head strides.  All in float32, one rounding.

    norm      x rsqrt(mean(x^2) + eps) (weight + weight_offset) where a weight [D] (of q's type or float32) is given.
    rotation  of the first ``2 * inv_freq.numel()`` channels (a multiple of 16) by positions [T] (int32 or int64) times inv_freq
              float32, cosine and sine times ``attention_factor``; pairs are (i, i + half) or, ``interleaved``, (2i, 2i + 1).
              Angles are exact to float32 at any position up to 2^53.  No inv_freq: no rotation.
    store     with k_cache (and v, v_cache) [blocks, block_size, HKV, D] and slot_mapping [T] (int32 or int64), token t goes to
              slot ``block * block_size + place``; a slot that is negative or past the cache is nowhere.  No two tokens may
              name one slot.
    8 bits    with k_scales (and v_scales) [blocks, HKV, block_size] float32 the caches are torch.float8_e4m3fn: a head of a token is
              stored as x / scale, rounded once from float32 to nearest, with scale max(largest |x|, 1e-30) / 448 beside it: off by
              2^-4 of itself or 2^-10 of the scale, whichever is more.  A NaN stays one, an infinity makes what its head stands for NaN.

    Returns (q_out, k_out): ``k_out`` is made if neither it nor a cache is given, and else what was passed.  q_out and k_out may be
    q and k themselves (the same rows), and share memory with nothing else.
    """
    if _sanity_enabled():
        from ._sanity import check_slots
        check_slots(slot_mapping, k_cache)
    return _compiled().fused_qk_norm_rope(q, k, positions, q_weight, k_weight, eps, weight_offset, inv_freq, attention_factor,
                                          interleaved, q_out, k_out, v, k_cache, v_cache, slot_mapping, k_scales, v_scales)


def paged_attention_decode(q, k_cache, v_cache, block_table, seq_lens, *, query_start_loc=None, request_indices=None,
                           max_query_len=1, scale=None, output_gate=None, out=None, k_scales=None, v_scales=None,
                           prefix_blocks=None, prefix_len=None):
    """Attention of new tokens over a paged cache that holds their keys and values already.

    q [T, HQ, D] (bf16 or fp16; D 64, 128 or 256; HQ a multiple of HKV), caches [blocks, block_size, HKV, D] of one shape and
    strides (block_size a multiple of 16; channels dense, the other strides any multiples of 8: tokens or heads first),
    block_table int32 [requests, blocks a request], seq_lens [N] the cached tokens with the window.

    Without ``query_start_loc`` row n is the one new token of request n.  With it (int32 or int64 [N+1]) rows
    query_start_loc[n] .. query_start_loc[n+1] - 1 are request n's window, at most ``max_query_len`` (up to 32) tokens; token j of
    a window of m sees the first seq_lens[n] - m + j + 1 positions.  A request whose window is empty, longer or not within q is
    passed over, and rows of no request are left as they are (anything, where ``out`` is made here); no two windows may share a row.
    A row that sees nothing is zeros.  Positions whose block is no block of the cache, or past the table, are left out; what the
    cache holds behind a request's end never counts, and a draft token's key or value that is infinite or NaN reaches no token
    before it.
    ``request_indices`` [N]: rows of the block table, n without it.

    Caches of 8-bit numbers (torch.float8_e4m3fn) come with ``k_scales`` and ``v_scales`` as ``fused_qk_norm_rope`` writes them, of common
    strides, none negative.  Numbers and scales are used as they are, without a rounding of their product.

    A prefix that all requests share, such as one instruction text, stands in blocks of its own, which no request's row of the table names:
    the first ``prefix_len`` [1] (int32 or int64, on the device) positions of ``prefix_blocks`` int32 [pages].  Every row that sees a
    position of its own sees the whole prefix too, before them (positions of new tokens count on from its end); keys and values of the
    prefix are read once for the whole batch.  Its weights are rounded once to q's type.  Not with 8-bit caches.  Rows of q that belong
    to no request are taken over the prefix as well, to no result: keep them few, and finite (else parts of the prefix are gone through twice).

    scale (default D^-0.5) applies to the scores; output_gate [T, HQ, D] multiplies the result by its sigmoid.  Scores, their
    maxima and sums and the outputs are float32; weights meet the values in two parts of q's type (off by 2^-16 of themselves at most,
    fp16 2^-22; over 8-bit caches 2^-16), outputs are rounded once.  A key of a 16-bit cache that a row sees has a weight of at least 2^-125
    (fp16 2^-37) of the row's largest, so an infinite value there counts.  Sums of weights no larger than one times the values have
    to stay within float32.  Returns ``out`` [T, HQ, D], which shares memory with no input.  Results do not depend on timing.
    """
    if _sanity_enabled():
        from ._sanity import check_attention, check_prefix
        check_attention(q, k_cache, block_table, seq_lens, query_start_loc, request_indices, max_query_len)
        check_prefix(k_cache, prefix_blocks, prefix_len)
    return _compiled().paged_attention_decode(q, k_cache, v_cache, block_table, seq_lens, query_start_loc, request_indices,
                                              max_query_len, scale, output_gate, out, k_scales, v_scales, prefix_blocks, prefix_len)
