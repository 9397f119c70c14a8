"""Softmax attention over whole prompts (``pla.prefill.attention``), for the layers between the linear-attention ones; no counterpart in the
reference.

``packed_attention_fwd``     of packed sequences over their own dense keys and values.
``paged_attention_prefill``  of packed windows of any length over the paged cache of ``pla.decode.paged``, which holds their keys.

Both are causal.  The compiled layer is the one of ``pla.decode.paged``.  Checks raise RuntimeError before any launch; nothing is read
back from the device, so a call can be captured in a graph.
"""

from ...decode import paged as _paged

__all__ = ["packed_attention_fwd", "paged_attention_prefill"]


def packed_attention_fwd(q, k, v, cu_seqlens, *, cu_seqlens_k=None, scale=None, output_gate=None, out=None):
    """softmax(scale q k^T) v of every sequence, causal, with the query heads in groups over the key-value heads.

    q [T, HQ, D], k and v [K, HKV, D] (bf16 or fp16; D 64, 128 or 256; HQ a multiple of HKV; dense channels, any 16-byte aligned token
    and head strides).  Sequence n has token rows cu_seqlens[n] .. cu_seqlens[n+1] - 1 (int32 or int64 [N+1]), and the same rows of k
    and v, or those of ``cu_seqlens_k`` where it has other, say earlier, keys too: token j of m with n keys sees the first n - m + j + 1.
    A row that sees nothing is zeros.  A sequence that is empty or not within the tensors is passed over, and rows of no sequence are
    left as they are (anything, where ``out`` is made here); no two sequences may share a row of q.  A key or value that is infinite or
    NaN reaches no token before it.  (``PLA_SANITY_CHECK=1`` takes a sequence of fewer keys than tokens for a mistake and names it.)

    scale (default D^-0.5) applies to the scores; output_gate [T, HQ, D] multiplies the result by its sigmoid.  Softmax statistics and
    sums are float32; weights are rounded once to q's type before they meet the values (off by half a step of it, as much as the
    output's own rounding), outputs once.  Returns ``out`` [T, HQ, D], which shares memory with no input.  Results do not depend on
    timing.
    """
    if _paged._sanity_enabled():
        from ...decode.paged._sanity import check_packed
        check_packed(q, k, cu_seqlens, cu_seqlens_k)
    return _paged._compiled().packed_attention_fwd(q, k, v, cu_seqlens, cu_seqlens_k, scale, output_gate, out)


def paged_attention_prefill(q, k_cache, v_cache, block_table, seq_lens, query_start_loc, *, request_indices=None, scale=None,
                            output_gate=None, out=None):
    """The same for windows of any length over a paged cache that holds their keys and values already: prompts, parts of prompts whose
    earlier tokens are cached, or both in one batch.

    Arguments, masks and what becomes of entries that are out of range are those of ``pla.decode.paged.paged_attention_decode``, with
    ``query_start_loc`` [N+1] always given, no longest window, and caches of q's type.  Windows of up to 32 tokens are better off there: it is made for few
    rows, and keeps twice the digits of a weight.
    """
    if _paged._sanity_enabled():
        from ...decode.paged._sanity import check_attention
        check_attention(q, k_cache, block_table, seq_lens, query_start_loc, request_indices, None, op="paged_attention_prefill")
    return _paged._compiled().paged_attention_prefill(q, k_cache, v_cache, block_table, seq_lens, query_start_loc, request_indices, scale,
                                                      output_gate, out)
