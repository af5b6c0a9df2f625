"""Serving from a paged key/value cache held in 4 bits (MXFP4).

* ``build_block_tables``: a step's request lengths become block tables,
  positions and cache slots, with new blocks off a stack of free ones;
* ``mxfp4_kv_quant_and_cache``: keys and values quantised into the cache;
* ``mxfp4_paged_attention``: causal attention of grouped heads over it, one
  query token per request or many.

The cache is uint8 [num_blocks, num_kv_heads, block_size, D + D / 16], D = 64, 128
or 256, block_size a multiple of 16.  Per block and head it holds block_size x
D / 2 bytes of key codes (E2M1, the even dim in the low nibble), as many of value
codes, then block_size x D / 32 bytes of key scales and as many of value
scales (UE8M0, one per 32 dims); 136 bytes a token and head at D = 128.  A step
runs::

    start, seq_lens, positions, slots, num_free = build_block_tables(
        context_lens, query_lens, block_table, free_blocks, num_free, block_size, max_num_tokens)
    ...                                          # q, k, v of the layer
    mxfp4_kv_quant_and_cache(k, v, kv_cache, slots)
    out, lse = mxfp4_paged_attention(q, kv_cache, block_table, seq_lens, scale, query_start_loc=start)

The argument checks, output allocation and launch run in C++
(``torch_ops.cpp``) through the C ABI ``fgv_build_block_tables``,
``fgv_mxfp4_kv_quant_and_cache`` and ``fgv_mxfp4_paged_attention``, on torch's
current stream of the tensors' device; a failed check raises AssertionError.
Nothing is read back to the host, so a step can be captured in a graph.
Inference only: a tensor that requires a gradient (in grad mode) or carries a
forward-mode tangent is refused, and so are lazily negated views and tensors
without memory.
"""
from typing import Optional, Tuple

import torch

from .. import _native


def build_block_tables(
    context_lens: torch.Tensor,
    query_lens: torch.Tensor,
    block_table: torch.Tensor,
    free_blocks: torch.Tensor,
    num_free: torch.Tensor,
    block_size: int,
    max_num_tokens: int,
    pad_id: int = -1,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Block tables, positions and slots of a step.

    Args:
        context_lens: int32 [R], tokens of each request that are cached already.
        query_lens: int32 [R], its new tokens (0: it sits the step out); negative
            lengths count as 0.
        block_table: int32 [R, W], contiguous rows of any row stride, written in
            place: the columns from ceil(context / block_size) on that the new
            tokens need get blocks, in the order of requests and columns, and -1
            where none is left.  Other columns are left as they are: a column of
            -1 is not filled by a later step, whose context holds it.
        free_blocks: int32 [F], a stack of block ids, free_blocks[num_free - 1] on
            top.  Not written: blocks of finished requests are put back by the
            caller, behind the num_free of them, with num_free raised.
        num_free: int32, one element: how many of them are free.
        block_size: tokens per block.
        max_num_tokens: rows of the step's buffers; new tokens past it, counted
            over the requests in order, are dropped (query lengths shortened).
        pad_id: the slot of rows without one.

    Returns:
        query_start_loc int32 [R + 1]; seq_lens int32 [R], context plus new
        tokens; positions int64 [max_num_tokens] (0 behind the last token);
        slot_mapping int64 [max_num_tokens], block * block_size + position %
        block_size, pad_id behind the last token and for tokens without a block
        (none left, a negative entry, or past the table's width); num_free int32
        [1] for the next step, negative where blocks were missing.
    """
    rc, out = _native.torch_ext().build_block_tables(context_lens, query_lens, block_table, free_blocks, num_free,
                                                     int(block_size), int(max_num_tokens), int(pad_id))
    if rc:
        _native.raise_status(rc, "build_block_tables")
    return out


def mxfp4_kv_quant_and_cache(k: torch.Tensor, v: torch.Tensor, kv_cache: torch.Tensor,
                             slot_mapping: torch.Tensor) -> None:
    """kv_cache[slot] = MXFP4 of k[t] and v[t], in place.

    Args:
        k, v: [T, num_kv_heads, D] bfloat16 or float16, contiguous rows of any
            other strides.
        kv_cache: see the module; each block contiguous, blocks of any stride.
        slot_mapping: int64 [<= T]; negative slots and slots past the cache are
            skipped.  Two tokens must not have the same slot.

    Per 32 values with largest magnitude a, the scale is 2^e, e = ceil(log2(a / 6))
    within -126 and 125, and the codes are the nearest to x / 2^e, ties to the
    even code.  A block that holds a NaN or an infinity is stored as NaN (byte
    255, codes 0).
    """
    rc = _native.torch_ext().mxfp4_insert(k, v, kv_cache, slot_mapping)
    if rc:
        _native.raise_status(rc, "mxfp4_kv_quant_and_cache")


def mxfp4_paged_attention(
    q: torch.Tensor,
    kv_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    softmax_scale: float,
    *,
    query_start_loc: Optional[torch.Tensor] = None,
    max_query_len: Optional[int] = None,
    max_seq_len: Optional[int] = None,
    window_size: Optional[int] = None,
    attn_sink: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Causal attention of grouped heads over an MXFP4 cache.

    Args:
        q: [T, Hq, D] bfloat16 or float16, contiguous rows of any other strides;
            Hq a multiple of the cache's heads.
        kv_cache: see the module.
        block_table: int32 [R, W], contiguous rows.  Entries that are not a block
            of the cache are as keys that nobody sees.
        seq_lens: int32 [R], each request's keys, the step's own tokens among them.
        softmax_scale: factor of q . k.
        query_start_loc: int32 [R + 1], the rows of q that are each request's: its
            last tokens.  An end before its start is a request without tokens;
            requests must not share rows (if some do, out and lse are undefined
            in all rows of requests; nothing else is written).  None: one token
            per request (T = R).
        max_query_len, max_seq_len: the most query tokens and keys of a request,
            as far as the caller knows them (T and W * block_size otherwise); they
            only choose how the work is cut.
        window_size: a token sees its own key and the window_size - 1 before it;
            None: all before it.
        attn_sink: float32 [Hq], added to each row's sum as exp(sink) (not to lse).
        out: like q, apart from the inputs; a new tensor if not given.  Rows that
            are no request's are left as they are (undefined in a new tensor).

    Returns:
        out [T, Hq, D] in q's type and lse [T, Hq] float32, the natural logarithm
        of each row's sum (to the accuracy of the scores, not of float32: errors of
        1e-6 to 5e-6 rms for bf16 queries, a tenth of that for fp16).  A row that sees no key has out 0 and lse +inf.  NaN
        where a row sees a key or value block that is NaN (byte 255; of values
        253 and 254 too, which no op here writes), or its query holds a NaN or
        an infinity.
    """
    rc, out, lse = _native.torch_ext().mxfp4_attention(
        q, kv_cache, block_table, seq_lens, float(softmax_scale), query_start_loc, max_query_len, max_seq_len,
        window_size, attn_sink, out)
    if rc:
        _native.raise_status(rc, "mxfp4_paged_attention")
    return out, lse


__all__ = ["build_block_tables", "mxfp4_kv_quant_and_cache", "mxfp4_paged_attention"]
