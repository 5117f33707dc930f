"""Filling a paged KV cache and choosing the blocks that a decode step reads.

The reference attends ready block tables and 16-bit pages
(interface.py:643-728) and leaves it to its caller to make them.  A step of a
serving loop over this package's paged decode is

    slots, cu_seqlens, head = paged_kvcache_allocate(block_table, lens, new_lens, free_blocks, ...)
    paged_kvcache_append(key, value, k_cache, v_cache, slots, k_scale=..., v_scale=..., key_bounds=...)
    index = paged_kvcache_select(query, key_bounds, block_table, lens + new_lens, 64, block_size=...)
    out = flash_attention_decode_paged(query, k_cache, v_cache, block_table, lens + new_lens,
                                       k_scale=..., v_scale=..., block_index=index)

with every argument on the GPU: nothing waits for the host, and the whole step
can be captured into a HIP graph.  All of it is inference-only.

The native operators check what they are given before anything is launched; a
call that they refuse is looked over again here, for this package's messages.
(All the checks in Python took longer than the kernels of a small step.)
"""

import torch

from . import _native
from ._validation import (
    validate_allocate_inputs,
    validate_append_inputs,
    validate_block_size,
    validate_count,
    validate_inference_only,
    validate_select_inputs,
)


def paged_kvcache_allocate(block_table, context_lens, new_lens, free_blocks, *, free_head=None, block_size,
                           num_tokens):
    """Give each sequence the blocks its new tokens need; slots of the tokens.

    Args:
        block_table: int32 ``(batch, max_blocks)``; the entries of new blocks
            are written in place, the others are left as they are.
        context_lens: int32 ``(batch,)`` tokens already in the cache.
        new_lens: int32 ``(batch,)`` tokens that come next, packed sequence
            after sequence.  Negative lengths count as 0.
        free_blocks: int32 ``(n,)`` ids of free blocks, handed out in order.
        free_head: int32 ``(1,)`` position of the first free block that was
            not handed out yet; default 0.
        block_size: tokens of a block, a power of two up to 256.
        num_tokens: rows of the slot map, at least the sum of ``new_lens`` for
            every token to have one.

    Returns:
        ``(slot_mapping, cu_seqlens, next_head)``: int64 ``(num_tokens,)``
        slots ``page * block_size + position``, -1 for rows past the last
        token and tokens without a block (``free_blocks`` used up, or past
        ``max_blocks``); int32 ``(batch + 1,)`` running sums of the new
        lengths, as :func:`flash_attention_varlen` takes them; int32 ``(1,)``
        ``free_head`` for the next call (beyond ``n`` by the blocks that were
        missing).  The sums and ``next_head`` stop at 2^31 - 1.  ``context_lens`` and ``free_head`` are not modified, and
        the same call again gives the same tables.
    """
    validate_block_size(block_size)
    validate_count("num_tokens", num_tokens, 0)
    try:
        return _native.ops().paged_allocate(block_table, context_lens, new_lens, free_blocks, free_head, block_size,
                                            num_tokens)
    except (RuntimeError, TypeError):
        validate_allocate_inputs(block_table, context_lens, new_lens, free_blocks, free_head)
        raise


def paged_kvcache_append(key, value, k_cache, v_cache, slot_mapping, *, k_scale=None, v_scale=None, key_bounds=None):
    """Write new keys and values into a paged cache, in place.

    Args:
        key, value: float16 or bfloat16 ``(tokens, kv_heads, head_dim)``.
        k_cache, v_cache: ``(num_blocks, block_size, kv_heads, head_dim)`` of
            the keys' dtype, ``torch.float8_e4m3fn`` or ``torch.int8``.
        slot_mapping: int64 ``(tokens,)`` as :func:`paged_kvcache_allocate`
            gives it.  Rows whose slot lies outside the cache are dropped.
            The others have slots of their own, and those of one block lie
            within ``block_size`` consecutive rows with none of another block
            between them (sequence after sequence, not position after
            position): one wave does all rows of a block.
        k_scale, v_scale: float32 ``(num_blocks, kv_heads)``, required for
            8-bit caches: what the codes of a block and head are multiplied by.
        key_bounds: optional ``(num_blocks, kv_heads, 2, head_dim)`` of the
            keys' dtype: least and greatest key of each block and head, for
            :func:`paged_kvcache_select`.

    A block whose position 0 is written starts afresh: its scales and bounds
    come from the new rows.  Otherwise the rows below the lowest new one are
    taken as valid; scales only grow, to powers of two that hold the largest
    new value, and a block whose scale grew has its valid rows rounded to the
    new scale.  Values are rounded to nearest, ties to even.  Infinities are
    stored as the largest code and have no part in the scale; NaN stays NaN
    (int8: 0) and has no part in scale or bounds.
    """
    for written in (k_cache, v_cache, k_scale, v_scale, key_bounds):
        if isinstance(written, torch.Tensor):
            validate_inference_only(written)
    try:
        _native.ops().paged_append(key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale, key_bounds)
    except (RuntimeError, TypeError):
        validate_append_inputs(key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale, key_bounds)
        raise


def paged_kvcache_select(query, key_bounds, block_table, context_lens, num_selected, *, block_size, keep_first=0,
                         keep_last=1):
    """Choose the blocks of each sequence and KV head that a query needs most.

    A block's score is an upper bound of the logits its keys can have,
    ``sum_d max(q_d, 0) * hi_d + min(q_d, 0) * lo_d`` (summed in 64 bits), the
    largest over the query heads of the KV head and over the query rows; NaN
    counts as infinity.

    Args:
        query: ``(batch, q_heads, head_dim)`` or ``(batch, q_heads, rows, head_dim)``.
        key_bounds: ``(num_blocks, kv_heads, 2, head_dim)`` of the query's
            dtype, kept by :func:`paged_kvcache_append`.
        block_table, context_lens: as in :func:`flash_attention_decode_paged`.
        num_selected: blocks to choose for each sequence and KV head.
        block_size: tokens of a block.
        keep_first, keep_last: first and last blocks of a sequence that are
            always chosen (together at most ``num_selected``).

    Returns:
        int32 ``(batch, kv_heads, num_selected)`` logical blocks in ascending
        order, -1 behind them where a sequence has fewer; the
        ``block_index`` of the paged decode.  Equal scores go to the lower
        index.
    """
    validate_block_size(block_size)
    validate_count("num_selected", num_selected, 1)
    validate_count("keep_first", keep_first, 0)
    validate_count("keep_last", keep_last, 0)
    if keep_first + keep_last > num_selected:
        raise ValueError("keep_first + keep_last must not exceed num_selected")
    try:
        validate_inference_only(query, key_bounds)
        return _native.ops().paged_select(query, key_bounds, block_table, context_lens, num_selected, block_size,
                                          keep_first, keep_last)
    except (RuntimeError, TypeError, AttributeError):
        validate_select_inputs(query, key_bounds, block_table, context_lens)
        raise
