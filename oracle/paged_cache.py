"""Paged KV cache operators from their definitions: plain loops, numpy, 64 bits.

`allocate`, `append`, `select` and `attend` are what the package's
paged_kvcache_allocate / _append / _select and its paged decode with block
scales and a block index are compared with.  Arrays hold values: codes of an
8-bit cache as the numbers they stand for.
"""

import math

import numpy as np

TOP = {"e4m3": 448.0, "int8": 127.0}
LEAST_EXPONENT = -100


def allocate(block_table, context_lens, new_lens, free_blocks, free_head, block_size, num_tokens):
    """-> (slots, cu_seqlens, next_head, block_table after)."""
    table = np.array(block_table)
    blocks = table.shape[1]
    head = max(int(free_head), 0)
    slots, cu = [], [0]
    for b, (ctx, new) in enumerate(zip(context_lens, new_lens)):
        ctx, new = max(int(ctx), 0), max(int(new), 0)
        have = -(-min(ctx, blocks * block_size) // block_size)
        for pos in range(ctx, ctx + new):
            at = pos // block_size
            if at >= blocks:
                slots.append(-1)
                continue
            if at >= have:
                table[b, at] = free_blocks[head] if head < len(free_blocks) else -1
                head += 1
                have = at + 1
            page = int(table[b, at])
            slots.append(page * block_size + pos % block_size if page >= 0 else -1)
        cu.append(cu[-1] + new)
    slots = (slots + [-1] * num_tokens)[:num_tokens]
    return np.array(slots, dtype=np.int64), np.array(cu), head, table


def scale_for(amax, cache):
    """Least power of two 2^e, e >= LEAST_EXPONENT, with amax <= top * 2^e."""
    e = LEAST_EXPONENT
    if amax > 0:
        m, x = math.frexp(amax / TOP[cache])  # amax / top = m 2^x, m in [0.5, 1)
        e = max(x - 1 if m == 0.5 else x, LEAST_EXPONENT)
        while TOP[cache] * 2.0 ** e < amax:  # (the division above was rounded)
            e += 1
        while e > LEAST_EXPONENT and TOP[cache] * 2.0 ** (e - 1) >= amax:
            e -= 1
    return 2.0 ** e


def to_code(x, cache):
    """Nearest value of the 8-bit type, ties to even; NaN stays NaN (int8: 0)."""
    x = np.clip(np.asarray(x, dtype=np.float64), -TOP[cache], TOP[cache])
    if cache == "int8":
        return np.where(np.isnan(x), 0.0, np.rint(x))
    exponent = np.maximum(np.frexp(np.where(np.isnan(x), 1.0, x))[1] - 1, -6)
    step = np.exp2(exponent - 3.0)
    return np.rint(x / step) * step


def append(rows, cache, scale, bounds, slots, kind):
    """One of K or V: `rows` (tokens, heads, dim), `cache` (blocks, block_size,
    heads, dim), `scale` (blocks, heads) for kind "e4m3" / "int8", `bounds`
    (blocks, heads, 2, dim) or None.  All three are updated in place."""
    blocks, size, heads, _ = cache.shape
    pages = {}
    for t, slot in enumerate(slots):
        if 0 <= slot < blocks * size:
            pages.setdefault(int(slot) // size, []).append((t, int(slot) % size))
    for page, tokens in pages.items():
        lowest = min(at for _, at in tokens)
        for h in range(heads):
            new = np.stack([rows[t, h] for t, _ in tokens])
            if bounds is not None:
                keep = np.where(np.isnan(new), np.inf, new).min(0), np.where(np.isnan(new), -np.inf, new).max(0)
                had = bounds[page, h] if lowest > 0 else (np.inf, -np.inf)
                bounds[page, h, 0] = np.minimum(keep[0], had[0])
                bounds[page, h, 1] = np.maximum(keep[1], had[1])
            if kind not in TOP:
                for t, at in tokens:
                    cache[page, at, h] = rows[t, h]
                continue
            finite = np.abs(new[np.isfinite(new)])
            after = scale_for(finite.max() if finite.size else 0.0, kind)
            if lowest > 0:
                before = scale[page, h]
                after = max(after, before)
                if after > before:
                    cache[page, :lowest, h] = to_code(cache[page, :lowest, h] * (before / after), kind)
            scale[page, h] = after
            for t, at in tokens:
                cache[page, at, h] = to_code(rows[t, h] / after, kind)


def select(query, bounds, block_table, context_lens, count, block_size, keep_first, keep_last):
    """query (batch, heads, rows, dim) -> (batch, kv_heads, count) int."""
    batch, heads = query.shape[:2]
    kv_heads = bounds.shape[1]
    group = heads // kv_heads
    out = np.full((batch, kv_heads, count), -1)
    for b in range(batch):
        n = min(-(-max(int(context_lens[b]), 0) // block_size), block_table.shape[1])
        for h in range(kv_heads):
            q = query[b, h * group:(h + 1) * group].reshape(-1, query.shape[-1])
            ranked = []
            for j in range(n):
                page = int(block_table[b, j])
                score = -math.inf
                if 0 <= page < bounds.shape[0]:
                    lo, hi = bounds[page, h]
                    with np.errstate(invalid="ignore"):
                        s = (np.maximum(q, 0) * hi).sum(-1) + (np.minimum(q, 0) * lo).sum(-1)
                    score = np.where(np.isnan(s), math.inf, s).max()
                always = j < keep_first or j >= n - keep_last
                ranked.append((not always, -score, j))
            chosen = sorted(j for _, _, j in sorted(ranked)[:count])
            out[b, h, :len(chosen)] = chosen
    return out


def attend(query, k_cache, v_cache, block_table, context_lens, k_scale=None, v_scale=None, block_index=None,
           causal=False, scale=None):
    """query (batch, heads, rows, dim); caches (blocks, block_size, kv_heads, dim)."""
    batch, heads, rows, dim = query.shape
    blocks, size, kv_heads, _ = k_cache.shape
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    out = np.zeros(query.shape)
    for b in range(batch):
        length = min(max(int(context_lens[b]), 0), block_table.shape[1] * size)
        for h in range(kv_heads):
            order = range(block_table.shape[1]) if block_index is None else [int(j) for j in block_index[b, h]]
            keys, values, at = [], [], []
            for j in order:
                if not 0 <= j * size < length:
                    continue
                page = int(block_table[b, j])
                if not 0 <= page < blocks:
                    continue
                here = min(size, length - j * size)
                keys.append(k_cache[page, :here, h] * (1.0 if k_scale is None else k_scale[page, h]))
                values.append(v_cache[page, :here, h] * (1.0 if v_scale is None else v_scale[page, h]))
                at.append(np.arange(j * size, j * size + here))
            if not keys:
                continue
            keys, values, at = np.concatenate(keys), np.concatenate(values), np.concatenate(at)
            for g in range(h * heads // kv_heads, (h + 1) * heads // kv_heads):
                for i in range(rows):
                    seen = at <= length - rows + i if causal else np.ones(len(at), dtype=bool)
                    if not seen.any():
                        continue
                    logits = keys[seen] @ query[b, g, i] * scale
                    w = np.exp(logits - logits.max())
                    out[b, g, i] = w @ values[seen] / w.sum()
    return out
