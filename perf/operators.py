"""What a user of this package has a paged key / value cache do, as timed cases over its public entry points.

A case is a dict of plain values; `op` says which operator it goes through:

* ``allocate``  paged_kvcache_allocate: block tables and slot maps from request lengths
* ``append``    paged_kvcache_append: new rows into a 16-bit, e4m3 or int8 cache, with scales and key bounds
* ``select``    paged_kvcache_select: the blocks whose key bounds promise the highest logits
* ``attend``    flash_attention_decode_paged / _paged_multi over 8-bit caches with a scale for each block and head,
                over all blocks or over selected ones

`listed` holds the fixed cases and `draw` further ones of the same ranges. `run` computes a case in its plain form,
or through the package where `own` is true.
"""

import functools
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_PACKAGE = os.path.abspath("flash-attention-rdna3_amd")
_DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16}
_CACHE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_TOP = {"e4m3": 448.0, "int8": 127.0}  # largest stored magnitude
_LEAST = -100                          # smallest exponent of a scale


@functools.lru_cache(maxsize=None)
def _fa():
    if _PACKAGE not in sys.path:
        sys.path.insert(1, _PACKAGE)
    import fa_rdna3

    return fa_rdna3


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _allocate(batch, context, new, block):
    return {"op": "allocate", "batch": batch, "context": context, "new": new, "block": block}


def _append(dtype, cache, batch, kv_heads, dim, block, context, new, bounds):
    return {"op": "append", "dtype": dtype, "cache": cache, "batch": batch, "kv_heads": kv_heads, "dim": dim,
            "block": block, "context": context, "new": new, "bounds": bounds}


def _select(dtype, batch, heads, kv_heads, dim, block, context, chosen, first=1, last=1):
    return {"op": "select", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "block": block, "context": context, "chosen": chosen, "first": first, "last": last}


def _attend(dtype, cache, batch, heads, kv_heads, rows, dim, block, context, chosen=0, ragged=True):
    return {"op": "attend", "dtype": dtype, "cache": cache, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "rows": rows, "dim": dim, "block": block, "context": context, "chosen": chosen, "ragged": ragged}


def listed():
    return [
        # A decode step of 64 requests: one token each, a block now and then.
        dict(_allocate(64, 8192, 1, 16), name="tables_step"),
        # 300 prompts scheduled at once, nothing of them cached yet.
        dict(_allocate(300, 0, 2048, 64), name="tables_prompts"),
        # The step's 64 new rows into an e4m3 cache, most into blocks that are partly filled.
        dict(_append("bf16", "e4m3", 64, 8, 128, 64, 2048, 1, True), name="append_step_e4m3"),
        # 16 prompts of up to 2048 tokens into an int8 cache.
        dict(_append("fp16", "int8", 16, 8, 128, 64, 0, 2048, False), name="append_prompts_int8"),
        # Chunks of prompts into a 16-bit cache that keeps key bounds; few narrow heads, small pages.
        dict(_append("bf16", "bf16", 7, 4, 64, 16, 1000, 333, True), name="append_chunk_bf16"),
        # Four requests of 16384 tokens in pages of 16: 64 pages of 1024 (the paged workload's shapes).
        dict(_select("fp16", 4, 32, 8, 128, 16, 16384, 64), name="select_step"),
        # 32 requests of up to 131072 tokens: 64 blocks of 64 tokens each.
        dict(_select("bf16", 32, 32, 8, 128, 64, 131072, 64, 1, 2), name="select_long"),
        # Three short requests, five query heads for each of four kv heads of 64: latency.
        dict(_attend("fp16", "e4m3", 3, 20, 4, 1, 64, 32, 777), name="attend_small"),
        # The paged workload's shapes over an e4m3 cache in pages of 16.
        dict(_attend("fp16", "e4m3", 4, 32, 8, 1, 128, 16, 16384, ragged=False), name="attend_e4m3"),
        # Long contexts of very different lengths over an int8 cache.
        dict(_attend("bf16", "int8", 4, 32, 8, 1, 128, 64, 131072), name="attend_long_int8"),
        # 64 selected blocks of long contexts, another choice for every kv head.
        dict(_attend("bf16", "e4m3", 16, 32, 8, 1, 128, 64, 65536, 64), name="attend_selected"),
        # A chunk of 512 prompt rows over what is already cached.
        dict(_attend("bf16", "int8", 2, 32, 8, 512, 128, 64, 8192), name="attend_chunk_int8"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: sizes spread over the listed ones' ranges, odd ones among them."""
    op = rng.choice(("allocate", "append", "select", "attend", "attend"))
    dtype, block = rng.choice(("fp16", "bf16")), rng.choice((8, 16, 16, 32, 64, 64, 128, 256))
    if op == "allocate":
        new = rng.choice((1, 1, _log(rng, 2, 2048)))
        return _allocate(_log(rng, 1, 300), rng.choice((0, _log(rng, 1, 16384))), new, block)
    kv_heads, dim = rng.choice((1, 2, 4, 8, 8)), rng.choice((32, 64, 128, 128, 128, 256))
    heads = kv_heads * rng.choice((1, 2, 4, 4, 5, 8))
    cache = rng.choice(("e4m3", "int8", "e4m3", "int8", dtype))
    if op == "append":
        context, new = rng.choice((0, _log(rng, 1, 2048))), rng.choice((1, _log(rng, 2, 2048)))
        most = max(1, min(64, (1 << 18) // (context + new), (1 << 25) // (new * kv_heads * dim)))
        return _append(dtype, cache, _log(rng, 1, most), kv_heads, dim, block, context, new, rng.random() < 0.5)
    if op == "select":
        context = _log(rng, 1, 131072)
        blocks = -(-context // block)
        most = max(1, min(32, (1 << 26) // (blocks * kv_heads * dim)))
        chosen = _log(rng, 3, 128)
        return _select(dtype, _log(rng, 1, most), heads, kv_heads, dim, block, context, chosen, rng.choice((0, 1)),
                       rng.choice((1, 2)))
    rows = rng.choice((1, 1, 1, _log(rng, 2, 8), _log(rng, 9, 512)))
    context = _log(rng, rows, 8192 if rows > 8 else 131072)
    chosen = _log(rng, 1, 128) if cache == dtype or (rows <= 8 and rng.random() < 0.4) else 0
    most = (1 << 28) // (context * kv_heads * dim)
    if rows > 8:
        most = min(most, (1 << 35) // (context * heads * dim * rows))
    return _attend(dtype, cache, _log(rng, 1, max(1, min(32, most))), heads, kv_heads, rows, dim, block, context,
                   chosen, rng.random() < 0.8)


def _lengths(count, longest, ragged=True, least=0):
    """`count` lengths up to `longest`, that one among them: the same for every seed, so that the work is known."""
    if not ragged:
        return [longest] * count
    rng = random.Random(count * 1000003 + longest)
    return [longest] + [rng.randint(min(least, longest), longest) for _ in range(count - 1)]


def _sizes(case):
    """(context lengths, new tokens or rows, blocks a request may have) of a case."""
    op, block = case["op"], case["block"]
    if op in ("allocate", "append"):
        contexts = _lengths(case["batch"], case["context"])
        news = [1] * case["batch"] if case["new"] == 1 else _lengths(case["batch"], case["new"])
        return contexts, news, max(1, -(-(case["context"] + case["new"]) // block))
    least = case.get("rows", 1)
    return _lengths(case["batch"], case["context"], case.get("ragged", True), least), None, -(-case["context"] // block)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _table(g, batch, blocks, spare=3):
    """A block table over a shuffled pool, and the pool's size."""
    pool = batch * blocks + spare
    ids = torch.randperm(pool, generator=g, device="cuda")[:batch * blocks]
    return ids.view(batch, blocks).to(torch.int32), pool


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _codes(g, shape, cache, dtype):
    """Cache contents: values of the 16-bit type, or codes that fill the 8-bit type's range."""
    if cache == "int8":
        return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)
    x = torch.empty(shape, dtype=_CACHE.get(cache, dtype), device="cuda")
    flat, step = x.view(-1), 1 << 26
    for at in range(0, flat.numel(), step):  # (a whole large cache in 32 bits would not fit three times)
        part = _randn(g, (min(step, flat.numel() - at),))
        flat[at:at + step] = (part * 100.0).clamp(-448.0, 448.0).to(x.dtype) if cache == "e4m3" else part.to(x.dtype)
    return x


def _scales(g, pool, kv_heads, cache):
    """Scales that bring the codes to about unit spread, each block and head with its own."""
    spread = {"e4m3": 100.0, "int8": 73.0}[cache]
    return torch.exp(0.5 * _randn(g, (pool, kv_heads))) / spread


def prepare(case, seed):
    g, op, block = _generator(seed), case["op"], case["block"]
    contexts, news, blocks = _sizes(case)
    batch = case["batch"]
    s = {"case": case, "context_lens": _int32(contexts)}
    if op == "allocate":
        table, pool = _table(g, batch, blocks)
        have = torch.tensor([-(-c // block) for c in contexts], device="cuda")
        mine = torch.arange(blocks, device="cuda") < have[:, None]
        free = torch.ones(pool, dtype=torch.bool, device="cuda")
        free[table[mine].long()] = False
        ids = free.nonzero().view(-1).to(torch.int32)
        s |= {"table": torch.where(mine, table, -1).to(torch.int32), "new_lens": _int32(news),
              "free": ids[torch.randperm(ids.numel(), generator=g, device="cuda")].contiguous(),
              "head": torch.zeros(1, dtype=torch.int32, device="cuda"), "tokens": sum(news)}
        return s
    kv_heads, dim, dtype = case["kv_heads"], case["dim"], _DTYPE[case["dtype"]]
    table, pool = _table(g, batch, blocks)
    if op == "append":
        cache = case["cache"]
        tokens = sum(news)
        owner = torch.repeat_interleave(torch.arange(batch, device="cuda"), torch.tensor(news, device="cuda"))
        at = torch.cat([torch.arange(c, c + n) for c, n in zip(contexts, news)]).cuda()
        s["slots"] = table[owner, at // block].long() * block + at % block
        for name in ("key", "value"):
            loud = torch.exp2(torch.randint(-2, 3, (tokens, kv_heads, 1), generator=g, device="cuda").float())
            s[name] = (_randn(g, (tokens, kv_heads, dim)) * loud).to(dtype)
        for name in ("k", "v"):
            s[name + "_cache"] = _codes(g, (pool, block, kv_heads, dim), cache, dtype)
            if cache in _CACHE:
                exponents = torch.randint(-8, -5, (pool, kv_heads), generator=g, device="cuda")
                s[name + "_scale"] = torch.exp2(exponents.float())
        if case["bounds"]:
            ends = _randn(g, (2, pool, kv_heads, dim), dtype)
            s["bounds"] = torch.stack([torch.minimum(ends[0], ends[1]), torch.maximum(ends[0], ends[1])], 2)
        return s
    s["table"] = table
    if op == "select":
        s["query"] = _randn(g, (batch, case["heads"], dim), dtype)
        middle, half = _randn(g, (pool, kv_heads, dim)) * 0.5, _randn(g, (pool, kv_heads, dim)).abs() + 0.5
        s["bounds"] = torch.stack([middle - half, middle + half], 2).to(dtype)
        return s
    s["query"] = _randn(g, (batch, case["heads"], case["rows"], dim), dtype) * 1.5
    for name in ("k", "v"):
        s[name + "_cache"] = _codes(g, (pool, block, kv_heads, dim), case["cache"], dtype)
        if case["cache"] in _CACHE:
            s[name + "_scale"] = _scales(g, pool, kv_heads, case["cache"])
    if case["chosen"]:
        # Distinct blocks of each request, ascending; -1 behind them where it has fewer.
        order = torch.rand((batch, kv_heads, blocks), generator=g, device="cuda")
        have = torch.tensor([-(-c // block) for c in contexts], device="cuda").view(-1, 1, 1)
        order = torch.where(torch.arange(blocks, device="cuda") < have, order, 2.0)
        take = min(case["chosen"], blocks)
        order, index = order.sort(-1)
        index = torch.where(order[..., :take] < 2.0, index[..., :take], blocks).sort(-1).values
        index = torch.where(index < blocks, index, -1)
        s["index"] = torch.nn.functional.pad(index, (0, case["chosen"] - take), value=-1).to(torch.int32)
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _plain_allocate(s):
    block, table, free = s["case"]["block"], s["table"], s["free"].long()
    ctx, new = s["context_lens"].long().clamp(min=0), s["new_lens"].long().clamp(min=0)
    batch, blocks = table.shape
    cap = blocks * block
    first = (ctx.clamp(max=cap) + block - 1) // block
    need = ((ctx + new).clamp(max=cap) + block - 1) // block - first
    start = s["head"].long() + need.cumsum(0) - need
    column = torch.arange(blocks, device="cuda")
    at = start[:, None] + column - first[:, None]
    fresh = (column >= first[:, None]) & (column < (first + need)[:, None])
    ids = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where(fresh, ids.to(torch.int32), table))
    ends = new.cumsum(0)
    token = torch.arange(s["tokens"], device="cuda")
    owner = torch.searchsorted(ends, token, right=True).clamp(max=batch - 1)
    at = ctx[owner] + token - (ends - new)[owner]
    page = table[owner, (at // block).clamp(max=blocks - 1)].long()
    ok = (token < ends[-1]) & (at < cap) & (page >= 0)
    slots = torch.where(ok, page * block + at % block, -1)
    cu = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    return slots, cu, table, (s["head"] + need.sum()).to(torch.int32)


def _round_codes(x, cache):
    x = x.clamp(-_TOP[cache], _TOP[cache])
    if cache == "int8":
        return torch.nan_to_num(x.round()).to(torch.int8)
    return x.to(torch.float8_e4m3fn)


def _scale_for(amax, cache):
    """The least power of two 2^e, e >= _LEAST, with amax <= top * 2^e."""
    mantissa, exponent = torch.frexp(amax)
    top_mantissa, top_exponent = math.frexp(_TOP[cache])
    e = exponent - top_exponent + (mantissa > top_mantissa)
    return torch.exp2(torch.where(amax > 0, e, _LEAST).clamp(min=_LEAST).float())


def _plain_append(s):
    case, slots = s["case"], s["slots"]
    cache, block, kv_heads = case["cache"], case["block"], case["kv_heads"]
    pool = s["k_cache"].shape[0]
    page, at = slots // block, slots % block
    lowest = torch.full((pool,), block, device="cuda").scatter_reduce(0, page, at, "amin")
    touched = (lowest < block).nonzero().view(-1)
    earlier = lowest[touched]  # rows of each touched block that were there before
    outs = []
    for name, tensor in (("k", s["key"]), ("v", s["value"])):
        rows, kept = tensor.float(), s[name + "_cache"]
        if cache in _CACHE:
            scale = s[name + "_scale"]
            amax = torch.where(rows.isfinite(), rows.abs(), 0.0).amax(-1)
            top = torch.zeros((pool, kv_heads), device="cuda").index_reduce(0, page, amax, "amax")[touched]
            before = torch.where(earlier[:, None] > 0, scale[touched], 0.0)
            after = torch.maximum(before, _scale_for(top, cache))
            old = kept[touched].float() * (before / after)[:, None, :, None]
            again = (torch.arange(block, device="cuda") < earlier[:, None])[:, :, None, None] & (after > before)[:, None, :, None]
            as_bytes = lambda t: t.view(torch.uint8)  # noqa: E731  (selected as bytes: 8-bit floats have no where)
            as_bytes(kept)[touched] = torch.where(again, as_bytes(_round_codes(old, cache)), as_bytes(kept[touched]))
            scale[touched] = after
            as_bytes(kept)[page, at] = as_bytes(_round_codes(rows * (1.0 / scale)[page][:, :, None], cache))
            outs += [kept, scale]
        else:
            kept[page, at] = tensor
            outs.append(kept)
    if case["bounds"]:
        rows, bounds, inf = s["key"].float(), s["bounds"], math.inf
        nan, fresh = rows.isnan(), (earlier == 0)[:, None, None]
        shape = (pool,) + tuple(rows.shape[1:])
        low = torch.full(shape, inf, device="cuda").index_reduce(0, page, torch.where(nan, inf, rows), "amin")[touched]
        high = torch.full(shape, -inf, device="cuda").index_reduce(0, page, torch.where(nan, -inf, rows), "amax")[touched]
        had = bounds[touched].float()
        low = torch.minimum(low, torch.where(fresh, inf, had[:, :, 0]))
        high = torch.maximum(high, torch.where(fresh, -inf, had[:, :, 1]))
        bounds[touched] = torch.stack([low, high], 2).to(bounds.dtype)
        outs.append(bounds)
    return outs


def _plain_select(s):
    case, table, bounds = s["case"], s["table"], s["bounds"]
    kv_heads, block, chosen = case["kv_heads"], case["block"], case["chosen"]
    batch, blocks = table.shape
    # In 64 bits: the order of a sum decides no block at the border.
    q = s["query"].double().view(batch, kv_heads, -1, case["dim"])
    low, high = (bounds[:, :, i][table.long()].permute(0, 2, 3, 1).double() for i in (0, 1))
    score = (torch.matmul(q.clamp(min=0), high) + torch.matmul(q.clamp(max=0), low))
    score = torch.where(score.isnan(), math.inf, score).amax(2)
    column = torch.arange(blocks, device="cuda")
    have = ((s["context_lens"].long() + block - 1) // block)[:, None, None]
    always = (column < case["first"]) | (column >= have - case["last"])
    rank = torch.where(column < have, 1 + always.long(), 0).expand(batch, kv_heads, blocks)
    order = score.sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, rank.gather(-1, order).sort(dim=-1, descending=True, stable=True).indices)
    index = order[..., :chosen]
    index = torch.where(index < have, index, blocks).sort(-1).values
    index = torch.where(index < blocks, index, -1)
    return torch.nn.functional.pad(index, (0, chosen - index.shape[-1]), value=-1).to(torch.int32)


def _plain_attend(s):
    case, table, q = s["case"], s["table"], s["query"]
    batch, heads, rows, dim = q.shape
    kv_heads, block = case["kv_heads"], case["block"]
    blocks = table.shape[1]
    if "index" in s:
        index = s["index"].long()
    else:
        index = torch.arange(blocks, device="cuda").expand(batch, 1, blocks)
    listed_here = index >= 0
    page = table[torch.arange(batch, device="cuda").view(-1, 1, 1), index.clamp(min=0)].long()
    at = index[..., None] * block + torch.arange(block, device="cuda")
    lens = s["context_lens"].long().view(-1, 1, 1, 1)
    there = (listed_here[..., None] & (at < lens)).flatten(2)
    at = at.flatten(2)

    def gather(name):  # (batch, kv_heads, keys, dim) in 32 bits, scaled
        kept = s[name + "_cache"]
        if index.shape[1] == 1:
            x = kept.view(torch.uint8)[page[:, 0]].view(kept.dtype).float()  # (batch, n, block, kv_heads, dim)
            if name + "_scale" in s:
                x *= s[name + "_scale"][page[:, 0]][:, :, None, :, None]
            return x.permute(0, 3, 1, 2, 4).reshape(batch, kv_heads, -1, dim)
        head = torch.arange(kv_heads, device="cuda").view(1, -1, 1)
        x = kept.view(torch.uint8).permute(0, 2, 1, 3)[page, head].view(kept.dtype).float()
        if name + "_scale" in s:
            x *= s[name + "_scale"][page, head][..., None, None]
        return x.flatten(2, 3)

    grouped = q.float().reshape(batch, kv_heads, -1, dim)  # rows of a group: (head of the group, row)
    logits = torch.matmul(grouped, gather("k").transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    row = torch.arange(rows, device="cuda").repeat(heads // kv_heads)
    seen = there[:, :, None] & (at[:, :, None] <= lens - rows + row.view(1, 1, -1, 1))
    logits = torch.where(seen, logits, -math.inf)
    top = logits.amax(-1, keepdim=True)
    weights = torch.exp(logits - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, gather("v")) / torch.where(total == 0, 1.0, total)
    return out.view(batch, heads, rows, dim).to(q.dtype)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if op == "allocate":
        if own:
            slots, cu, head = _fa().paged_kvcache_allocate(
                s["table"], s["context_lens"], s["new_lens"], s["free"], free_head=s["head"], block_size=case["block"],
                num_tokens=s["tokens"])
            return slots, cu, s["table"], head
        return _plain_allocate(s)
    if op == "append":
        if own:
            _fa().paged_kvcache_append(s["key"], s["value"], s["k_cache"], s["v_cache"], s["slots"],
                                       k_scale=s.get("k_scale"), v_scale=s.get("v_scale"), key_bounds=s.get("bounds"))
            names = ("k_cache", "k_scale", "v_cache", "v_scale", "bounds")
            return [s[name] for name in names if name in s]
        return _plain_append(s)
    if op == "select":
        if own:
            return _fa().paged_kvcache_select(s["query"], s["bounds"], s["table"], s["context_lens"], case["chosen"],
                                              block_size=case["block"], keep_first=case["first"], keep_last=case["last"])
        return _plain_select(s)
    if not own:
        return _plain_attend(s)
    more = {"k_scale": s.get("k_scale"), "v_scale": s.get("v_scale"), "block_index": s.get("index")}
    if case["rows"] == 1:
        return _fa().flash_attention_decode_paged(s["query"][:, :, 0], s["k_cache"], s["v_cache"], s["table"],
                                                  s["context_lens"], **more)[:, :, None]
    return _fa().flash_attention_decode_paged_multi(s["query"], s["k_cache"], s["v_cache"], s["table"],
                                                    s["context_lens"], causal=True, **more)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    op, block, batch = case["op"], case["block"], case["batch"]
    contexts, news, blocks = _sizes(case)
    if op == "allocate":
        fresh = sum(-(-(c + n) // block) + -c // block for c, n in zip(contexts, news))
        return {"bytes": 8 * sum(news) + 8 * fresh + 16 * batch, "flops": 0}
    kv_heads, dim = case["kv_heads"], case["dim"]
    width = 1 if case.get("cache") in _CACHE else 2
    if op == "append":
        tokens = sum(news)
        fresh = sum(-(-(c + n) // block) - c // block for c, n in zip(contexts, news))
        extra = (16 if width == 1 else 0) + (4 * dim if case["bounds"] else 0)
        return {"bytes": tokens * (kv_heads * dim * 2 * (2 + width) + 8) + fresh * kv_heads * extra, "flops": 0}
    if op == "select":
        count = sum(-(-c // block) for c in contexts)
        return {"bytes": count * (kv_heads * 4 * dim + 4) + batch * (case["heads"] * dim * 2 + kv_heads * case["chosen"] * 4),
                "flops": 2 * count * case["heads"] * dim}
    keys = 0
    for c in contexts:
        whole = -(-c // block)
        share = min(case["chosen"], whole) / max(1, whole) if case["chosen"] else 1.0
        keys += c * share
    rows, heads = case["rows"], case["heads"]
    per_key = kv_heads * 2 * dim * width + (kv_heads * 8 / block if width == 1 else 0)
    return {"bytes": keys * per_key + 4 * batch * heads * rows * dim, "flops": 4 * keys * heads * rows * dim}


# ---------------------------------------------------------------------------
# In 64 bits, from the definitions
# ---------------------------------------------------------------------------

def exact(case, seed):
    op = case["op"]
    if op in ("allocate", "select"):
        return None  # whole numbers
    if op == "append":
        return _exact_append(case, prepare(case, seed))
    return _exact_attend(case, prepare(case, seed))


def _nearest(x, cache):
    """float64 values to the nearest value of the 8-bit type, ties to even."""
    x = np.clip(x, -_TOP[cache], _TOP[cache])
    if cache == "int8":
        return np.rint(x)
    exponent = np.maximum(np.frexp(x)[1] - 1, -6)
    step = np.exp2(exponent - 3.0)
    return np.rint(x / step) * step


def _exact_append(case, s):
    cache, block = case["cache"], case["block"]
    if s["k_cache"].numel() > 1 << 28:
        return None
    slots, host = s["slots"].cpu().numpy(), lambda t: t.float().cpu().numpy().astype(np.float64)  # noqa: E731
    groups = {}
    for token, slot in enumerate(slots.tolist()):
        groups.setdefault(slot // block, []).append(token)
    kept = {name: host(s[name]) for name in ("k_cache", "k_scale", "v_cache", "v_scale", "bounds") if name in s}
    rows = {"k": host(s["key"]), "v": host(s["value"])}
    for page, tokens in groups.items():
        at = slots[tokens] % block
        for name in ("k", "v"):
            new, store = rows[name][tokens], kept[name + "_cache"]
            if cache not in _CACHE:
                store[page, at] = new
                continue
            top = np.abs(new).max(axis=(0, 2))
            with np.errstate(divide="ignore"):
                need = np.maximum(np.ceil(np.log2(top / _TOP[cache])), _LEAST)
            now, scale = np.exp2(need), kept[name + "_scale"]
            if at.min() > 0:
                now = np.maximum(now, scale[page])
                grown, before = now > scale[page], at.min()
                again = _nearest(store[page, :before] * (scale[page] / now)[None, :, None], cache)
                store[page, :before] = np.where(grown[None, :, None], again, store[page, :before])
            scale[page] = now
            store[page, at] = _nearest(new / now[None, :, None], cache)
        if "bounds" in kept:
            low, high = rows["k"][tokens].min(0), rows["k"][tokens].max(0)
            if at.min() > 0:
                low, high = np.minimum(low, kept["bounds"][page, :, 0]), np.maximum(high, kept["bounds"][page, :, 1])
            kept["bounds"][page, :, 0], kept["bounds"][page, :, 1] = low, high
    whole = cache == "int8"
    return [None if whole and name.endswith("_cache") else torch.from_numpy(kept[name])
            for name in ("k_cache", "k_scale", "v_cache", "v_scale", "bounds") if name in kept]


def _exact_attend(case, s):
    q = s["query"].double()
    batch, heads, rows, dim = q.shape
    kv_heads, block = case["kv_heads"], case["block"]
    out = torch.zeros_like(q)
    for b, length in enumerate(s["context_lens"].tolist()):
        for h in range(kv_heads):
            if "index" in s:
                order = s["index"][b, h]
                order = order[order >= 0].long()
            else:
                order = torch.arange(-(-length // block), device="cuda")
            pages = s["table"][b, order].long()
            at = (order[:, None] * block + torch.arange(block, device="cuda")).reshape(-1)
            keys, values = (s[name + "_cache"][:, :, h].view(torch.uint8)[pages].view(s[name + "_cache"].dtype).double()
                            for name in ("k", "v"))
            if "k_scale" in s:
                keys = keys * s["k_scale"][pages, h].double()[:, None, None]
                values = values * s["v_scale"][pages, h].double()[:, None, None]
            keep = at < length
            keys, values, at = keys.reshape(-1, dim)[keep], values.reshape(-1, dim)[keep], at[keep]
            for head in range(h * heads // kv_heads, (h + 1) * heads // kv_heads):
                logits = q[b, head] @ keys.T / math.sqrt(dim)
                late = at[None, :] > length - rows + torch.arange(rows, device="cuda")[:, None]
                logits = logits.masked_fill(late, -math.inf)
                empty = late.all(1)
                out[b, head] = torch.softmax(logits.masked_fill(empty[:, None], 0.0), -1) @ values
                out[b, head][empty] = 0.0
    return out
