"""Paged decode over 8-bit caches with block scales and over listed blocks,
against the 64-bit oracle on the same codes.

The bound of a value, from the roundings between the two: A is the same
attention over |v|; p v is summed with p rounded to the products' type (fp16
over 8-bit caches: 2^-11 of p, and 2^-25 of the scales' range where it is
subnormal; else the query's type), the logits are sums of D fp32 products, the
output sums of n fp32 products, and the result is rounded once to its type.
"""

import numpy as np
import pytest
import torch

from fa_rdna3 import (
    _native,
    flash_attention_decode_paged,
    flash_attention_decode_paged_multi,
    paged_kvcache_allocate,
    paged_kvcache_append,
    paged_kvcache_select,
)
from oracle import paged_cache as oracle
from paged_cases import CACHES, codes, f64, int32, scales, table_of

pytestmark = pytest.mark.gpu
DEVICE = "cuda"
ROUNDING = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _case(seed, kind, dtype, batch, heads, kv_heads, rows, dim, block, lens, n_index=0, spare=3):
    g = torch.Generator().manual_seed(seed)
    blocks = max(1, -(-max(lens) // block))
    table, pool = table_of(g, batch, blocks, spare)
    c = dict(q=(torch.randn(batch, heads, rows, dim, generator=g) * 1.5).to(dtype),
             k=codes(g, (pool, block, kv_heads, dim), kind, dtype), v=codes(g, (pool, block, kv_heads, dim), kind, dtype),
             table=table, lens=int32(lens), ks=None, vs=None, index=None, kind=kind)
    if kind in CACHES:
        c["ks"], c["vs"] = scales(g, pool, kv_heads, kind), scales(g, pool, kv_heads, kind)
    if n_index:
        c["index"] = torch.stack([torch.stack([
            torch.cat([torch.randperm(blocks, generator=g)[:n_index].sort().values,
                       torch.full((max(0, n_index - blocks),), -1)]) for _ in range(kv_heads)])
            for _ in range(batch)]).to(torch.int32)
    return c


def _run(c, causal, **more):
    dev = {k: v.to(DEVICE) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    args = dev["k"], dev["v"], dev["table"], dev["lens"]
    kw = dict(k_scale=dev["ks"], v_scale=dev["vs"], block_index=dev["index"], **more)
    if c["q"].shape[2] == 1:
        return flash_attention_decode_paged(dev["q"][:, :, 0], *args, **kw)[:, :, None]
    return flash_attention_decode_paged_multi(dev["q"], *args, causal=causal, **kw)


def _bound(c, want, causal):
    q, k, v = f64(c["q"]), f64(c["k"]), np.abs(f64(c["v"]))
    dim, n = q.shape[-1], c["table"].shape[1] * k.shape[1]
    f = lambda name: None if c[name] is None else f64(c[name])  # noqa: E731
    ks, vs, index = f("ks"), f("vs"), None if c["index"] is None else c["index"].numpy()
    n = max(n, 0 if index is None else index.shape[2] * k.shape[1])
    near = oracle.attend(q, k, v, c["table"].numpy(), c["lens"].tolist(), ks, vs, index, causal)
    key = (np.abs(k).max() if ks is None else (np.abs(k).max((1, 3)) * np.abs(ks)).max())
    logit = (dim + 8) * 2.0 ** -24 * np.abs(q).sum(-1, keepdims=True) * key / np.sqrt(dim)
    out = ROUNDING[c["q"].dtype]
    p = 2.0 ** -11 if c["kind"] in CACHES else out
    tiny = n * 2.0 ** -25 * 2 * (vs.max() * v.max() if vs is not None else v.max())
    return near * (p + (n + 16) * 2.0 ** -23 + 2 * logit) * (1 + out) + tiny + out * np.abs(want) + 1e-30


def _check(c, causal=True, **more):
    got = f64(_run(c, causal, **more))
    f = lambda name: None if c[name] is None else f64(c[name])  # noqa: E731
    want = oracle.attend(f64(c["q"]), f64(c["k"]), f64(c["v"]), c["table"].numpy(), c["lens"].tolist(), f("ks"), f("vs"),
                         None if c["index"] is None else c["index"].numpy(), causal)
    bound = _bound(c, want, causal)
    # Results whose bound reaches 65520 may round to fp16's infinity (its largest value is 65504, the next step 65536).
    over = (c["q"].dtype == torch.float16) & (np.abs(want) + bound >= 65520) & np.isinf(got) & (np.sign(got) == np.sign(want))
    off = np.where(over, 0.0, np.abs(np.where(over, 0.0, got) - want) - bound)
    assert (off <= 0).all(), (off.max(), np.argwhere(off > 0)[:5])
    return got


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,rows,dim,block,lens", [
    (4, 4, 1, 32, 16, [1, 31, 32, 33]), (8, 2, 1, 64, 16, [700, 1, 0, 65]), (32, 8, 1, 128, 64, [1000, 64, 63]),
    (20, 4, 1, 128, 32, [777, 5]), (8, 1, 1, 256, 128, [300, 129]), (3, 1, 1, 512, 16, [100, 17, 1]),
    (8, 2, 5, 128, 16, [333, 5, 4, 70]), (8, 2, 8, 64, 32, [500, 9]), (4, 1, 40, 128, 64, [200, 40, 41]),
    (16, 2, 17, 32, 256, [400, 20]), (2, 1, 100, 64, 16, [150, 100]), (4, 2, 3, 256, 16, [90, 3])])
def test_block_scales(kind, dtype, heads, kv_heads, rows, dim, block, lens):
    _check(_case(dim + block, kind, dtype, len(lens), heads, kv_heads, rows, dim, block, lens))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("block", [1, 2, 4, 8])
@pytest.mark.parametrize("heads,kv_heads,rows,dim", [(8, 2, 1, 128), (4, 2, 3, 64), (2, 1, 20, 32), (2, 2, 1, 256)])
def test_small_pages(kind, block, heads, kv_heads, rows, dim):
    _check(_case(block + dim, kind, torch.float16, 3, heads, kv_heads, rows, dim, block, [150, 33, rows]))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,rows,dim,block,lens,n_index", [
    (8, 2, 33, 128, 16, [300, 33, 64], 0), (4, 1, 64, 128, 32, [500, 64, 65, 700], 0), (2, 2, 129, 64, 64, [129, 200], 0),
    (5, 1, 50, 64, 128, [1000, 51], 0), (4, 2, 70, 128, 256, [300, 257], 0), (4, 1, 100, 64, 16, [1500, 100], 11),
    (8, 1, 16, 128, 64, [3000, 16, 17, 900], 5)])
def test_many_rows(kind, dtype, heads, kv_heads, rows, dim, block, lens, n_index):
    c = _case(dim + rows, kind, dtype, len(lens), heads, kv_heads, rows, dim, block, lens, n_index)
    _check(c)
    _check(c, causal=False, num_splits=3)
    c["table"][0, 1] = -1
    c["table"][-1, 0] = 10 ** 9
    c["q"] = c["q"] * 8
    _check(c)


def test_many_rows_keep_low_logits():
    # every logit far below zero: the first maximum is not 0
    c = _case(30, "int8", torch.float16, 2, 4, 1, 40, 64, 16, [400, 60])
    c["q"], c["k"] = -c["q"].abs() * 30, c["k"].clamp(min=1)
    _check(c)
    c["ks"] *= -1  # and far above
    _check(c)


def test_small_pages_wide_heads():
    _check(_case(1, "e4m3", torch.bfloat16, 2, 4, 2, 2, 512, 8, [70, 9]))


@pytest.mark.parametrize("kind", ["e4m3", "int8", "same"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,rows,dim,block,lens,n_index", [
    (8, 2, 1, 128, 16, [700, 300, 17, 0], 7), (4, 2, 1, 64, 64, [1000, 64], 20), (4, 1, 3, 32, 4, [100, 9], 11),
    (8, 4, 2, 256, 32, [400, 50], 5), (2, 1, 1, 512, 16, [333], 9), (4, 2, 1, 512, 2, [100], 20),
    (8, 2, 9, 128, 16, [333, 20], 12), (2, 2, 1, 128, 128, [1000], 1)])
def test_listed_blocks(kind, dtype, heads, kv_heads, rows, dim, block, lens, n_index):
    _check(_case(dim + n_index, kind, dtype, len(lens), heads, kv_heads, rows, dim, block, lens, n_index))


def test_listed_blocks_of_a_cache_with_one_scale():
    c = _case(2, "e4m3", torch.float16, 2, 8, 2, 1, 128, 16, [500, 90], 6)
    c["ks"], c["vs"] = torch.full_like(c["ks"], 0.02), torch.full_like(c["vs"], 0.03)
    tensors = _check(c)
    dev = {k: v.to(DEVICE) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    numbers = flash_attention_decode_paged(dev["q"][:, :, 0], dev["k"], dev["v"], dev["table"], dev["lens"], k_scale=0.02,
                                           v_scale=0.03, block_index=dev["index"])
    np.testing.assert_array_equal(f64(numbers)[:, :, None], tensors)


def test_all_blocks_listed_is_no_list():
    c = _case(3, "int8", torch.float16, 2, 8, 2, 2, 128, 16, [500, 90])
    plain = _check(c)
    c["index"] = torch.arange(c["table"].shape[1], dtype=torch.int32).expand(2, 2, -1)
    assert np.abs(_check(c) - plain).max() < 1e-2


def test_lists_with_holes_strays_and_repeats():
    c = _case(4, "e4m3", torch.float16, 1, 4, 1, 1, 64, 16, [100])
    c["index"] = torch.tensor([[[-1, 5, -7, 2, 7, 1000, 2, 2 ** 31 - 1, 6, -2 ** 31]]], dtype=torch.int32)
    _check(c)


@pytest.mark.parametrize("splits", [1, 2, 7, 32])
@pytest.mark.parametrize("kind", ["e4m3", "same"])
def test_shares(splits, kind):
    lens = [3000, 1, 0, 1500, 64, 2999]
    c = _case(5, kind, torch.bfloat16, 6, 8, 2, 1, 64, 16, lens, 40 if kind == "same" else 0)
    _check(c, num_splits=splits)


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("rows", [1, 6, 30])
def test_both_merges(fused, rows, monkeypatch):
    monkeypatch.setattr(_native, "FUSED_SPLIT_MERGE", fused)
    _check(_case(6, "int8", torch.float16, 3, 8, 2, rows, 128, 32, [2000, 40, 1111]))


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("heads,kv_heads,rows,dim,lens", [
    (8, 8, 1, 32, [1500, 700, 901]),                                # many rounds of a wave: no pads
    (4, 1, 1, 128, [1] * 40 + [9000] + [0, 33] * 30),               # one long sequence among short ones
    (8, 1, 20, 64, [20] * 70 + [2500, 64, 65]), (8, 1, 20, 64, [2500, 3100])])  # blocks of many rows
def test_shares_of_uneven_sequences(fused, heads, kv_heads, rows, dim, lens, monkeypatch):
    monkeypatch.setattr(_native, "FUSED_SPLIT_MERGE", fused)
    _check(_case(40 + dim, "int8", torch.float16, len(lens), heads, kv_heads, rows, dim, 32, lens))


def test_many_sequences():
    g = torch.Generator().manual_seed(7)
    lens = torch.randint(0, 90, (150,), generator=g).tolist()
    _check(_case(7, "int8", torch.float16, 150, 4, 2, 1, 64, 16, lens))
    _check(_case(8, "e4m3", torch.float16, 150, 2, 1, 1, 32, 8, lens))


def test_context_past_the_table_and_negative():
    c = _case(9, "int8", torch.float16, 3, 4, 2, 1, 64, 16, [64, 64, 64])
    c["lens"] = int32([10 ** 6, -5, 2 ** 31 - 1])
    _check(c)


def test_pages_that_are_none():
    c = _case(10, "e4m3", torch.bfloat16, 2, 8, 2, 2, 128, 16, [300, 200])
    c["table"][0, 3], c["table"][0, 7], c["table"][1, 0] = -1, 10 ** 9, -2 ** 31
    _check(c)
    c = _case(11, "e4m3", torch.bfloat16, 2, 8, 2, 2, 64, 8, [300, 200])
    c["table"][0, 3:9], c["table"][1, 1] = -1, 10 ** 9
    _check(c)
    c["table"][:] = -1
    assert (_check(c) == 0).all()


@pytest.mark.parametrize("kind,block", [("e4m3", 16), ("e4m3", 4), ("same", 16), ("same", 8)])
def test_nan_behind_the_context_and_in_absent_pages(kind, block):
    # page 0 (which absent keys read instead), the rows behind the context and unused pages hold NaN
    c = _case(12, kind, torch.float16, 2, 8, 2, 2, 64, block, [45, 21], 12 if kind == "same" else 0, spare=4)
    used = torch.zeros(c["k"].shape[:2], dtype=torch.bool)
    c["table"][0, 1] = -1
    for b, n in enumerate([45, 21]):
        for at in range(n):
            page = int(c["table"][b, at // block])
            if page >= 0:
                used[page, at % block] = True
    for name in ("k", "v"):
        x = c[name].float()
        x[~used] = float("nan")
        c[name] = x.to(c[name].dtype)
    if c["ks"] is not None:
        empty = ~used.any(1)
        c["ks"][empty], c["vs"][empty] = float("nan"), float("nan")
    dev = f64(_run(c, True))
    assert np.isfinite(dev).all()
    for name in ("k", "v", "ks", "vs"):
        if c[name] is not None:
            c[name] = torch.nan_to_num(c[name].float()).to(c[name].dtype)
    _check(c)


@pytest.mark.parametrize("kind", ["e4m3", "same"])
@pytest.mark.parametrize("block,rows,what", [(16, 5, float("nan")), (4, 5, float("nan")), (64, 40, float("nan")),
                                             (16, 5, float("inf"))])
def test_not_finite_values_that_a_row_does_not_see(kind, block, rows, what):
    # the last key is the last row's only: the rows before stay as they are
    if kind == "e4m3" and what == float("inf"):
        pytest.skip("e4m3 has no infinity")
    c = _case(13, kind, torch.float16, 2, 4, 2, rows, 64, block, [70, 41], 30 if kind == "same" else 0)
    if kind == "same":
        c["index"] = torch.arange(c["table"].shape[1], dtype=torch.int32).expand(2, 2, -1)
    clean = _check(c)
    page, at = int(c["table"][1, 40 // block]), 40 % block
    v = c["v"].float()
    v[page, at, 1, 3] = what
    c["v"] = v.to(c["v"].dtype)
    got = f64(_run(c, True))
    hit = np.zeros(got.shape, dtype=bool)
    hit[1, 2:, -1, 3] = True
    assert (np.isnan(got[hit]) if np.isnan(what) else np.isinf(got[hit])).all()
    np.testing.assert_array_equal(got[~hit], clean[~hit])


def test_extreme_scales_and_queries():
    c = _case(14, "int8", torch.float16, 2, 8, 2, 1, 64, 16, [500, 90])
    c["vs"] *= torch.exp2(torch.randint(-30, 30, c["vs"].shape).float())  # far apart within a sequence
    _check(c)
    c["vs"][:] = 0.0
    assert (f64(_run(c, True)) == 0).all()
    c = _case(15, "e4m3", torch.bfloat16, 2, 8, 2, 1, 64, 16, [500, 90])
    c["q"], c["ks"] = (c["q"].float() * 2.0 ** 100).bfloat16(), c["ks"] * 2.0 ** -100
    _check(c)
    c["q"], c["ks"] = (c["q"].float() * 2.0 ** -220).bfloat16(), c["ks"] * 2.0 ** 120 * 2.0 ** 100
    _check(c)
    c["q"][:] = 0
    _check(c)


def test_peaked_logits():
    # logits over hundreds: the running maximum moves often
    c = _case(16, "int8", torch.float16, 2, 8, 2, 1, 128, 16, [900, 90])
    c["q"] = c["q"] * 40
    _check(c)


def test_a_query_that_is_not_finite_stays_its_rows_own():
    c = _case(17, "int8", torch.bfloat16, 1, 8, 2, 3, 64, 16, [90])
    clean = _check(c)
    c["q"][0, 5, 1, 7] = float("nan")
    got = f64(_run(c, True))
    assert np.isnan(got[0, 5, 1]).all()
    got[0, 5, 1] = clean[0, 5, 1]
    np.testing.assert_array_equal(got, clean)


def test_strided():
    c = _case(18, "e4m3", torch.float16, 2, 8, 2, 2, 64, 16, [200, 90], 7)
    want = f64(_run(c, True))
    q = torch.zeros(2, 2, 8, 96, dtype=torch.float16, device=DEVICE)
    q[..., :64] = c["q"].transpose(1, 2).to(DEVICE)
    both = torch.stack([c["k"].view(torch.uint8), c["v"].view(torch.uint8)], 1).to(DEVICE).view(torch.float8_e4m3fn)
    kv = torch.stack([c["ks"], c["vs"]], -1).to(DEVICE)
    lens = torch.stack([c["lens"], c["lens"]], 1).to(DEVICE)[:, 0]
    index = c["index"].permute(2, 0, 1).contiguous().to(DEVICE).permute(1, 2, 0)
    got = flash_attention_decode_paged_multi(q[..., :64].transpose(1, 2), both[:, 0], both[:, 1],
                                             c["table"].t().contiguous().to(DEVICE).t(), lens, k_scale=kv[..., 0],
                                             v_scale=kv[..., 1], block_index=index)
    np.testing.assert_array_equal(f64(got), want)


def test_far_pages_of_a_large_cache():
    # byte offsets past 32 bits
    blocks, block, heads, dim = 2 ** 16 + 8, 256, 2, 128
    g = torch.Generator().manual_seed(19)
    c = _case(19, "int8", torch.float16, 1, 4, heads, 1, dim, block, [700])
    k, v = (torch.zeros(blocks, block, heads, dim, dtype=torch.int8, device=DEVICE) for _ in range(2))
    ks, vs = (torch.ones(blocks, heads, device=DEVICE) for _ in range(2))
    far = torch.randperm(8, generator=g)[:3] + 2 ** 16
    for i, page in enumerate(far.tolist()):
        near = int(c["table"][0, i])
        k[page], v[page] = c["k"][near].to(DEVICE), c["v"][near].to(DEVICE)
        ks[page], vs[page] = c["ks"][near].to(DEVICE), c["vs"][near].to(DEVICE)
    got = flash_attention_decode_paged(c["q"][:, :, 0].to(DEVICE), k, v, far.to(torch.int32)[None].to(DEVICE),
                                       c["lens"].to(DEVICE), k_scale=ks, v_scale=vs)
    np.testing.assert_array_equal(f64(got)[:, :, None], _check(c))


def test_same_call_same_bits():
    c = _case(20, "int8", torch.float16, 4, 8, 2, 1, 128, 64, [3000, 100, 2222, 4000])
    first = f64(_run(c, True))
    for _ in range(5):
        np.testing.assert_array_equal(f64(_run(c, True)), first)


def test_two_streams():
    cs = [_case(21 + i, "e4m3", torch.float16, 3, 8, 2, 1, 128, 16, [3000, 100, 2222]) for i in range(4)]
    want = [f64(_run(c, True)) for c in cs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    torch.cuda.synchronize()
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(_run(cs[i % 4], True))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        np.testing.assert_array_equal(f64(g), want[i % 4])


@pytest.mark.parametrize("warm", [True, False])
def test_captured_and_replayed(warm):
    c = _case(25, "int8", torch.bfloat16, 3, 8, 2, 1, 128, 16, [3000, 100, 2222])
    dev = {k: v.to(DEVICE) if isinstance(v, torch.Tensor) else v for k, v in c.items()}

    def call():
        return flash_attention_decode_paged(dev["q"][:, :, 0], dev["k"], dev["v"], dev["table"], dev["lens"],
                                            k_scale=dev["ks"], v_scale=dev["vs"])

    eager = [call()]
    stream = torch.cuda.Stream()
    if warm:
        with torch.cuda.stream(stream):
            call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = call()
    for lens in ([3000, 100, 2222], [17, 3000, 0], [2999, 1, 64]):
        dev["lens"].copy_(int32(lens))
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert (out.float() - want.float()).abs().max() <= 2.0 ** -6 * want.float().abs().max()
        _ = (dev["q"].float() * 2).sum().item()
        c["lens"] = int32(lens)
        _check(c)
    assert eager[0].shape == out.shape


def test_a_step_of_a_serving_loop():
    """allocate, append, select and attend together over three steps: a prompt
    chunk and two single tokens; each sequence's result is the oracle's over
    the oracle's own cache."""
    g = torch.Generator().manual_seed(26)
    batch, heads, kv_heads, dim, block, pool = 3, 8, 2, 64, 16, 40
    kind = "e4m3"
    table = torch.full((batch, 12), -1, dtype=torch.int32, device=DEVICE)
    free = torch.randperm(pool, generator=g).to(torch.int32).to(DEVICE)
    head = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    lens = torch.zeros(batch, dtype=torch.int32, device=DEVICE)
    k_cache, v_cache = (codes(g, (pool, block, kv_heads, dim), kind, torch.float16).to(DEVICE) for _ in range(2))
    ks, vs = (torch.ones(pool, kv_heads, device=DEVICE) for _ in range(2))
    bounds = torch.zeros(pool, kv_heads, 2, dim, dtype=torch.float16, device=DEVICE)
    ref = [f64(t) for t in (k_cache, v_cache, ks, vs, bounds)]
    ref_table, ref_head, ref_lens = f64(table).astype(int), 0, [0] * batch
    for news in ([100, 7, 31], [1, 1, 1], [1, 0, 1]):
        tokens = sum(news)
        key, value = (torch.randn(tokens, kv_heads, dim, generator=g).half() for _ in range(2))
        q = (torch.randn(batch, heads, dim, generator=g) * 2).half()
        new = int32(news).to(DEVICE)
        slots, cu, head = paged_kvcache_allocate(table, lens, new, free, free_head=head, block_size=block, num_tokens=tokens)
        paged_kvcache_append(key.to(DEVICE), value.to(DEVICE), k_cache, v_cache, slots, k_scale=ks, v_scale=vs,
                             key_bounds=bounds)
        lens = lens + new
        index = paged_kvcache_select(q.to(DEVICE), bounds, table, lens, 4, block_size=block, keep_first=1)
        dense = flash_attention_decode_paged(q.to(DEVICE), k_cache, v_cache, table, lens, k_scale=ks, v_scale=vs)
        sparse = flash_attention_decode_paged(q.to(DEVICE), k_cache, v_cache, table, lens, k_scale=ks, v_scale=vs,
                                              block_index=index)
        ref_slots, _, ref_head, ref_table = oracle.allocate(ref_table, ref_lens, news, free.tolist(), ref_head, block, tokens)
        oracle.append(f64(key), ref[0], ref[2], ref[4], ref_slots, kind)
        oracle.append(f64(value), ref[1], ref[3], None, ref_slots, kind)
        ref_lens = [a + b for a, b in zip(ref_lens, news)]
        ref_index = oracle.select(f64(q)[:, :, None], ref[4], ref_table, ref_lens, 4, block, 1, 1)
        np.testing.assert_array_equal(slots.cpu().numpy(), ref_slots)
        np.testing.assert_array_equal(index.cpu().numpy(), ref_index)
        for got, chosen in ((dense, None), (sparse, ref_index)):
            want = oracle.attend(f64(q)[:, :, None], ref[0], ref[1], ref_table, ref_lens, ref[2], ref[3], chosen)
            case = dict(q=q[:, :, None], k=torch.from_numpy(ref[0]), v=torch.from_numpy(ref[1]),
                        table=torch.from_numpy(ref_table), lens=int32(ref_lens), ks=torch.from_numpy(ref[2]),
                        vs=torch.from_numpy(ref[3]), index=None if chosen is None else torch.from_numpy(chosen), kind=kind)
            assert (np.abs(f64(got)[:, :, None] - want) <= _bound(case, want, False)).all()
