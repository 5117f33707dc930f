"""paged_kvcache_allocate, _append and _select against the 64-bit oracle.

Every result here is exact: tables and indices are whole numbers, scales are
powers of two (a quotient by one is exact, so a code is the single rounding of
the value), and bounds are keys.  Selection sums exact products in 64 bits;
its random scores differ by far more than the 2^-45 the order of 512 terms can
make.
"""

import numpy as np
import pytest
import torch

from fa_rdna3 import paged_kvcache_allocate, paged_kvcache_append, paged_kvcache_select
from oracle import paged_cache as oracle
from paged_cases import CACHES, codes, f64, int32, same_values, slots_of, table_of

pytestmark = pytest.mark.gpu
DEVICE = "cuda"


def _generator(seed):
    return torch.Generator().manual_seed(seed)


# ---------------------------------------------------------------------------
# Tables and slots
# ---------------------------------------------------------------------------

def _allocate(table, ctx, new, free, head, block, tokens):
    dev = torch.as_tensor(table, dtype=torch.int32).to(DEVICE)
    free_d = int32(list(free)).to(DEVICE)
    slots, cu, nxt = paged_kvcache_allocate(dev, int32(ctx).to(DEVICE), int32(new).to(DEVICE), free_d,
                                            free_head=None if head is None else int32([head]).to(DEVICE),
                                            block_size=block, num_tokens=tokens)
    want = oracle.allocate(np.asarray(table), ctx, new, list(free), head or 0, block, tokens)
    assert slots.dtype == torch.int64 and cu.dtype == nxt.dtype == torch.int32
    np.testing.assert_array_equal(slots.cpu().numpy(), want[0])
    np.testing.assert_array_equal(cu.cpu().numpy(), want[1])
    assert nxt.item() == want[2]
    np.testing.assert_array_equal(dev.cpu().numpy(), want[3])


@pytest.mark.parametrize("batch,block,longest_ctx,longest_new", [
    (1, 1, 0, 1), (1, 16, 0, 1000), (3, 4, 30, 9), (64, 16, 500, 1), (65, 64, 100, 300), (257, 8, 40, 7),
    (1024, 32, 90, 3), (1025, 32, 90, 3), (2500, 16, 20, 2), (5, 256, 2000, 600)])
def test_allocate(batch, block, longest_ctx, longest_new):
    r = np.random.RandomState(batch + block)
    ctx = r.randint(0, longest_ctx + 1, batch).tolist()
    new = r.randint(0, longest_new + 1, batch).tolist()
    blocks = -(-(longest_ctx + longest_new) // block) + 1
    free = r.permutation(batch * blocks + 7)
    table = r.randint(0, 1000, (batch, blocks))
    _allocate(table, ctx, new, free, 3, block, sum(new) + 5)


def test_allocate_edges():
    # nothing new; negative lengths; a slot map shorter than the tokens; no free blocks; a table that ends
    _allocate([[4, 5]], [3], [0], [], None, 4, 0)
    _allocate([[4, 5], [6, 7]], [-3, 2], [2, -1], [8, 9], None, 4, 3)
    _allocate([[4, 5, 6]], [1], [11], [8, 9, 10], 1, 4, 4)
    _allocate([[4, 5], [6, 7]], [4, 8], [3, 3], [], 0, 4, 6)
    _allocate([[-1, 5], [6, 7]], [2, 7], [3, 30], [11], -2, 4, 40)


def test_allocate_of_lengths_without_bound():
    # The work is the tensors', not the lengths': each sequence asks for 2^31 - 1
    # tokens and gets its table's 8 blocks, while the list lasts; sums stop at 2^31 - 1.
    top = 2 ** 31 - 1
    table = torch.full((300, 8), 5, dtype=torch.int32, device=DEVICE)
    free = torch.arange(2000, dtype=torch.int32, device=DEVICE)
    slots, cu, nxt = paged_kvcache_allocate(table, torch.zeros(300, dtype=torch.int32, device=DEVICE),
                                            torch.full((300,), top, dtype=torch.int32, device=DEVICE), free,
                                            block_size=16, num_tokens=200)
    torch.testing.assert_close(table.flatten().cpu(), torch.where(torch.arange(2400) < 2000, torch.arange(2400), -1).int())
    assert slots.tolist() == list(range(128)) + [-1] * 72
    assert cu.tolist() == [0] + [top] * 300
    assert nxt.item() == 2400
    head = int32([top - 5]).to(DEVICE)
    nxt = paged_kvcache_allocate(table, torch.zeros(300, dtype=torch.int32, device=DEVICE),
                                 torch.full((300,), 20, dtype=torch.int32, device=DEVICE), free, free_head=head,
                                 block_size=16, num_tokens=6000)[2]
    assert nxt.item() == top


def test_allocate_strided_and_repeated():
    wide = torch.full((3, 8), 77, dtype=torch.int32, device=DEVICE)
    table = wide[:, ::2]
    lens = int32([5, 9, 0, 9, 8, 9]).to(DEVICE)[::2]
    new = int32([6, 1, 3]).to(DEVICE)
    free = torch.arange(40, dtype=torch.int32, device=DEVICE)[::3]
    want = oracle.allocate(table.cpu().numpy(), lens.tolist(), new.tolist(), free.tolist(), 0, 4, 10)
    for _ in range(2):
        slots, cu, nxt = paged_kvcache_allocate(table, lens, new, free, block_size=4, num_tokens=10)
        np.testing.assert_array_equal(slots.cpu().numpy(), want[0])
        np.testing.assert_array_equal(table.cpu().numpy(), want[3])
        assert nxt.item() == want[2] and (wide[:, 1::2] == 77).all()


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------

def _check_append(key, value, kc, vc, slots, kind, ks=None, vs=None, bounds=None, calls=1):
    dev = [None if t is None else t.to(DEVICE) for t in (kc, vc, ks, vs, bounds)]
    for _ in range(calls):
        paged_kvcache_append(key.to(DEVICE), value.to(DEVICE), dev[0], dev[1], slots.to(DEVICE), k_scale=dev[2],
                             v_scale=dev[3], key_bounds=dev[4])
    ref = [None if t is None else f64(t) for t in (kc, vc, ks, vs, bounds)]
    oracle.append(f64(key), ref[0], ref[2], ref[4], slots.tolist(), kind)
    oracle.append(f64(value), ref[1], ref[3], None, slots.tolist(), kind)
    for got, want in zip(dev, ref):
        if got is not None:
            same_values(got, want)
    return dev


def _append_case(seed, kind, dtype, heads, dim, block, contexts, news, bounds=True):
    g = _generator(seed)
    blocks = -(-max(c + n for c, n in zip(contexts, news)) // block)
    table, pool = table_of(g, len(contexts), blocks)
    slots = slots_of(table, contexts, news, block)
    rows = [(torch.randn(len(slots), heads, dim, generator=g)
             * torch.exp2(torch.randint(-3, 4, (len(slots), heads, 1), generator=g).float())).to(dtype) for _ in range(2)]
    caches = [codes(g, (pool, block, heads, dim), kind, dtype) for _ in range(2)]
    scale = [torch.exp2(torch.randint(-9, -4, (pool, heads), generator=g).float()) if kind in CACHES else None
             for _ in range(2)]
    ends = torch.randn(2, pool, heads, dim, generator=g).to(dtype)
    bnd = torch.stack([torch.minimum(*ends), torch.maximum(*ends)], 2) if bounds else None
    return dict(key=rows[0], value=rows[1], kc=caches[0], vc=caches[1], slots=slots, kind=kind, ks=scale[0],
                vs=scale[1], bounds=bnd)


@pytest.mark.parametrize("kind", ["e4m3", "int8", "same"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,dim,block,contexts,news", [
    (1, 32, 1, [3], [2]), (2, 64, 16, [0, 15, 16, 33], [1, 1, 1, 1]), (8, 128, 64, [63, 64, 10, 0], [1, 2, 100, 257]),
    (3, 256, 8, [5, 0], [21, 3]), (1, 512, 32, [40], [30]), (5, 128, 256, [250, 3], [300, 5]), (2, 128, 128, [7], [122])])
def test_append(kind, dtype, heads, dim, block, contexts, news):
    _check_append(**_append_case(heads + dim, kind, dtype, heads, dim, block, contexts, news))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_many_tokens(kind):
    # enough tokens for several of them to share a workgroup
    _check_append(**_append_case(3, kind, torch.bfloat16, 4, 64, 16, [0, 5, 31] * 20, [64, 90, 1] * 20, bounds=False))


def test_append_head_dim_16():
    _check_append(**_append_case(4, "same", torch.float16, 3, 16, 16, [5, 0], [40, 3]))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_append_twice_is_append_once(kind):
    _check_append(calls=3, **_append_case(5, kind, torch.float16, 2, 64, 16, [3, 17, 16], [2, 20, 1]))


@pytest.mark.parametrize("kind", ["e4m3", "int8", "same"])
def test_append_drops_slots_outside_the_cache(kind):
    case = _append_case(6, kind, torch.bfloat16, 2, 64, 16, [3, 17], [5, 20])
    pool = case["kc"].shape[0]
    case["slots"][2] = -1
    case["slots"][7] = pool * 16
    case["slots"][11] = 2 ** 40
    case["slots"][12] = -2 ** 40
    _check_append(**case)
    case["slots"][:] = -1
    _check_append(**case)


@pytest.mark.parametrize("kind", ["e4m3", "int8", "same"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_not_finite_zero_and_extreme_values(kind, dtype):
    case = _append_case(7, kind, dtype, 2, 64, 16, [3, 16, 0], [6, 16, 3])
    key, value = case["key"], case["value"]
    key[0, 0, 3], key[1, 0, 5], key[2, 1, 0] = float("nan"), float("inf"), -float("inf")
    value[4, 1, :] = float("nan")
    value[7:, 0] = 0.0
    key[10, 1] = torch.finfo(dtype).max
    value[11, 1] = torch.finfo(dtype).smallest_normal / 4
    _check_append(**case)


def test_append_in_any_order_within_a_block():
    case = _append_case(8, "e4m3", torch.float16, 2, 64, 16, [20], [10])
    order = torch.tensor([3, 1, 0, 2, 9, 8, 7, 6, 5, 4])
    case["key"], case["value"] = case["key"][order].contiguous(), case["value"][order].contiguous()
    case["slots"] = case["slots"][order]
    _check_append(**case)


def test_append_strided_inputs_and_caches():
    case = _append_case(9, "int8", torch.bfloat16, 2, 64, 16, [20, 3], [10, 30])
    key = torch.randn(40, 2, 64).bfloat16()
    wide = torch.zeros(40, 4, 128, dtype=torch.bfloat16, device=DEVICE)
    wide[:, 1:3, 64:] = key.to(DEVICE)
    pool = case["kc"].shape[0]
    both = torch.stack([case["kc"], case["vc"]], 1).to(DEVICE)  # K and V of a block side by side
    kv = torch.stack([case["ks"], case["vs"]], -1).to(DEVICE)
    bounds = case["bounds"].to(DEVICE)
    slots = torch.stack([case["slots"], case["slots"]], 1).to(DEVICE)[:, 1]
    paged_kvcache_append(wide[:, 1:3, 64:], case["value"].to(DEVICE).transpose(0, 1).contiguous().transpose(0, 1),
                         both[:, 0], both[:, 1], slots, k_scale=kv[..., 0], v_scale=kv[..., 1], key_bounds=bounds)
    ref = [f64(case[n]) for n in ("kc", "vc", "ks", "vs", "bounds")]
    oracle.append(f64(key), ref[0], ref[2], ref[4], case["slots"].tolist(), "int8")
    oracle.append(f64(case["value"]), ref[1], ref[3], None, case["slots"].tolist(), "int8")
    for got, want in zip((both[:, 0], both[:, 1], kv[..., 0], kv[..., 1], bounds), ref):
        same_values(got, want)
    assert both.shape[0] == pool


def test_append_no_tokens():
    case = _append_case(10, "e4m3", torch.float16, 2, 64, 16, [20], [10])
    for name in ("key", "value", "slots"):
        case[name] = case[name][:0]
    _check_append(**case)


def test_append_far_into_a_large_cache():
    # slots and byte offsets past 32 bits: the last blocks of a cache of 4.3 GB
    blocks, block, heads, dim = 2 ** 16 + 3, 256, 2, 128
    kc = torch.zeros(blocks, block, heads, dim, dtype=torch.int8, device=DEVICE)
    vc = torch.zeros_like(kc)
    ks, vs = (torch.ones(blocks, heads, device=DEVICE) for _ in range(2))
    rows = torch.randn(4, heads, dim, generator=_generator(1)).half()
    slots = torch.tensor([0, blocks * block - 2, blocks * block - 1, (blocks - 2) * block])
    paged_kvcache_append(rows.to(DEVICE), rows.to(DEVICE), kc, vc, slots.to(DEVICE), k_scale=ks, v_scale=vs)
    flat, small = kc.view(-1, heads, dim), np.zeros((3, block, heads, dim))
    scale = np.ones((3, heads))
    near = [0, 2 * block + block - 2, 2 * block + block - 1, block]
    oracle.append(f64(rows), small, scale, None, near, "int8")
    for at, far in zip(near, slots.tolist()):
        same_values(flat[far], small.reshape(-1, heads, dim)[at])
    assert int(kc.view(torch.int32).count_nonzero()) <= 4 * heads * dim // 4


# ---------------------------------------------------------------------------
# Selection
# ---------------------------------------------------------------------------

def _check_select(q, bounds, table, ctx, count, block, first, last):
    index = paged_kvcache_select(q.to(DEVICE), bounds.to(DEVICE), table.to(DEVICE), ctx.to(DEVICE), count,
                                 block_size=block, keep_first=first, keep_last=last)
    assert index.dtype == torch.int32
    rows = q if q.dim() == 4 else q[:, :, None]
    want = oracle.select(f64(rows), f64(bounds), table.numpy(), ctx.tolist(), count, block, first, last)
    np.testing.assert_array_equal(index.cpu().numpy(), want)


def _select_case(seed, dtype, heads, kv_heads, rows, dim, blocks, batch):
    g = _generator(seed)
    table, pool = table_of(g, batch, blocks)
    q = torch.randn(batch, heads, rows, dim, generator=g).to(dtype)
    ends = torch.randn(2, pool, kv_heads, dim, generator=g).to(dtype)
    return q, torch.stack([torch.minimum(*ends), torch.maximum(*ends)], 2), table


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,rows,dim", [(4, 4, 1, 32), (8, 2, 1, 64), (32, 8, 1, 128), (10, 2, 1, 256),
                                                     (3, 1, 1, 512), (8, 2, 3, 128), (16, 1, 1, 64)])
@pytest.mark.parametrize("blocks,count,first,last", [(1, 1, 0, 1), (70, 8, 1, 2), (300, 33, 0, 0)])
def test_select(dtype, heads, kv_heads, rows, dim, blocks, count, first, last):
    q, bounds, table = _select_case(dim + blocks, dtype, heads, kv_heads, rows, dim, blocks, 3)
    ctx = int32([blocks * 16, max(1, blocks * 16 - 37), 16 * min(blocks, count) - 3])
    _check_select(q if rows > 1 else q[:, :, 0], bounds, table, ctx, count, 16, first, last)


@pytest.mark.parametrize("blocks", [1000, 5000, 9001])
def test_select_among_many(blocks):
    q, bounds, table = _select_case(1, torch.bfloat16, 4, 1, 1, 32, blocks, 2)
    _check_select(q, bounds, table, int32([blocks * 8, blocks * 8 - 1000]), 257, 8, 1, 3)


def test_select_ties_go_to_the_lower_index():
    q, bounds, table = _select_case(2, torch.float16, 4, 2, 1, 64, 200, 1)
    table = table % 5  # forty blocks of each of five scores
    for count in (1, 7, 40, 41, 199):
        _check_select(q, bounds, table, int32([200 * 16]), count, 16, 0, 1)
    _check_select(torch.zeros_like(q), bounds, table, int32([200 * 16]), 9, 16, 2, 2)


def test_select_empty_negative_and_long_contexts():
    q, bounds, table = _select_case(3, torch.float16, 4, 2, 1, 64, 20, 4)
    _check_select(q, bounds, table, int32([0, -5, 10 ** 6, 2 ** 31 - 1]), 4, 16, 1, 1)


def test_select_pages_that_are_none():
    q, bounds, table = _select_case(4, torch.bfloat16, 4, 2, 1, 64, 40, 2)
    table[0, ::3] = -1
    table[1, 5:] = 10 ** 6
    _check_select(q, bounds, table, int32([640, 640]), 12, 16, 1, 1)


def test_select_not_finite():
    q, bounds, table = _select_case(5, torch.bfloat16, 4, 2, 1, 64, 90, 1)
    page = table[0].tolist()
    bounds[page[3], :, 1, 7], bounds[page[50], :, 0, 9] = float("inf"), -float("inf")
    bounds[page[60], 0, 0], bounds[page[60], 0, 1] = float("inf"), -float("inf")  # (a block of NaN keys)
    bounds[page[70], 1, 1, 2] = float("nan")
    _check_select(q, bounds, table, int32([1440]), 5, 16, 0, 1)
    q[0, 1, 0, 4] = float("nan")
    _check_select(q, bounds, table, int32([1440]), 5, 16, 0, 1)


def test_select_extreme_bfloat16_values():
    # products past the 32-bit range are ordered all the same
    q, bounds, table = _select_case(6, torch.bfloat16, 2, 1, 1, 64, 90, 1)
    _check_select(q * 1e30, (bounds.float() * 1e37).bfloat16(), table, int32([1440]), 11, 16, 0, 1)
    _check_select((q.float() * 1e-30).bfloat16(), (bounds.float() * 1e-37).bfloat16(), table, int32([1440]), 11, 16, 0, 1)


def test_select_strided():
    q, bounds, table = _select_case(7, torch.float16, 8, 2, 2, 64, 50, 2)
    want = oracle.select(f64(q), f64(bounds), table.numpy(), [800, 333], 6, 16, 1, 1)
    wide = torch.zeros(2, 2, 8, 96, dtype=torch.float16, device=DEVICE)
    wide[..., :64] = q.transpose(1, 2).to(DEVICE)
    tall = torch.zeros(bounds.shape[0], 2, 2, 2, 64, dtype=torch.float16, device=DEVICE)
    tall[:, :, 1] = bounds.to(DEVICE)
    lens = int32([800, 0, 333, 0]).to(DEVICE)[::2]
    got = paged_kvcache_select(wide[..., :64].transpose(1, 2), tall[:, :, 1], table.to(DEVICE).t().contiguous().t(), lens,
                               6, block_size=16, keep_first=1)
    np.testing.assert_array_equal(got.cpu().numpy(), want)


# ---------------------------------------------------------------------------
# Streams, graphs, transforms
# ---------------------------------------------------------------------------

def test_captured_and_replayed():
    case = _append_case(11, "e4m3", torch.float16, 2, 64, 16, [20, 3], [1, 1])
    table = torch.full((2, 6), -1, dtype=torch.int32)
    table[0, :2], table[1, 0] = int32([4, 1]), 7
    dev = {k: v.to(DEVICE) for k, v in case.items() if isinstance(v, torch.Tensor)}
    table_d, free = table.to(DEVICE), torch.arange(8, 20, dtype=torch.int32, device=DEVICE)
    pool = 20
    for name in ("kc", "vc"):
        dev[name] = torch.zeros(pool, 16, 2, 64, dtype=torch.float8_e4m3fn, device=DEVICE)
    dev |= {name: torch.ones(pool, 2, device=DEVICE) for name in ("ks", "vs")}
    dev["bounds"] = torch.zeros(pool, 2, 2, 64, dtype=torch.float16, device=DEVICE)
    lens, new, head = int32([20, 3]).to(DEVICE), int32([1, 1]).to(DEVICE), int32([0]).to(DEVICE)
    query = torch.randn(2, 4, 64, device=DEVICE).half()

    def step():
        slots, _, nxt = paged_kvcache_allocate(table_d, lens, new, free, free_head=head, block_size=16, num_tokens=2)
        paged_kvcache_append(dev["key"], dev["value"], dev["kc"], dev["vc"], slots, k_scale=dev["ks"],
                             v_scale=dev["vs"], key_bounds=dev["bounds"])
        index = paged_kvcache_select(query, dev["bounds"], table_d, lens + new, 2, block_size=16)
        head.copy_(nxt)
        lens.add_(new)
        return slots, index

    state = [table_d, lens, head] + [dev[n] for n in ("kc", "vc", "ks", "vs", "bounds")]
    start = [t.clone() for t in state]
    rows = [(torch.randn(2, 2, 64).half().to(DEVICE), torch.randn(2, 2, 64).half().to(DEVICE)) for _ in range(40)]
    eager = []
    for k, v in rows:
        dev["key"].copy_(k), dev["value"].copy_(v)
        eager.append([t.clone() for t in step()])
    end = [t.clone() for t in state]
    for t, s in zip(state, start):
        t.copy_(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t, s in zip(state, start):
        t.copy_(s)
    for i, (k, v) in enumerate(rows):
        dev["key"].copy_(k), dev["value"].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        _ = (query.float() * i).sum().item()
        assert all(torch.equal(a, b) for a, b in zip(out, eager[i])), i
    for t, s in zip(state, end):
        assert torch.equal(t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t,
                           s.view(torch.uint8) if s.dtype == torch.float8_e4m3fn else s)


def test_rows_of_a_projection_that_is_trained_stay_outside_autograd():
    case = _append_case(12, "same", torch.float16, 2, 64, 16, [20], [3])
    dev = {k: v.to(DEVICE) for k, v in case.items() if isinstance(v, torch.Tensor)}
    key = dev["key"].requires_grad_() * 1.0
    paged_kvcache_append(key, dev["value"], dev["kc"], dev["vc"], dev["slots"])
    assert not dev["kc"].requires_grad
    with torch.inference_mode():
        cache = torch.zeros_like(dev["kc"])
    paged_kvcache_append(dev["key"].detach(), dev["value"], cache, dev["vc"], dev["slots"])
    assert cache.abs().sum() > 0


def test_transforms_are_refused():
    case = _append_case(13, "same", torch.float16, 2, 64, 16, [20], [3])
    dev = {k: v.to(DEVICE) for k, v in case.items() if isinstance(v, torch.Tensor)}
    keys = torch.stack([dev["key"], dev["key"]])

    def append(key):
        torch.ops.fa_mi355x.paged_append(key, dev["value"], dev["kc"], dev["vc"], dev["slots"], None, None, None)
        return key

    with pytest.raises(RuntimeError, match="transforms"):
        torch.vmap(append)(keys)
