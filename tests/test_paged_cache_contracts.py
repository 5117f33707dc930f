"""Refusals of the paged cache operators (CPU: each comes before the platform
check), their C entry points' checks, and the oracle against hand-made cases."""

import ctypes

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
from paged_cases import int32


def _allocate_args():
    return dict(block_table=torch.zeros(2, 4, dtype=torch.int32), context_lens=int32([3, 0]), new_lens=int32([1, 5]),
                free_blocks=int32([5, 6, 7]), free_head=int32([0]), block_size=4, num_tokens=6)


def _append_args(cache=torch.float8_e4m3fn, dim=64):
    shape = (5, 16, 2, dim)
    return dict(key=torch.zeros(3, 2, dim, dtype=torch.float16), value=torch.zeros(3, 2, dim, dtype=torch.float16),
                k_cache=torch.zeros(shape, dtype=torch.float32).to(cache),
                v_cache=torch.zeros(shape, dtype=torch.float32).to(cache), slot_mapping=torch.arange(3),
                k_scale=torch.ones(5, 2), v_scale=torch.ones(5, 2),
                key_bounds=torch.zeros(5, 2, 2, dim, dtype=torch.float16))


def _select_args():
    return dict(query=torch.zeros(2, 8, 64, dtype=torch.bfloat16),
                key_bounds=torch.zeros(9, 2, 2, 64, dtype=torch.bfloat16),
                block_table=torch.zeros(2, 4, dtype=torch.int32), context_lens=int32([40, 64]), num_selected=3,
                block_size=16, keep_first=1, keep_last=1)


CALLS = {"allocate": (paged_kvcache_allocate, _allocate_args), "append": (paged_kvcache_append, _append_args),
         "select": (paged_kvcache_select, _select_args)}


def _call(name, **changes):
    function, make = CALLS[name]
    args = make()
    for key, change in changes.items():
        args[key] = change(args[key]) if callable(change) else change
    names = {"allocate": 4, "append": 5, "select": 5}[name]
    values = list(args.items())
    return function(*(v for _, v in values[:names]), **dict(values[names:]))


@pytest.mark.parametrize("name", sorted(CALLS))
def test_complete_calls_reach_the_platform_check(name):
    with pytest.raises(RuntimeError, match="requires|supports"):
        _call(name)


REFUSED = [
    ("allocate", "block_table", lambda t: t.long(), "block_table must be a int32"),
    ("allocate", "block_table", lambda t: t[0], "block_table must be a int32"),
    ("allocate", "block_table", lambda t: t[:, :0], "at least one"),
    ("allocate", "block_table", lambda t: t[:1].expand(2, 4), "expanded"),
    ("allocate", "context_lens", lambda t: t[:1], "context_lens must be"),
    ("allocate", "new_lens", lambda t: t.float(), "new_lens must be"),
    ("allocate", "free_blocks", lambda t: t[None], "free_blocks must be"),
    ("allocate", "free_head", lambda t: t.long(), "free_head must be"),
    ("allocate", "block_size", 3, "power of two"), ("allocate", "block_size", 512, "power of two"),
    ("allocate", "block_size", 0, "block_size must be an integer"), ("allocate", "block_size", True, "block_size"),
    ("allocate", "num_tokens", -1, "num_tokens"), ("allocate", "num_tokens", 2.0, "num_tokens"),
    ("append", "key", lambda t: t.float(), "key must be a float16"), ("append", "key", lambda t: t[0], "key must be"),
    ("append", "value", lambda t: t.bfloat16(), "value must be"), ("append", "value", lambda t: t[:2], "value must be"),
    ("append", "k_cache", lambda t: t.float(), "key's dtype"),
    ("append", "k_cache", lambda t: t[..., :32], "k_cache must be"),
    ("append", "v_cache", lambda t: t[:4], "v_cache must be"),
    ("append", "v_cache", lambda t: t.float().half(), "v_cache must be"),
    ("append", "k_cache", lambda t: t[:, :1].expand(5, 16, 2, 64), "expanded"),
    ("append", "k_cache", lambda t: t.transpose(1, 3).contiguous().transpose(1, 3), "unit last stride"),
    ("append", "slot_mapping", lambda t: t.int(), "slot_mapping must be"),
    ("append", "slot_mapping", lambda t: t[:2], "slot_mapping must be"),
    ("append", "k_scale", None, "k_scale must be a torch.Tensor"),
    ("append", "v_scale", lambda t: t.half(), "v_scale must be"),
    ("append", "k_scale", lambda t: t[:, :1], "k_scale must be"),
    ("append", "k_scale", lambda t: t[:, :1].expand(5, 2), "expanded"),
    ("append", "key_bounds", lambda t: t.bfloat16(), "key_bounds must be"),
    ("append", "key_bounds", lambda t: t[:, :, :1], "key_bounds must be"),
    ("append", "key_bounds", lambda t: t[:1].expand(5, 2, 2, 64), "expanded"),
    ("select", "query", lambda t: t.float(), "query must be"), ("select", "query", lambda t: t[0], "query must be"),
    ("select", "query", lambda t: t[:, :7], "multiple of cache heads"),
    ("select", "query", lambda t: t[:, :, None][:, :, :0], "must be positive"),
    ("select", "key_bounds", lambda t: t.half(), "key_bounds must be"),
    ("select", "key_bounds", lambda t: t[:, :, :1], "key_bounds must be"),
    ("select", "block_table", lambda t: t[:1], "block_table must be"),
    ("select", "block_table", lambda t: t[:, :0], "at least one logical block"),
    ("select", "context_lens", lambda t: t.long(), "context_lens must be"),
    ("select", "num_selected", 0, "num_selected"), ("select", "num_selected", 1, "must not exceed"),
    ("select", "keep_first", -1, "keep_first"), ("select", "keep_last", 3, "must not exceed"),
    ("select", "block_size", 24, "power of two"),
]


@pytest.mark.parametrize("name,argument,change,message", REFUSED)
def test_refused(name, argument, change, message):
    with pytest.raises((ValueError, TypeError), match=message):
        _call(name, **{argument: change})


@pytest.mark.parametrize("dtype,dim", [(torch.float8_e4m3fn, 16), (torch.int8, 48), (torch.float16, 48)])
def test_head_dims_of_a_cache(dtype, dim):
    args = _append_args(dtype, dim)
    if dtype == torch.float16:
        args["k_scale"] = args["v_scale"] = None
    with pytest.raises(ValueError, match="head_dim"):
        paged_kvcache_append(**args)


def test_scales_are_for_8_bit_caches():
    with pytest.raises(ValueError, match="apply to"):
        paged_kvcache_append(**_append_args(torch.float16))


def test_caches_that_require_grad_are_refused(monkeypatch):
    import fa_rdna3._validation as validation

    monkeypatch.setattr(validation, "_require_platform", lambda device: None)
    args = _append_args(torch.float16) | {"k_scale": None, "v_scale": None}
    args["k_cache"] = args["k_cache"].half().requires_grad_()
    with pytest.raises(RuntimeError, match="inference-only"):
        paged_kvcache_append(**args)


def test_entry_points_check_before_they_launch():
    lib = _native.lib()
    for name, struct in (("fa_paged_allocate", _native.AllocateParams), ("fa_paged_append", _native.PagedAppendParams),
                         ("fa_paged_select", _native.SelectParams)):
        fn = getattr(lib, name)
        assert fn(None, None) == 1
        p = struct()
        assert fn(ctypes.byref(p), None) == 1
        assert b"abi_version" in lib.fa_last_error_string()
        p.abi_version = _native.ABI_VERSION
        assert fn(ctypes.byref(p), None) != 0
    p = _native.PagedAppendParams()
    p.abi_version, p.kv_format, p.head_dim, p.heads_kv, p.num_blocks, p.block_size = _native.ABI_VERSION, 1, 64, 1, 1, 16
    assert lib.fa_paged_append(ctypes.byref(p), None) == 0  # no tokens
    p.num_tokens = 1
    assert lib.fa_paged_append(ctypes.byref(p), None) == 1
    p.head_dim = 16
    assert lib.fa_paged_append(ctypes.byref(p), None) == 2
    assert lib.fa_select_workspace_bytes(2, 4, 100) == 2 * 4 * 100 * 8
    assert lib.fa_select_workspace_bytes(0, 4, 100) == 0


def test_oracle_allocates_in_order():
    table = np.full((3, 3), 9)
    slots, cu, head, after = oracle.allocate(table, [3, 0, 4], [2, 0, 7], [20, 21, 22], 1, 4, 12)
    # sequence 0: token 3 in its page 9, token 4 in page 21; sequence 2: page 22, then none left, then past the table
    assert slots.tolist() == [39, 84] + [88, 89, 90, 91] + [-1] * 6
    assert cu.tolist() == [0, 2, 2, 9] and head == 4
    assert after.tolist() == [[9, 21, 9], [9, 9, 9], [9, 22, -1]]


@pytest.mark.parametrize("cache,amax,exponent", [
    ("e4m3", 448.0, 0), ("e4m3", 448.5, 1), ("e4m3", 224.0, -1), ("e4m3", 1.0, -8), ("int8", 127.0, 0),
    ("int8", 127.5, 1), ("int8", 1.0, -6), ("int8", 0.0, -100), ("e4m3", 2.0 ** -133, -100), ("e4m3", 65504.0, 8)])
def test_oracle_scales(cache, amax, exponent):
    assert oracle.scale_for(amax, cache) == 2.0 ** exponent


def test_oracle_codes_are_the_type_s():
    x = torch.randn(4000, generator=torch.Generator().manual_seed(0)) * torch.logspace(-4, 3, 4000)
    x = torch.cat([x, torch.tensor([448.0, -448.0, 0.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10])]).clamp(-448, 448)
    np.testing.assert_array_equal(oracle.to_code(x.double().numpy(), "e4m3"),
                                  x.to(torch.float8_e4m3fn).double().numpy())
    np.testing.assert_array_equal(oracle.to_code(np.array([0.5, 1.5, -2.5, 300.0, np.nan]), "int8"), [0, 2, -2, 127, 0])


def test_oracle_block_scales_and_index_reduce_to_the_plain_paged_decode():
    from oracle import attention

    r = np.random.RandomState(1)
    q, k, v = r.randn(2, 4, 3, 8), r.randn(9, 4, 2, 8), r.randn(9, 4, 2, 8)
    table, lens = r.permutation(9)[:8].reshape(2, 4), [14, 5]
    ks, vs = r.rand(9, 2) + 0.5, r.rand(9, 2) + 0.5
    got = oracle.attend(q, k / ks[:, None, :, None], v / vs[:, None, :, None], table, lens, ks, vs,
                        np.tile(np.arange(4), (2, 2, 1)), causal=True)
    want = attention.paged_attention(q, k, v, table, np.array(lens), causal=True)
    np.testing.assert_allclose(got, want, atol=1e-5)


# ---------------------------------------------------------------------------
# Paged decode over block scales and listed blocks
# ---------------------------------------------------------------------------

def _decode_args(cache=torch.int8, dim=64, index=True):
    shape = (9, 16, 2, dim)
    return dict(query=torch.zeros(2, 8, dim, dtype=torch.float16), k_cache=torch.zeros(shape).to(cache),
                v_cache=torch.zeros(shape).to(cache), block_table=torch.zeros(2, 4, dtype=torch.int32),
                context_lens=int32([40, 64]), k_scale=torch.ones(9, 2), v_scale=torch.ones(9, 2),
                block_index=torch.zeros(2, 2, 3, dtype=torch.int32) if index else None)


@pytest.mark.parametrize("cache,scales,index", [
    (torch.int8, True, False), (torch.int8, True, True), (torch.float8_e4m3fn, True, False),
    (torch.float8_e4m3fn, False, True), (torch.float16, False, True)])
@pytest.mark.parametrize("rows", [0, 3])
def test_complete_decodes_reach_the_platform_check(cache, scales, index, rows):
    args = _decode_args(cache, index=index)
    if not scales:
        args["k_scale"] = args["v_scale"] = None
    if rows:
        args["query"] = torch.zeros(2, 8, rows, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="requires|supports"):
        (flash_attention_decode_paged_multi if rows else flash_attention_decode_paged)(**args)


@pytest.mark.parametrize("argument,change,message", [
    ("query", lambda t: t.float(), "float16 or bfloat16"), ("query", lambda t: t[0], "paged query must be"),
    ("query", lambda t: t[..., :48], "need head_dim"), ("query", lambda t: t[..., :32], "head_dim"),
    ("query", lambda t: t[:, :7], "multiple of cache heads"), ("query", lambda t: None, "paged query must be"),
    ("k_cache", lambda t: t.half(), "share a dtype"), ("k_cache", lambda t: t[0], "caches must be"),
    ("v_cache", lambda t: t[:5], "same shape"), ("v_cache", lambda t: t.to(torch.float8_e4m3fn), "share a dtype"),
    ("k_scale", lambda t: 1.0, "k_scale must be a torch.Tensor"), ("v_scale", lambda t: None, "v_scale must be"),
    ("k_scale", lambda t: t.half(), "k_scale must be"), ("v_scale", lambda t: t[:, :1], "v_scale must be"),
    ("k_scale", lambda t: t[:4], "k_scale must be"),
    ("block_index", lambda t: t.long(), "block_index must be"), ("block_index", lambda t: t[0], "block_index must be"),
    ("block_index", lambda t: t[:, :1], "block_index must be"), ("block_index", lambda t: t[..., :0], "at least one block"),
    ("block_table", lambda t: t.long(), "block_table must be"), ("context_lens", lambda t: t[:1], "context_lens"),
])
def test_refused_decodes(argument, change, message):
    args = _decode_args()
    args[argument] = change(args[argument])
    with pytest.raises((ValueError, TypeError), match=message):
        flash_attention_decode_paged(**args)


def test_refused_decodes_by_cache():
    args = _decode_args(torch.float16)
    with pytest.raises(ValueError, match="apply to"):
        flash_attention_decode_paged(**args)
    args = _decode_args(torch.float8_e4m3fn) | {"k_scale": 0.5}
    with pytest.raises(TypeError, match="k_scale"):
        flash_attention_decode_paged(**args)
    args = _decode_args(torch.float8_e4m3fn) | {"k_scale": -0.5, "v_scale": None}
    with pytest.raises(ValueError, match="positive finite"):
        flash_attention_decode_paged(**args)
    args = _decode_args(torch.float16, 16) | {"k_scale": None, "v_scale": None}
    with pytest.raises(ValueError, match="need head_dim"):
        flash_attention_decode_paged(**args)
    args = _decode_args()
    for bad in (0, 33, True):
        with pytest.raises((ValueError, RuntimeError)):
            flash_attention_decode_paged(**args, num_splits=bad)


def test_paged_blocks_entry_point_checks_before_it_launches():
    lib = _native.lib()
    assert lib.fa_decode_paged_blocks(None, None) == 1
    p = _native.PagedBlocksParams()
    assert lib.fa_decode_paged_blocks(ctypes.byref(p), None) == 1 and b"abi_version" in lib.fa_last_error_string()
    p.abi_version, p.kv_format, p.head_dim = _native.ABI_VERSION, 2, 64
    p.batch, p.heads_q, p.heads_kv, p.seqlen_q = 2, 8, 2, 1
    p.num_blocks, p.max_blocks, p.block_size, p.shares = 9, 4, 16, 5
    assert lib.fa_decode_paged_blocks(ctypes.byref(p), None) == 1 and b"rows" in lib.fa_last_error_string()
    # two partials for each share, KV head and query row of its group: D sums, a maximum and a total
    assert lib.fa_paged_blocks_workspace_bytes(ctypes.byref(p)) == 2 * 5 * 2 * 4 * (64 + 2) * 4
    for field, value, status in (("kv_format", 3, 1), ("head_dim", 48, 2), ("block_size", 24, 1), ("shares", 4097, 1),
                                 ("max_blocks", 2 ** 27, 2), ("heads_kv", 3, 1), ("batch", 70000, 1)):
        old = getattr(p, field)
        setattr(p, field, value)
        assert lib.fa_decode_paged_blocks(ctypes.byref(p), None) == status, field
        assert lib.fa_paged_blocks_workspace_bytes(ctypes.byref(p)) == 0, field
        setattr(p, field, old)
