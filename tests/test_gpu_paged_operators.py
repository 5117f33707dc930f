"""The operators of the paged cache called by themselves check what their
kernels read and write, and leave everything as it was when they refuse."""

import threading

import pytest
import torch

from fa_rdna3 import _native, flash_attention_decode_paged, flash_attention_decode_paged_multi

pytestmark = pytest.mark.gpu
BATCH, HEADS, KV_HEADS, DIM, BLOCK, TABLE = 2, 8, 2, 64, 16, 5
PAGES = BATCH * TABLE


def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _rand(*shape):
    return torch.randn(shape, device="cuda").half()


def _cache():
    return torch.randint(-90, 90, (PAGES, BLOCK, KV_HEADS, DIM), dtype=torch.int8, device="cuda")


def _scale():
    return torch.rand(PAGES, KV_HEADS, device="cuda") / 64


def _table():
    return torch.arange(PAGES, dtype=torch.int32, device="cuda").view(BATCH, TABLE)


ARGS = {
    "paged_allocate": lambda: dict(block_table=_table(), context_lens=_int([3, 16]), new_lens=_int([30, 1]),
                                   free_blocks=_int([9, 8, 7]), free_head=_int([0]), block_size=BLOCK, num_tokens=31),
    "paged_append": lambda: dict(key=_rand(5, KV_HEADS, DIM), value=_rand(5, KV_HEADS, DIM), k_cache=_cache(),
                                 v_cache=_cache(), slot_mapping=_int([0, 1, 2, 40, 41], torch.int64), k_scale=_scale(),
                                 v_scale=_scale(), key_bounds=_rand(PAGES, KV_HEADS, 2, DIM)),
    "paged_select": lambda: dict(query=_rand(BATCH, HEADS, DIM), key_bounds=_rand(PAGES, KV_HEADS, 2, DIM),
                                 block_table=_table(), context_lens=_int([80, 33]), num_selected=3, block_size=BLOCK,
                                 keep_first=0, keep_last=1),
    "decode_paged_blocks": lambda: dict(q=_rand(BATCH, HEADS, DIM), k_cache=_cache(), v_cache=_cache(),
                                        block_table=_table(), context_lens=_int([80, 33]), k_scale=_scale(),
                                        v_scale=_scale(), block_index=_int([[[0, 2], [1, 2]], [[0, 1], [2, -1]]]),
                                        causal=False, scale=0.125, shares=0, fused_merge=True),
}
BAD = [
    ("paged_allocate", "block_table", lambda t: t.cpu()), ("paged_allocate", "block_table", lambda t: t.long()),
    ("paged_allocate", "block_table", lambda t: t[0]), ("paged_allocate", "block_table", lambda t: t[:, :0]),
    ("paged_allocate", "block_table", lambda t: t[:, :1].expand(-1, TABLE)),
    ("paged_allocate", "context_lens", lambda t: t[:1]), ("paged_allocate", "new_lens", lambda t: t.cpu()),
    ("paged_allocate", "new_lens", lambda t: t.long()), ("paged_allocate", "free_blocks", lambda t: t.view(1, 3)),
    ("paged_allocate", "free_head", lambda t: t.repeat(2)), ("paged_allocate", "block_size", lambda n: 48),
    ("paged_allocate", "block_size", lambda n: 512), ("paged_allocate", "num_tokens", lambda n: -1),
    ("paged_append", "key", lambda t: t.float()), ("paged_append", "key", lambda t: t.cpu()),
    ("paged_append", "key", lambda t: t[:4]), ("paged_append", "value", lambda t: t.bfloat16()),
    ("paged_append", "value", lambda t: t[..., :32]), ("paged_append", "k_cache", lambda t: t[:, :12]),
    ("paged_append", "k_cache", lambda t: t[:4]), ("paged_append", "v_cache", lambda t: t.half()),
    ("paged_append", "v_cache", lambda t: t[:1].expand(PAGES, -1, -1, -1)),
    ("paged_append", "v_cache", lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)),
    ("paged_append", "slot_mapping", lambda t: t.int()), ("paged_append", "slot_mapping", lambda t: t[:4]),
    ("paged_append", "k_scale", lambda t: None), ("paged_append", "k_scale", lambda t: t[:4]),
    ("paged_append", "v_scale", lambda t: t.half()), ("paged_append", "v_scale", lambda t: t[:1].expand(PAGES, -1)),
    ("paged_append", "key_bounds", lambda t: t[:, :, 0]), ("paged_append", "key_bounds", lambda t: t.bfloat16()),
    ("paged_select", "query", lambda t: t.float()), ("paged_select", "query", lambda t: t[:1]),
    ("paged_select", "query", lambda t: t[:, :7]), ("paged_select", "query", lambda t: t[..., :32]),
    ("paged_select", "key_bounds", lambda t: t.cpu()), ("paged_select", "key_bounds", lambda t: t[:, :, :1]),
    ("paged_select", "block_table", lambda t: t.long()), ("paged_select", "block_table", lambda t: t[:, :0]),
    ("paged_select", "context_lens", lambda t: t[:1]), ("paged_select", "num_selected", lambda n: 0),
    ("paged_select", "keep_first", lambda n: 3), ("paged_select", "keep_last", lambda n: -1),
    ("paged_select", "block_size", lambda n: 24),
    ("decode_paged_blocks", "q", lambda t: t.float()), ("decode_paged_blocks", "q", lambda t: t[:, :7]),
    ("decode_paged_blocks", "q", lambda t: t[..., :32]), ("decode_paged_blocks", "q", lambda t: t[0]),
    ("decode_paged_blocks", "k_cache", lambda t: t.bfloat16()), ("decode_paged_blocks", "k_cache", lambda t: t[:4]),
    ("decode_paged_blocks", "v_cache", lambda t: t.cpu()), ("decode_paged_blocks", "block_table", lambda t: t[:1]),
    ("decode_paged_blocks", "block_table", lambda t: t.cpu()),
    ("decode_paged_blocks", "context_lens", lambda t: t.long()),
    ("decode_paged_blocks", "k_scale", lambda t: None), ("decode_paged_blocks", "v_scale", lambda t: t[:, :1]),
    ("decode_paged_blocks", "block_index", lambda t: t[:, :1]), ("decode_paged_blocks", "block_index", lambda t: t.long()),
    ("decode_paged_blocks", "block_index", lambda t: t[..., :0]), ("decode_paged_blocks", "shares", lambda n: 5000),
]


@pytest.mark.parametrize("name", sorted(ARGS))
def test_operators_run_with_what_they_ask_for(name):
    getattr(_native.ops(), name)(**ARGS[name]())
    torch.cuda.synchronize()


@pytest.mark.parametrize("case", range(len(BAD)), ids=[f"{o}-{n}-{i}" for i, (o, n, _) in enumerate(BAD)])
def test_operator_refuses(case):
    name, argument, change = BAD[case]
    args = ARGS[name]()
    before = {n: t.clone() for n, t in args.items() if isinstance(t, torch.Tensor) and n != argument}
    args[argument] = change(args[argument])
    with pytest.raises((RuntimeError, NotImplementedError)):
        getattr(_native.ops(), name)(**args)
    torch.cuda.synchronize()
    for n, t in before.items():
        assert torch.equal(args[n], t), n


def test_two_threads_on_a_stream_each():
    # Each stream has counters of its own for the merge of shares; one thread's calls are of growing sizes.
    def call(rows, args):
        q = args["q"][:, :, None].repeat(1, 1, rows, 1)
        return flash_attention_decode_paged_multi(q, *(args[n] for n in ("k_cache", "v_cache", "block_table",
                                                                         "context_lens")),
                                                  k_scale=args["k_scale"], v_scale=args["v_scale"], num_splits=3)

    args = [ARGS["decode_paged_blocks"]() for _ in range(2)]
    sizes = [range(1, 33), [32] * 32]
    want = [[call(rows, a) for rows in s] for a, s in zip(args, sizes)]
    torch.cuda.synchronize()
    got, failed = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[i] = [call(rows, args[i]) for rows in sizes[i]]
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # (a thread's exception ends the thread only)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_an_index_written_by_another_stream_s_work_is_waited_for_by_its_user():
    # Caches made on one stream and read on another after an event, their
    # memory handed back while the read may still run.
    args = ARGS["decode_paged_blocks"]()
    want = flash_attention_decode_paged(*(args[n] for n in ("q", "k_cache", "v_cache", "block_table", "context_lens")),
                                        k_scale=args["k_scale"], v_scale=args["v_scale"], block_index=args["block_index"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        copies = {n: args[n].clone() for n in ("k_cache", "v_cache", "k_scale", "v_scale", "block_index")}
    torch.cuda.current_stream().wait_stream(side)
    for t in copies.values():
        t.record_stream(torch.cuda.current_stream())
    got = flash_attention_decode_paged(args["q"], copies["k_cache"], copies["v_cache"], args["block_table"],
                                       args["context_lens"], k_scale=copies["k_scale"], v_scale=copies["v_scale"],
                                       block_index=copies["block_index"])
    del copies
    assert torch.equal(got, want)
