"""Inputs of the paged cache tests: tensors on the CPU, and their values in 64 bits."""

import numpy as np
import torch

CACHES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def f64(t):
    """Values of a tensor (codes of an 8-bit one) as float64."""
    return t.detach().cpu().to(torch.float32).double().numpy()


def int32(values):
    return torch.tensor(values, dtype=torch.int32)


def table_of(g, batch, blocks, spare=3):
    """A block table over a shuffled pool, and the pool's size."""
    pool = batch * blocks + spare
    return torch.randperm(pool, generator=g)[:batch * blocks].view(batch, blocks).to(torch.int32), pool


def slots_of(table, contexts, news, block_size):
    """Slots of `news` tokens behind `contexts`, packed sequence after sequence."""
    slots = []
    for b, (ctx, new) in enumerate(zip(contexts, news)):
        slots += [int(table[b, p // block_size]) * block_size + p % block_size for p in range(ctx, ctx + new)]
    return torch.tensor(slots, dtype=torch.int64)


def codes(g, shape, cache, dtype):
    if cache == "int8":
        return torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)
    x = torch.randn(shape, generator=g)
    return (x * 100).clamp(-448, 448).to(torch.float8_e4m3fn) if cache == "e4m3" else x.to(dtype)


def scales(g, pool, heads, cache):
    return torch.exp(0.5 * torch.randn(pool, heads, generator=g)) / {"e4m3": 100.0, "int8": 73.0}[cache]


def same_values(got, want):
    """Equal, NaN where NaN."""
    np.testing.assert_array_equal(f64(got), want)
