"""Input contracts and platform detection for the public attention APIs.

Same contracts and error messages as the reference
(fa_rdna3/_validation.py:9-209); the platform gate accepts gfx950 (MI355X)
instead of gfx1100.  Every check runs on the host before any kernel launch.
"""

from functools import lru_cache
import math
from numbers import Integral, Real

import torch

SUPPORTED_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
SUPPORTED_HEAD_DIMS = (16, 32, 64, 128, 256, 512)
LOW_PRECISION_DTYPES = (torch.float16, torch.bfloat16)
SUPPORTED_ARCH = "gfx950"
_MIN_TORCH_VERSION = (2, 8)
_TORCH_VERSION = tuple(int(part) for part in torch.__version__.split("+", 1)[0].split(".")[:2])


@lru_cache(maxsize=None)
def _device_arch(device_index):
    properties = torch.cuda.get_device_properties(device_index)
    return getattr(properties, "gcnArchName", "").split(":", 1)[0]


def unsupported_reason(device=None):
    """Why the MI355X kernels cannot run on ``device``; None when they can."""
    if _TORCH_VERSION < _MIN_TORCH_VERSION:
        return "fa-rdna3 requires PyTorch 2.8 or newer"
    if device is not None:
        device = torch.device(device)
    if torch.version.hip is None:
        return "fa-rdna3 requires a ROCm build of PyTorch"
    if not torch.cuda.is_available():
        return "fa-rdna3 requires an available ROCm GPU"
    if device is not None and device.type != "cuda":
        return f"fa-rdna3 requires a ROCm GPU tensor, got device {device}"
    index = torch.cuda.current_device() if device is None or device.index is None else device.index
    arch = _device_arch(index)
    if arch != SUPPORTED_ARCH:
        return f"fa-rdna3 supports {SUPPORTED_ARCH}, got {arch or 'an unknown GPU architecture'}"
    return None


def is_available(device=None):
    return unsupported_reason(device) is None


def _require_platform(device):
    reason = unsupported_reason(device)
    if reason is not None:
        raise RuntimeError(reason)


def _require_tensor(name, tensor):
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")


def validate_dense_inputs(query, key, value, *, allow_gqa=True, dtypes=SUPPORTED_DTYPES):
    for name, tensor in (("query", query), ("key", key), ("value", value)):
        _require_tensor(name, tensor)
        if tensor.dim() != 4:
            raise ValueError(f"{name} must have shape (batch, heads, seqlen, head_dim)")
    if query.device != key.device or query.device != value.device:
        raise ValueError("query, key and value must be on the same device")
    if query.dtype not in dtypes:
        names = ", ".join(str(d).removeprefix("torch.") for d in dtypes)
        raise ValueError(f"unsupported dtype {query.dtype}; expected {names}")
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise ValueError("query, key and value must have the same dtype")
    if query.shape[0] != key.shape[0] or query.shape[0] != value.shape[0]:
        raise ValueError("query, key and value must have the same batch size")
    if key.shape[1] != value.shape[1]:
        raise ValueError("key and value must have the same number of heads")
    if key.shape[2] != value.shape[2]:
        raise ValueError("key and value must have the same sequence length")
    if query.shape[3] != key.shape[3] or query.shape[3] != value.shape[3]:
        raise ValueError("query, key and value must have the same head_dim")
    if min(query.shape[0], query.shape[1], key.shape[1], query.shape[2], key.shape[2], query.shape[3]) <= 0:
        raise ValueError("batch, heads, sequence lengths and head_dim must be positive")
    if query.shape[3] > SUPPORTED_HEAD_DIMS[-1]:
        raise ValueError(f"head_dim {query.shape[3]} exceeds the supported maximum {SUPPORTED_HEAD_DIMS[-1]}")
    if query.shape[1] != key.shape[1]:
        if not allow_gqa:
            raise ValueError("different query and key/value head counts require enable_gqa=True")
        if query.shape[1] % key.shape[1] != 0:
            raise ValueError("query heads must be a multiple of key/value heads")
    _require_platform(query.device)


def validate_softmax_scale(softmax_scale):
    if softmax_scale is None:
        return
    if isinstance(softmax_scale, bool) or not isinstance(softmax_scale, Real):
        raise TypeError("softmax_scale must be a real number or None")
    if not math.isfinite(float(softmax_scale)):
        raise ValueError("softmax_scale must be finite")


def validate_attention_options(query, key, *, softmax_scale, window_size, softcap, bias,
                               alibi_slopes, dropout_p):
    validate_softmax_scale(softmax_scale)
    if not isinstance(window_size, (tuple, list)) or len(window_size) != 2:
        raise ValueError("window_size must contain exactly (left, right)")
    if any(isinstance(s, bool) or not isinstance(s, Integral) or s < -1 for s in window_size):
        raise ValueError("window_size values must be integers greater than or equal to -1")
    if isinstance(softcap, bool) or not isinstance(softcap, Real) or not math.isfinite(float(softcap)):
        raise ValueError("softcap must be a finite nonnegative number")
    if softcap < 0:
        raise ValueError("softcap must be nonnegative")
    if isinstance(dropout_p, bool) or not isinstance(dropout_p, Real) or not 0.0 <= dropout_p < 1.0:
        raise ValueError("dropout_p must satisfy 0 <= dropout_p < 1")
    batch, heads, seqlen_q = query.shape[:3]
    if bias is not None:
        _require_tensor("bias", bias)
        if bias.device != query.device:
            raise ValueError("bias must be on the same device as query")
        if bias.dtype not in (query.dtype, torch.float32):
            raise ValueError("bias dtype must match query dtype or be float32")
        if bias.requires_grad:
            raise ValueError("bias gradients are not supported")
        target = (batch, heads, seqlen_q, key.shape[2])
        try:
            broadcast = torch.broadcast_shapes(tuple(bias.shape), target)
        except RuntimeError:
            broadcast = None
        if broadcast != target:
            raise ValueError("bias must be broadcastable to (batch, heads, seqlen_q, seqlen_k)")
    if alibi_slopes is not None:
        _require_tensor("alibi_slopes", alibi_slopes)
        if alibi_slopes.device != query.device:
            raise ValueError("alibi_slopes must be on the same device as query")
        if not alibi_slopes.dtype.is_floating_point:
            raise ValueError("alibi_slopes must have a floating-point dtype")
        if alibi_slopes.requires_grad:
            raise ValueError("ALiBi slope gradients are not supported")
        if alibi_slopes.shape != (heads,):
            raise ValueError(f"alibi_slopes must have shape ({heads},)")


def validate_inference_only(*tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("this decode API is inference-only and does not support autograd")


def validate_varlen_inputs(query, key, value, cu_seqlens_q, cu_seqlens_k,
                           max_seqlen_q, max_seqlen_k):
    for name, tensor in (("query", query), ("key", key), ("value", value)):
        _require_tensor(name, tensor)
        if tensor.dim() != 3:
            raise ValueError(f"{name} must have shape (total_tokens, heads, head_dim)")
    if query.device != key.device or query.device != value.device:
        raise ValueError("query, key and value must be on the same device")
    if query.dtype not in LOW_PRECISION_DTYPES or key.dtype != query.dtype or value.dtype != query.dtype:
        raise ValueError("varlen query, key and value must share a float16 or bfloat16 dtype")
    if key.shape != value.shape:
        raise ValueError("varlen key and value must have the same shape")
    if query.shape[2] != key.shape[2]:
        raise ValueError("varlen query, key and value must have the same head_dim")
    if min(query.shape[0], key.shape[0], query.shape[1], key.shape[1], query.shape[2]) <= 0:
        raise ValueError("total tokens, heads and head_dim must be positive")
    if query.shape[1] % key.shape[1] != 0:
        raise ValueError("query heads must be a multiple of key/value heads")
    if query.shape[2] not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"head_dim {query.shape[2]} is not supported by varlen attention")
    for name, cumulative in (("cu_seqlens_q", cu_seqlens_q), ("cu_seqlens_k", cu_seqlens_k)):
        _require_tensor(name, cumulative)
        if cumulative.device != query.device or cumulative.dtype != torch.int32 or not cumulative.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor on {query.device}")
        if cumulative.dim() != 1 or cumulative.numel() < 2:
            raise ValueError(f"{name} must have shape (batch + 1,)")
    if cu_seqlens_q.numel() != cu_seqlens_k.numel():
        raise ValueError("cu_seqlens_q and cu_seqlens_k must describe the same batch size")
    for name, maximum, total in (("max_seqlen_q", max_seqlen_q, query.shape[0]),
                                 ("max_seqlen_k", max_seqlen_k, key.shape[0])):
        if isinstance(maximum, bool) or not isinstance(maximum, Integral) or not 0 < maximum <= total:
            raise ValueError(f"{name} must be a positive integer no larger than total tokens")
    _require_platform(query.device)


def validate_paged_inputs(query, key, value, block_table, context_lens):
    _require_tensor("query", query)
    _require_tensor("k_cache", key)
    _require_tensor("v_cache", value)
    if query.dim() != 3 or key.dim() != 4 or value.dim() != 4:
        raise ValueError("paged query must be (batch, heads, dim) and caches must be (blocks, block, heads, dim)")
    if key.shape != value.shape:
        raise ValueError("paged key and value caches must have the same shape")
    if query.device != key.device or query.device != value.device:
        raise ValueError("paged query, key and value must be on the same device")
    if query.dtype not in LOW_PRECISION_DTYPES or key.dtype != query.dtype or value.dtype != query.dtype:
        raise ValueError("paged query, key and value must share a float16 or bfloat16 dtype")
    if query.shape[2] != key.shape[3] or query.shape[2] not in SUPPORTED_HEAD_DIMS:
        raise ValueError("paged query and cache head_dim must match a supported head dimension")
    if min(query.shape[0], query.shape[1], query.shape[2], key.shape[0], key.shape[1], key.shape[2]) <= 0:
        raise ValueError("paged batch, heads, blocks, block size and head_dim must be positive")
    if query.shape[1] % key.shape[2] != 0:
        raise ValueError("query heads must be a multiple of cache heads")
    block_size = key.shape[1]
    if block_size & (block_size - 1):
        raise ValueError("paged cache block size must be a power of two")
    for name, metadata, expected_shape in (
        ("block_table", block_table, (query.shape[0], None)),
        ("context_lens", context_lens, (query.shape[0],)),
    ):
        _require_tensor(name, metadata)
        if metadata.device != query.device or metadata.dtype != torch.int32:
            raise ValueError(f"{name} must be an int32 tensor on {query.device}")
        if metadata.dim() != len(expected_shape) or metadata.shape[0] != expected_shape[0]:
            raise ValueError(f"{name} has an invalid shape for batch size {query.shape[0]}")
    if block_table.shape[1] <= 0:
        raise ValueError("block_table must contain at least one logical block")
    _require_platform(query.device)


# ---------------------------------------------------------------------------
# Filling a paged cache and choosing its blocks (paged.py)
# ---------------------------------------------------------------------------

EIGHT_BIT_DTYPES = (torch.float8_e4m3fn, torch.int8)
EIGHT_BIT_HEAD_DIMS = (32, 64, 128, 256, 512)


def validate_count(name, value, least):
    """A 32-bit whole number of at least `least`."""
    if isinstance(value, bool) or not isinstance(value, Integral) or not least <= value < 2 ** 31:
        raise ValueError(f"{name} must be an integer of at least {least}")


def validate_block_size(block_size):
    """Tokens of a paged cache's block."""
    validate_count("block_size", block_size, 1)
    if block_size > 256 or block_size & (block_size - 1):
        raise ValueError("paged cache block size must be a power of two up to 256")


def _require_like(name, tensor, dtype, shape, device):
    """A tensor of this dtype, shape (None: any extent) and device."""
    _require_tensor(name, tensor)
    if (tensor.device != device or tensor.dtype != dtype or tensor.dim() != len(shape)
            or any(want is not None and got != want for got, want in zip(tensor.shape, shape))):
        want = ", ".join("n" if n is None else str(n) for n in shape)
        raise ValueError(f"{name} must be a {str(dtype).removeprefix('torch.')} tensor of shape ({want}) on {device}")


def _require_writable(name, tensor, rows=False):
    """A tensor that a kernel can write in place: no element twice and, for
    `rows`, 16-byte pieces."""
    if any(n > 1 and st == 0 for n, st in zip(tensor.shape, tensor.stride())):
        raise ValueError(f"{name} is written in place and must not be expanded")
    esize = tensor.element_size()
    if rows and (tensor.stride(-1) != 1 or tensor.data_ptr() % 16
                 or any(n > 1 and (st * esize) % 16 for st, n in zip(tensor.stride()[:-1], tensor.shape[:-1]))):
        raise ValueError(f"{name} must have a unit last stride and 16-byte aligned rows to be updated in place")


def validate_allocate_inputs(block_table, context_lens, new_lens, free_blocks, free_head):
    _require_tensor("block_table", block_table)
    device = block_table.device
    _require_like("block_table", block_table, torch.int32, (None, None), device)
    batch, blocks = block_table.shape
    if batch <= 0 or blocks <= 0:
        raise ValueError("block_table must have at least one sequence and one block")
    _require_like("context_lens", context_lens, torch.int32, (batch,), device)
    _require_like("new_lens", new_lens, torch.int32, (batch,), device)
    _require_like("free_blocks", free_blocks, torch.int32, (None,), device)
    if free_head is not None:
        _require_like("free_head", free_head, torch.int32, (1,), device)
    _require_writable("block_table", block_table)
    _require_platform(device)


def validate_append_inputs(key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale, key_bounds):
    _require_tensor("key", key)
    device = key.device
    if key.dim() != 3 or key.dtype not in LOW_PRECISION_DTYPES:
        raise ValueError("key must be a float16 or bfloat16 tensor of shape (tokens, kv_heads, head_dim)")
    tokens, heads, dim = key.shape
    _require_like("value", value, key.dtype, (tokens, heads, dim), device)
    _require_tensor("k_cache", k_cache)
    if k_cache.dtype != key.dtype and k_cache.dtype not in EIGHT_BIT_DTYPES:
        raise ValueError("caches must have key's dtype, float8_e4m3fn or int8")
    _require_like("k_cache", k_cache, k_cache.dtype, (None, None, heads, dim), device)
    _require_like("v_cache", v_cache, k_cache.dtype, k_cache.shape, device)
    if min(heads, dim, k_cache.shape[0]) <= 0:
        raise ValueError("kv_heads, head_dim and blocks must be positive")
    validate_block_size(k_cache.shape[1])
    eight = k_cache.dtype in EIGHT_BIT_DTYPES
    if dim not in (EIGHT_BIT_HEAD_DIMS if eight else SUPPORTED_HEAD_DIMS):
        raise ValueError(f"head_dim {dim} is not supported by a paged cache of {str(k_cache.dtype).removeprefix('torch.')}")
    _require_like("slot_mapping", slot_mapping, torch.int64, (tokens,), device)
    for name, scale in (("k_scale", k_scale), ("v_scale", v_scale)):
        if eight:
            _require_like(name, scale, torch.float32, (k_cache.shape[0], heads), device)
            _require_writable(name, scale)
        elif scale is not None:
            raise ValueError("k_scale and v_scale apply to float8_e4m3fn and int8 caches only")
    _require_writable("k_cache", k_cache, rows=True)
    _require_writable("v_cache", v_cache, rows=True)
    if key_bounds is not None:
        _require_like("key_bounds", key_bounds, key.dtype, (k_cache.shape[0], heads, 2, dim), device)
        _require_writable("key_bounds", key_bounds, rows=True)
    _require_platform(device)


def validate_select_inputs(query, key_bounds, block_table, context_lens):
    _require_tensor("query", query)
    device = query.device
    if query.dim() not in (3, 4) or query.dtype not in LOW_PRECISION_DTYPES:
        raise ValueError("query must be a float16 or bfloat16 tensor (batch, q_heads[, rows], head_dim)")
    batch, heads, dim = query.shape[0], query.shape[1], query.shape[-1]
    _require_like("key_bounds", key_bounds, query.dtype, (None, None, 2, dim), device)
    if min(query.shape) <= 0 or min(key_bounds.shape) <= 0:
        raise ValueError("batch, heads, rows, blocks and head_dim must be positive")
    if dim not in EIGHT_BIT_HEAD_DIMS:
        raise ValueError(f"head_dim {dim} is not supported by block selection")
    if heads % key_bounds.shape[1]:
        raise ValueError("query heads must be a multiple of cache heads")
    _require_like("block_table", block_table, torch.int32, (batch, None), device)
    if block_table.shape[1] <= 0:
        raise ValueError("block_table must contain at least one logical block")
    _require_like("context_lens", context_lens, torch.int32, (batch,), device)
    _require_platform(device)


def validate_paged_blocks_inputs(query, k_cache, v_cache, block_table, context_lens, k_scale, v_scale, block_index):
    """Contracts of the paged decode over block scales and a block index, for
    a 4-D query: the paged shape rules, checked on stand-ins of the query's
    type, and the rules of scales and index."""
    if query.dtype not in LOW_PRECISION_DTYPES:
        raise ValueError("query must be float16 or bfloat16")
    _require_tensor("k_cache", k_cache)
    _require_tensor("v_cache", v_cache)
    eight = k_cache.dtype in EIGHT_BIT_DTYPES
    if k_cache.dtype != v_cache.dtype or not (eight or k_cache.dtype == query.dtype):
        raise ValueError("k_cache and v_cache must share a dtype: the query's, float8_e4m3fn or int8")
    stand_in = lambda t: torch.empty_strided(t.shape, [0] * t.dim(), dtype=query.dtype, device=t.device)  # noqa: E731
    if query.shape[-1] not in EIGHT_BIT_HEAD_DIMS:
        raise ValueError("block scales and block_index need head_dim 32, 64, 128, 256 or 512")
    if k_cache.dim() == 4:
        validate_block_size(k_cache.shape[1])
        if eight:
            for name, scale in (("k_scale", k_scale), ("v_scale", v_scale)):
                _require_like(name, scale, torch.float32, (k_cache.shape[0], k_cache.shape[2]), query.device)
        elif k_scale is not None or v_scale is not None:
            raise ValueError("k_scale and v_scale apply to float8_e4m3fn and int8 caches only")
        if block_index is not None:
            _require_like("block_index", block_index, torch.int32, (query.shape[0], k_cache.shape[2], None), query.device)
            if block_index.shape[2] <= 0:
                raise ValueError("block_index must list at least one block")
    validate_paged_inputs(query.select(2, 0), stand_in(k_cache), stand_in(v_cache), block_table, context_lens)
