"""Input contracts and the platform gate of the public attention API.

Mirrors fa_rdna3/_validation.py of the reference: the same exception classes and the same messages
(callers and tests match on them), with the gfx1100/ROCm gate (fa_rdna3/_validation.py:22-37) replaced
by "a CUDA GPU of compute capability 10.x whose C-ABI library loads".
"""
from functools import lru_cache
import math
from numbers import Integral, Real

import torch

SUPPORTED_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
SUPPORTED_HEAD_DIMS = (16, 32, 64, 128, 256, 512)
LOW_PRECISION_DTYPES = (torch.float16, torch.bfloat16)
_MIN_TORCH_VERSION = (2, 8)
_TORCH_VERSION = tuple(int(part) for part in torch.__version__.split("+", 1)[0].split(".")[:2])


@lru_cache(maxsize=None)
def _device_arch(device_index):
    """(major, minor) compute capability of a CUDA device."""
    return tuple(torch.cuda.get_device_capability(device_index))


_supported_devices = set()   # indices already found able to run the kernels (the answer cannot change)


def unsupported_reason(device=None):
    """None when the kernels can run on `device`, else a one-line reason (fa_rdna3/_validation.py:22-37)."""
    if isinstance(device, torch.device) and device.type == "cuda" and device.index in _supported_devices:
        return None
    if _TORCH_VERSION < _MIN_TORCH_VERSION:
        return "fa-b200 requires PyTorch 2.8 or newer"
    if device is not None:
        device = torch.device(device)
    if torch.version.cuda is None:
        return "fa-b200 requires a CUDA build of PyTorch"
    if not torch.cuda.is_available():
        return "fa-b200 requires an available CUDA GPU"
    if device is not None and device.type != "cuda":
        return f"fa-b200 requires a CUDA GPU tensor, got device {device}"
    index = torch.cuda.current_device() if device is None or device.index is None else device.index
    arch = _device_arch(index)
    if arch[0] != 10:
        return f"fa-b200 supports compute capability 10.x (B200), got {arch[0]}.{arch[1]}"
    _supported_devices.add(index)
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


def _dtype_names(dtypes):
    return ", ".join(str(d).removeprefix("torch.") for d in dtypes)


def validate_dense_inputs(query, key, value, *, allow_gqa=True, dtypes=SUPPORTED_DTYPES):
    """Contracts of (batch, heads, seqlen, head_dim) inputs (fa_rdna3/_validation.py:55-86)."""
    named = (("query", query), ("key", key), ("value", value))
    for name, tensor in named:
        _require_tensor(name, tensor)
        if tensor.dim() != 4:
            raise ValueError(f"{name} must have shape (batch, heads, seqlen, head_dim)")
    if not (query.device == key.device == value.device):
        raise ValueError("query, key and value must be on the same device")
    if query.dtype not in dtypes:
        raise ValueError(f"unsupported dtype {query.dtype}; expected {_dtype_names(dtypes)}")
    if not (query.dtype == key.dtype == value.dtype):
        raise ValueError("query, key and value must have the same dtype")
    qb, qh, qs, qd = query.shape
    kb, kh, ks, kd = key.shape
    vb, vh, vs, vd = value.shape
    if not (qb == kb == vb):
        raise ValueError("query, key and value must have the same batch size")
    if kh != vh:
        raise ValueError("key and value must have the same number of heads")
    if ks != vs:
        raise ValueError("key and value must have the same sequence length")
    if not (qd == kd == vd):
        raise ValueError("query, key and value must have the same head_dim")
    if min(qb, qh, kh, qs, ks, qd) <= 0:
        raise ValueError("batch, heads, sequence lengths and head_dim must be positive")
    if qd > SUPPORTED_HEAD_DIMS[-1]:
        raise ValueError(f"head_dim {qd} exceeds the supported maximum {SUPPORTED_HEAD_DIMS[-1]}")
    if qh != kh:
        if not allow_gqa:
            raise ValueError("different query and key/value head counts require enable_gqa=True")
        if qh % kh != 0:
            raise ValueError("query heads must be a multiple of key/value heads")
    _require_platform(query.device)


def validate_softmax_scale(softmax_scale):
    if softmax_scale is None:
        return
    if isinstance(softmax_scale, bool) or not isinstance(softmax_scale, Real):
        raise TypeError("softmax_scale must be a real number or None")
    if not math.isfinite(float(softmax_scale)):
        raise ValueError("softmax_scale must be finite")


def _is_plain_int(x):
    return isinstance(x, Integral) and not isinstance(x, bool)


def _is_plain_real(x):
    return isinstance(x, Real) and not isinstance(x, bool)


def validate_attention_options(query, key, *, softmax_scale, window_size, softcap, bias,
                               alibi_slopes, dropout_p):
    """Contracts of the score modifiers (fa_rdna3/_validation.py:96-133)."""
    validate_softmax_scale(softmax_scale)
    if not isinstance(window_size, (tuple, list)) or len(window_size) != 2:
        raise ValueError("window_size must contain exactly (left, right)")
    if not all(_is_plain_int(side) and side >= -1 for side in window_size):
        raise ValueError("window_size values must be integers greater than or equal to -1")
    if not _is_plain_real(softcap) or not math.isfinite(float(softcap)):
        raise ValueError("softcap must be a finite nonnegative number")
    if softcap < 0:
        raise ValueError("softcap must be nonnegative")
    if not _is_plain_real(dropout_p) or not 0.0 <= dropout_p < 1.0:
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
            fits = torch.broadcast_shapes(tuple(bias.shape), target) == target
        except RuntimeError:
            fits = False
        if not fits:
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


def validate_varlen_inputs(query, key, value, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k):
    """Contracts of packed (total_tokens, heads, head_dim) inputs (fa_rdna3/_validation.py:141-175)."""
    for name, tensor in (("query", query), ("key", key), ("value", value)):
        _require_tensor(name, tensor)
        if tensor.dim() != 3:
            raise ValueError(f"{name} must have shape (total_tokens, heads, head_dim)")
    if not (query.device == key.device == value.device):
        raise ValueError("query, key and value must be on the same device")
    if query.dtype not in LOW_PRECISION_DTYPES or not (query.dtype == key.dtype == value.dtype):
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
    for name, cu in (("cu_seqlens_q", cu_seqlens_q), ("cu_seqlens_k", cu_seqlens_k)):
        _require_tensor(name, cu)
        if cu.device != query.device or cu.dtype != torch.int32 or not cu.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor on {query.device}")
        if cu.dim() != 1 or cu.numel() < 2:
            raise ValueError(f"{name} must have shape (batch + 1,)")
    if cu_seqlens_q.numel() != cu_seqlens_k.numel():
        raise ValueError("cu_seqlens_q and cu_seqlens_k must describe the same batch size")
    for name, maximum, total in (("max_seqlen_q", max_seqlen_q, query.shape[0]),
                                 ("max_seqlen_k", max_seqlen_k, key.shape[0])):
        if not _is_plain_int(maximum) or not 0 < maximum <= total:
            raise ValueError(f"{name} must be a positive integer no larger than total tokens")
    _require_platform(query.device)


def validate_paged_inputs(query, key, value, block_table, context_lens):
    """Contracts of paged-KV decode inputs (fa_rdna3/_validation.py:178-209)."""
    _require_tensor("query", query)
    _require_tensor("k_cache", key)
    _require_tensor("v_cache", value)
    if query.dim() != 3 or key.dim() != 4 or value.dim() != 4:
        raise ValueError("paged query must be (batch, heads, dim) and caches must be (blocks, block, heads, dim)")
    if key.shape != value.shape:
        raise ValueError("paged key and value caches must have the same shape")
    if not (query.device == key.device == value.device):
        raise ValueError("paged query, key and value must be on the same device")
    if query.dtype not in LOW_PRECISION_DTYPES or not (query.dtype == key.dtype == value.dtype):
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
    for name, meta, ndim in (("block_table", block_table, 2), ("context_lens", context_lens, 1)):
        _require_tensor(name, meta)
        if meta.device != query.device or meta.dtype != torch.int32:
            raise ValueError(f"{name} must be an int32 tensor on {query.device}")
        if meta.dim() != ndim or meta.shape[0] != query.shape[0]:
            raise ValueError(f"{name} has an invalid shape for batch size {query.shape[0]}")
    if block_table.shape[1] <= 0:
        raise ValueError("block_table must contain at least one logical block")
    _require_platform(query.device)


# ---------------------------------------------------------------------------------------------------
# paged 8-bit KV cache
# ---------------------------------------------------------------------------------------------------
CACHE8_DTYPES = (torch.float8_e4m3fn, torch.int8)
CACHE8_HEAD_DIMS = (16, 32, 64, 128, 256)
PLAN_MAX_BATCH = 8192


def _validate_cache8(k_cache, v_cache, k_scales, v_scales):
    """Contracts of the caches (blocks, block, heads, dim) and their scales (blocks, heads)."""
    for name, cache in (("k_cache", k_cache), ("v_cache", v_cache)):
        _require_tensor(name, cache)
        if cache.dim() != 4:
            raise ValueError("8-bit caches must be (blocks, block, heads, dim)")
        if cache.dtype not in CACHE8_DTYPES:
            raise ValueError("8-bit caches must be float8_e4m3fn or int8")
    shape = k_cache.shape
    if shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError("8-bit key and value caches must have the same shape and dtype")
    blocks, block_size, heads, dim = shape
    if min(blocks, block_size, heads, dim) <= 0:
        raise ValueError("8-bit cache blocks, block size, heads and head_dim must be positive")
    if block_size & (block_size - 1):
        raise ValueError("paged cache block size must be a power of two")
    if dim not in CACHE8_HEAD_DIMS:
        raise ValueError(f"head_dim {dim} not supported by 8-bit caches; expected one of {CACHE8_HEAD_DIMS}")
    for name, cache in (("k_cache", k_cache), ("v_cache", v_cache)):
        st = cache.stride()
        # (the library refuses a base address off a 16-byte boundary: a traced tensor has none to look at)
        if st[3] != 1 or any(n > 1 and (s <= 0 or s % 16) for n, s in zip(shape[:3], st[:3])):
            raise ValueError(f"{name} must have unit inner stride, no broadcast dimension and rows aligned to 16 bytes")
    for name, scales in (("k_scales", k_scales), ("v_scales", v_scales)):
        _require_tensor(name, scales)
        if scales.dtype != torch.float32 or scales.shape != (blocks, heads):
            raise ValueError(f"{name} must be float32 of shape (blocks, heads) = ({blocks}, {heads})")
    device = k_cache.device
    if not (v_cache.device == k_scales.device == v_scales.device == device):
        raise ValueError("8-bit caches and scales must be on the same device")


def validate_paged8_inputs(query, k_cache, v_cache, k_scales, v_scales, block_table, context_lens):
    """Contracts of decode over the 8-bit cache."""
    _validate_cache8(k_cache, v_cache, k_scales, v_scales)
    _require_tensor("query", query)
    if query.dim() != 3:
        raise ValueError("paged query must be (batch, heads, dim)")
    if query.dtype not in LOW_PRECISION_DTYPES:
        raise ValueError("paged query must be float16 or bfloat16")
    batch, heads, dim = query.shape
    if min(batch, heads) <= 0:
        raise ValueError("paged batch and heads must be positive")
    if dim != k_cache.shape[3]:
        raise ValueError("paged query and cache head_dim must match")
    if heads % k_cache.shape[2]:
        raise ValueError("query heads must be a multiple of cache heads")
    device = query.device
    if k_cache.device != device:
        raise ValueError("paged query and caches must be on the same device")
    for name, meta, ndim in (("block_table", block_table, 2), ("context_lens", context_lens, 1)):
        _require_tensor(name, meta)
        if meta.device != device or meta.dtype != torch.int32:
            raise ValueError(f"{name} must be an int32 tensor on {device}")
        if meta.dim() != ndim or meta.shape[0] != batch:
            raise ValueError(f"{name} has an invalid shape for batch size {batch}")
    if block_table.shape[1] <= 0:
        raise ValueError("block_table must contain at least one logical block")
    _require_platform(device)


def validate_paged8_append_inputs(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping):
    """Contracts of the rounding of new keys and values into the 8-bit cache."""
    _validate_cache8(k_cache, v_cache, k_scales, v_scales)
    for name, scales in (("k_scales", k_scales), ("v_scales", v_scales)):
        if any(n > 1 and s <= 0 for n, s in zip(scales.shape, scales.stride())):
            raise ValueError(f"{name} must have no broadcast dimension")
    _require_tensor("key", key)
    _require_tensor("value", value)
    if key.dim() != 3 or key.shape != value.shape:
        raise ValueError("key and value must have the same shape (tokens, heads, dim)")
    if key.dtype not in LOW_PRECISION_DTYPES or key.dtype != value.dtype:
        raise ValueError("key and value must share a float16 or bfloat16 dtype")
    if key.shape[1:] != k_cache.shape[2:]:
        raise ValueError("key and cache must have the same heads and head_dim")
    _require_tensor("slot_mapping", slot_mapping)
    device = key.device
    if not (value.device == k_cache.device == device):
        raise ValueError("key, value and caches must be on the same device")
    if slot_mapping.device != device or slot_mapping.dtype != torch.int64:
        raise ValueError(f"slot_mapping must be an int64 tensor on {device}")
    if slot_mapping.shape != (key.shape[0],):
        raise ValueError("slot_mapping must have one entry for each token")
    _require_platform(device)


def validate_paged_plan_inputs(context_lens, new_lens, block_table, free_blocks, free_count, num_tokens, block_size,
                               inplace=False):
    """Contracts of page planning."""
    for name, t, ndim in (("context_lens", context_lens, 1), ("new_lens", new_lens, 1), ("block_table", block_table, 2),
                          ("free_blocks", free_blocks, 1), ("free_count", free_count, 1)):
        _require_tensor(name, t)
        if t.dtype != torch.int32 or t.device != context_lens.device:
            raise ValueError(f"{name} must be an int32 tensor on {context_lens.device}")
        if t.dim() != ndim:
            raise ValueError(f"{name} must have {ndim} dimension{'s' if ndim > 1 else ''}")
    batch = context_lens.shape[0]
    if new_lens.shape[0] != batch or block_table.shape[0] != batch:
        raise ValueError("context_lens, new_lens and block_table must describe the same batch size")
    if not 0 < batch <= PLAN_MAX_BATCH:
        raise ValueError(f"plan takes 1 to {PLAN_MAX_BATCH} requests")
    if block_table.shape[1] <= 0 or free_blocks.shape[0] <= 0:
        raise ValueError("block_table must contain at least one logical block and free_blocks one page")
    if block_table.stride(1) != 1 or (batch > 1 and block_table.stride(0) < block_table.shape[1]):
        raise ValueError("block_table must have unit inner stride and rows that do not overlap")
    if free_blocks.stride(0) != 1:
        raise ValueError("free_blocks must be contiguous")
    if free_count.shape[0] != 1:
        raise ValueError("free_count must have one element")
    if inplace and batch > 1 and context_lens.stride(0) != 1:
        raise ValueError("context_lens must be contiguous to be updated in place")
    if not _is_plain_int(num_tokens) or not 0 <= num_tokens < 2 ** 31:
        raise ValueError("num_tokens must be a nonnegative integer below 2^31")
    if not _is_plain_int(block_size) or block_size <= 0 or block_size & (block_size - 1):
        raise ValueError("paged cache block size must be a power of two")
    if block_table.shape[1] * block_size >= 2 ** 31:
        raise ValueError("block_table must span fewer than 2^31 tokens")
    _require_platform(context_lens.device)
