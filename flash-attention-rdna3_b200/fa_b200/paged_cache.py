"""A paged KV cache held in 8 bits: page planning, rounding of new keys and values, and decode attention over it.

The reference attends over 16-bit caches that its caller fills (fa_rdna3/interface.py:643-728) and has nothing for the
rest of a server's step; these are the operators around `flash_attention_decode_paged`:

  paged_kv_plan                       pages and slots for the tokens of a step, on the GPU
  paged_kv_append                     new keys and values -> 8-bit codes in their pages
  flash_attention_decode_paged_8bit   one query token for each request against the cache
  PagedKVCache8                       a cache of several layers that runs the three together

Each function first offers its arguments to the compiled binding (csrc/fa_paged8_bind.cpp), which launches at once or
declines; what it declines - refusals, copies, traced tensors - is handled here.

Caches are ``(num_blocks, block_size, kv_heads, head_dim)`` in ``torch.float8_e4m3fn`` or ``torch.int8`` with fp32 scales
``(num_blocks, kv_heads)``: a code c of block p and head h stands for ``c * scales[p, h]``.
"""
import ctypes as C
import functools
import math

import torch

from . import _lib
from ._validation import (
    CACHE8_DTYPES,
    validate_inference_only,
    validate_paged8_append_inputs,
    validate_paged8_inputs,
    validate_paged_plan_inputs,
    validate_softmax_scale,
)
from .interface import _DTYPE_CODE, _status_word, _stream, _vector_friendly

_CACHE_CODE = {torch.float8_e4m3fn: _lib.FA_CACHE_E4M3, torch.int8: _lib.FA_CACHE_INT8}


def _direct(t):
    """True when `t` can go straight to the library: an ordinary tensor, nothing being traced. Everything else takes the
    registered op, which fake tensors and torch.compile see through (and which costs a dispatch of some microseconds)."""
    if type(t) is not torch.Tensor or torch.compiler.is_compiling():
        return False
    try:
        return torch._C._len_torch_dispatch_stack() == 0
    except AttributeError:
        return False


def _rows16(t):
    """`t`, or a copy of it whose rows can be read with 16-byte loads (a tensor that begins off such a boundary may be
    contiguous all the same)."""
    return t if _vector_friendly(t) else t.clone(memory_format=torch.contiguous_format)


def _call(fn, params, device):
    """Launch on torch's current stream of `device`, whichever device is current."""
    if torch.cuda.current_device() == device.index:
        rc = fn(C.byref(params), _stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(C.byref(params), _stream(device))
    if rc:
        _lib.check(rc)


# ---------------------------------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------------------------------
def _plan_impl(context_lens, new_lens, block_table, free_blocks, free_count, num_tokens, block_size, inplace=False):
    lib = _lib.load()
    device, batch = context_lens.device, context_lens.shape[0]
    slots = torch.empty(num_tokens, dtype=torch.int64, device=device)
    cu = torch.empty(batch + 1, dtype=torch.int32, device=device)
    lens_out, count_out = context_lens, free_count
    if not inplace:
        lens_out = torch.empty(batch, dtype=torch.int32, device=device)
        count_out = torch.empty(1, dtype=torch.int32, device=device)
    p = _lib.PagedPlanParams(
        batch, block_table.shape[1], free_blocks.shape[0], block_size, num_tokens,
        context_lens.data_ptr(), context_lens.stride(0), new_lens.data_ptr(), new_lens.stride(0),
        block_table.data_ptr(), block_table.stride(0), free_blocks.data_ptr(), free_count.data_ptr(),
        slots.data_ptr(), cu.data_ptr(), lens_out.data_ptr(), count_out.data_ptr())
    _call(lib.fa_paged_plan, p, device)
    return slots, cu, lens_out, count_out


@torch.library.custom_op("fa_b200::paged_kv_plan", mutates_args=("block_table", "free_blocks"))
def _plan_op(context_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_blocks: torch.Tensor,
             free_count: torch.Tensor, num_tokens: int,
             block_size: int) -> "tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]":
    return _plan_impl(context_lens, new_lens, block_table, free_blocks, free_count, num_tokens, block_size)


@_plan_op.register_fake
def _(context_lens, new_lens, block_table, free_blocks, free_count, num_tokens, block_size):
    batch = context_lens.shape[0]
    return (context_lens.new_empty((num_tokens,), dtype=torch.int64), context_lens.new_empty((batch + 1,)),
            context_lens.new_empty((batch,)), free_count.new_empty((1,)))


def paged_kv_plan(context_lens, new_lens, block_table, free_blocks, free_count, num_tokens, block_size, *,
                  inplace=False):
    """Pages and slots for the tokens of one step, built on the GPU from the requests' lengths.

    ``context_lens`` and ``new_lens`` int32 ``(batch,)``: tokens that request b has in the cache, and tokens that it
    brings (packed one request after the other); a negative ``new_lens[b]`` ends the request. ``block_table`` int32
    ``(batch, max_blocks)`` and the stack of free pages ``free_blocks`` int32 ``(num_blocks,)`` with ``free_count`` int32
    ``(1,)`` are read and updated. ``num_tokens`` is the length of the packed batch (the sum of the new tokens, or more
    where it is padded).

    The pages of ending requests go onto the stack first. Then the requests pop their new pages in order; one whose
    tokens do not fit into its row of the table or into ``num_tokens``, or for which (after those before it that fit) no
    pages are left, is not served: its length and its table stay as they are and its tokens have no slots.

    Returns ``(slot_mapping, cu_seqlens, context_lens, free_count)``: int64 ``(num_tokens,)`` with
    ``page * block_size + offset`` of every token, -1 where it has none; int32 ``(batch + 1,)`` offsets of the requests in
    the packed batch (as ``flash_attention_varlen`` takes them); the lengths after the step (0 for ended requests) and
    the pages then left. The last two are new tensors, or with ``inplace=True`` the given ones, overwritten.
    """
    if not torch.compiler.is_compiling():
        planned = _lib.paged_binding().plan(context_lens, new_lens, block_table, free_blocks, free_count, num_tokens,
                                            block_size, bool(inplace))
        if planned is not None:
            return planned
    validate_paged_plan_inputs(context_lens, new_lens, block_table, free_blocks, free_count, num_tokens, block_size,
                               inplace)
    num_tokens, block_size = int(num_tokens), int(block_size)
    if _direct(context_lens):
        return _plan_impl(context_lens, new_lens, block_table, free_blocks, free_count, num_tokens, block_size, inplace)
    slots, cu, lens, count = _plan_op(context_lens, new_lens, block_table, free_blocks, free_count, num_tokens,
                                      block_size)
    if inplace:
        lens, count = context_lens.copy_(lens), free_count.copy_(count)
    return slots, cu, lens, count


# ---------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------
def _append_impl(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping):
    if key.shape[0] == 0:
        return
    lib = _lib.load()
    device = key.device
    key, value = _rows16(key), _rows16(value)
    p = _lib.Paged8AppendParams(
        _DTYPE_CODE[key.dtype], _CACHE_CODE[k_cache.dtype], key.shape[1], key.shape[2], k_cache.shape[0],
        k_cache.shape[1], key.shape[0], key.data_ptr(), key.stride(), value.data_ptr(), value.stride(),
        k_cache.data_ptr(), k_cache.stride(), v_cache.data_ptr(), v_cache.stride(), k_scales.data_ptr(),
        k_scales.stride(), v_scales.data_ptr(), v_scales.stride(), slot_mapping.data_ptr(), slot_mapping.stride(0),
        _status_word(device).data_ptr())
    _call(lib.fa_paged8_append, p, device)
    _lib.paged_binding().set_status(device.index, p.status)


@torch.library.custom_op("fa_b200::paged_kv_append", mutates_args=("k_cache", "v_cache", "k_scales", "v_scales"))
def _append_op(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
               k_scales: torch.Tensor, v_scales: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    _append_impl(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping)


@_append_op.register_fake
def _(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping):
    return None


def paged_kv_append(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping):
    """Round new keys and values to 8 bits at their slots of a paged cache.

    ``key`` and ``value`` ``(tokens, kv_heads, head_dim)`` float16 or bfloat16; the caches and scales of the module's
    description are updated; ``slot_mapping`` int64 ``(tokens,)`` as `paged_kv_plan` gives it (negative or too large:
    skipped). Scales are powers of two: for each page and head the smallest that the largest finite magnitude among its
    new tokens fits under (448 for e4m3, 127 for int8). A page whose first new token is not its first slot keeps the
    tokens in front of it; its scale never shrinks, and where it grows those tokens are rounded again to the new one.
    Codes are rounded to nearest, ties to even. Infinities become the largest code, NaN stays NaN (in int8: 0).

    The new tokens of a page have to be neighbours in ``slot_mapping`` with slots that rise by one, and a page belongs to
    one request: what a page holds is unspecified otherwise (other pages are as they should be). `check_status` raises
    after a call in which a token's slot is in the page of the one before it but not the next there; tokens of a page that
    lie apart, with other tokens or ones without a slot between them, are not noticed. Inference-only.
    """
    if not torch.compiler.is_compiling() and _lib.paged_binding().append(key, value, k_cache, v_cache, k_scales, v_scales,
                                                                         slot_mapping):
        return
    validate_paged8_append_inputs(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping)
    validate_inference_only(key, value, k_cache, v_cache, k_scales, v_scales)
    if _direct(key):
        _append_impl(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping)
    else:
        _append_op(key, value, k_cache, v_cache, k_scales, v_scales, slot_mapping)


# ---------------------------------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=4096)
def _workspace_bytes(device_index, batch, heads_q, heads_kv, head_dim, block_size):
    p = _lib.Paged8Params(batch=batch, heads_q=heads_q, heads_kv=heads_kv, head_dim=head_dim, block_size=block_size)
    with torch.cuda.device(device_index):
        n = _lib.load().fa_workspace_bytes(_lib.FA_WS_PAGED8, C.byref(p))
    if n < 0:
        _lib.check(n)
    return n


def _decode8_impl(query, k_cache, v_cache, k_scales, v_scales, block_table, context_lens, softmax_scale):
    lib = _lib.load()
    device = query.device
    batch, heads_q, head_dim = query.shape
    blocks, block_size, heads_kv, _ = k_cache.shape
    query = _rows16(query)
    out = torch.empty((batch, heads_q, head_dim), dtype=query.dtype, device=device)
    nbytes = _workspace_bytes(device.index, batch, heads_q, heads_kv, head_dim, block_size)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
    p = _lib.Paged8Params(
        _DTYPE_CODE[query.dtype], _CACHE_CODE[k_cache.dtype], batch, heads_q, heads_kv, head_dim, blocks, block_size,
        block_table.shape[1], query.data_ptr(), query.stride(), k_cache.data_ptr(), k_cache.stride(),
        v_cache.data_ptr(), v_cache.stride(), k_scales.data_ptr(), k_scales.stride(), v_scales.data_ptr(),
        v_scales.stride(), block_table.data_ptr(), block_table.stride(), context_lens.data_ptr(),
        context_lens.stride(0), out.data_ptr(), out.stride(), softmax_scale, workspace.data_ptr(), nbytes,
        _status_word(device).data_ptr())
    _call(lib.fa_decode_paged8, p, device)
    _lib.paged_binding().set_status(device.index, p.status)
    return out


@torch.library.custom_op("fa_b200::decode_paged8", mutates_args=())
def _decode8_op(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scales: torch.Tensor,
                v_scales: torch.Tensor, block_table: torch.Tensor, context_lens: torch.Tensor,
                softmax_scale: float) -> torch.Tensor:
    return _decode8_impl(query, k_cache, v_cache, k_scales, v_scales, block_table, context_lens, softmax_scale)


@_decode8_op.register_fake
def _(query, k_cache, v_cache, k_scales, v_scales, block_table, context_lens, softmax_scale):
    return query.new_empty(query.shape)


def flash_attention_decode_paged_8bit(query, k_cache, v_cache, k_scales, v_scales, block_table, context_lens,
                                      softmax_scale=None):
    """Decode attention over a paged KV cache held in 8 bits: `flash_attention_decode_paged` for the caches that
    `paged_kv_append` fills.

    query ``(batch, q_heads, head_dim)`` float16 or bfloat16 (head_dim 16, 32, 64, 128 or 256); caches and scales as in
    the module's description, any finite fp32 scales; ``block_table`` int32 ``(batch, max_blocks_per_seq)``; ``context_lens``
    int32 ``(batch,)``, clamped to the table. Pages out of range contribute nothing and an empty context gives zeros.
    Products and sums are fp32 over fp16 operands. Keys and values are exact in fp16; probability times value scale is
    rounded to it, off by 2^-11 of itself or by 2^-35 of its row's largest, whichever is more; bf16 queries are exact
    down to 2^-31 of the row's largest value, and off by at most 2^-39 of that below. Values (code times scale) up to 2^117
    leave no sum's range. Non-causal, inference-only.
    """
    if not torch.compiler.is_compiling():
        out = _lib.paged_binding().decode(query, k_cache, v_cache, k_scales, v_scales, block_table, context_lens,
                                          softmax_scale)
        if out is not None:
            return out
    validate_paged8_inputs(query, k_cache, v_cache, k_scales, v_scales, block_table, context_lens)
    validate_inference_only(query, k_cache, v_cache, k_scales, v_scales)
    validate_softmax_scale(softmax_scale)
    softmax_scale = 1.0 / math.sqrt(query.shape[2]) if softmax_scale is None else float(softmax_scale)
    impl = _decode8_impl if _direct(query) else _decode8_op
    return impl(query, k_cache, v_cache, k_scales, v_scales, block_table, context_lens, softmax_scale)


# ---------------------------------------------------------------------------------------------------
# the three together
# ---------------------------------------------------------------------------------------------------
class PagedKVCache8:
    """A pool of 8-bit pages for `layers` layers and up to `max_batch` requests, with its block table on the GPU.

    A step is ``slots, cu = cache.plan(new_lens, num_tokens)``, then in every layer ``cache.append(layer, key, value,
    slots)`` and ``cache.decode(layer, query)``. Nothing reads back to the host, so a step can be captured in a CUDA graph.
    Row b of every tensor is request b; a row without a request has length 0 and gets 0 new tokens.
    """

    def __init__(self, layers, num_blocks, block_size, kv_heads, head_dim, max_batch, max_blocks, *,
                 dtype=torch.float8_e4m3fn, device="cuda"):
        sizes = {"layers": layers, "num_blocks": num_blocks, "block_size": block_size, "kv_heads": kv_heads,
                 "head_dim": head_dim, "max_batch": max_batch, "max_blocks": max_blocks}
        for name, n in sizes.items():
            if isinstance(n, bool) or not isinstance(n, int) or n <= 0:
                raise ValueError(f"{name} must be a positive integer")
        if dtype not in CACHE8_DTYPES:
            raise ValueError("dtype must be torch.float8_e4m3fn or torch.int8")
        self.block_size = block_size
        shape = (layers, num_blocks, block_size, kv_heads, head_dim)
        self.k_cache = torch.zeros(shape, dtype=torch.int8, device=device).view(dtype)
        self.v_cache = torch.zeros(shape, dtype=torch.int8, device=device).view(dtype)
        self.k_scales = torch.ones((layers, num_blocks, kv_heads), dtype=torch.float32, device=device)
        self.v_scales = torch.ones((layers, num_blocks, kv_heads), dtype=torch.float32, device=device)
        self._layers = list(zip(self.k_cache.unbind(), self.v_cache.unbind(), self.k_scales.unbind(),
                                self.v_scales.unbind()))
        self.block_table = torch.full((max_batch, max_blocks), -1, dtype=torch.int32, device=device)
        self.context_lens = torch.zeros(max_batch, dtype=torch.int32, device=device)
        self.free_blocks = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), num_blocks, dtype=torch.int32, device=device)

    def plan(self, new_lens, num_tokens):
        """`paged_kv_plan` for ``new_lens`` int32 ``(max_batch,)``; returns ``(slot_mapping, cu_seqlens)``."""
        slots, cu, _, _ = paged_kv_plan(self.context_lens, new_lens, self.block_table, self.free_blocks,
                                        self.free_count, num_tokens, self.block_size, inplace=True)
        return slots, cu

    def append(self, layer, key, value, slot_mapping):
        """`paged_kv_append` into one layer."""
        paged_kv_append(key, value, *self._layers[layer], slot_mapping)

    def decode(self, layer, query, softmax_scale=None):
        """`flash_attention_decode_paged_8bit` of ``query`` ``(max_batch, q_heads, head_dim)`` against one layer."""
        return flash_attention_decode_paged_8bit(query, *self._layers[layer], self.block_table, self.context_lens,
                                                 softmax_scale)
