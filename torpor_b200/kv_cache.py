"""Key/value cache operators on device tensors, over the C ABI (``tsw_kv_append``,
``tsw_prefix_attention``).

A served language-model function needs, beside its weights, the keys and values of the tokens it has
read.  They lie in pages; a function's own prompt, which all its requests share, is one more list of
pages, often among the function's parameters, so that a swap-in brings it along with the weights.

* ``kv_append``        -- rotate the new keys and queries by position, write keys and values into pages
* ``prefix_attention`` -- attention of the new tokens over the shared prefix and their sequence's pages

Tensors are torch tensors on one CUDA device; the calls run on that device's current stream, allocate only
what they return (and a workspace, from torch's allocator), and may be captured into a graph.  They serve: there is
no backward pass, and operands that require a gradient are refused while gradients are recorded.
``MemoryManager.kv_append`` and ``MemoryManager.prefix_attention`` are the same on a function's own
client addresses.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _cabi
from ._cabi import check

_DTYPES = {torch.float16: _cabi.F16, torch.bfloat16: _cabi.BF16}


def rope_frequencies(rotary_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """``theta ** (-2 c / rotary_dim)`` for every pair c, in 64 bits: the ``inv_freq`` of ``kv_append``.
    Scaled variants (stretched positions, per-band factors) are this tensor multiplied by the caller."""
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even")
    return float(theta) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / max(rotary_dim, 1))


# The C structures take 32 bits of a size without a word; what does not fit is refused here.
_MAX_TOKENS = 1 << 28
_MAX_KEYS = 0x7fffff00

# The checks cost host time on calls that take a few microseconds on the device: messages are only put together
# when they are raised.

def _int_table(name: str, t: torch.Tensor, dim: int, device) -> None:
    if t.dtype is not torch.int32 or t.dim() != dim or t.device != device or (t.stride(-1) != 1 and t.numel() > 1):
        raise ValueError(f"{name} must be an int32 tensor of {dim} dimension(s) on {device}, contiguous along the last")


def _rows(name: str, t: torch.Tensor, dtype, device):
    """(address, token stride, head stride in bytes, shape) of a [tokens, heads, head_dim] operand."""
    shape = t.shape
    if len(shape) != 3 or t.dtype is not dtype or t.device != device:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], {dtype}, on {device}")
    st = t.stride()
    if st[2] != 1 and shape[2] != 1:
        raise ValueError(f"{name}: the elements of a head must be contiguous")
    if shape[0] > _MAX_TOKENS or shape[1] > 65536 or shape[2] > 512:
        raise ValueError(f"{name}: at most 2^28 tokens, 65536 heads and 512 elements to a head")
    return t.data_ptr(), 2 * st[0], 2 * st[1], shape


def _pages(k: torch.Tensor, v: torch.Tensor, dtype, device, name: str) -> _cabi.KvPages:
    shape = k.shape
    if len(shape) != 4 or shape != v.shape or k.dtype is not dtype or v.dtype is not dtype or k.device != device or v.device != device:
        raise ValueError(f"{name}: keys and values must be [pages, page_size, kv_heads, head_dim], {dtype}, on {device}")
    ks, vs = k.stride(), v.stride()
    if (ks[3] != 1 or vs[3] != 1) and shape[3] != 1:
        raise ValueError(f"{name}: the elements of a head must be contiguous")
    if shape[0] > 0x7fffffff or shape[1] > 1 << 20 or shape[2] > 4096:
        raise ValueError(f"{name}: at most 2^31 - 1 pages of 2^20 tokens and 4096 heads")
    return _cabi.KvPages(k.data_ptr(), v.data_ptr(), 2 * ks[0], 2 * ks[1], 2 * ks[2], 2 * vs[0], 2 * vs[1], 2 * vs[2], shape[0], shape[1])


def _batch(page_table, seq_lens, cu_q, tokens: int, device) -> _cabi.KvBatch:
    _int_table("page_table", page_table, 2, device)
    _int_table("seq_lens", seq_lens, 1, device)
    _int_table("cu_q", cu_q, 1, device)
    n, (rows, width) = seq_lens.shape[0], page_table.shape
    if cu_q.shape[0] != n + 1 or rows != n:
        raise ValueError("page_table, seq_lens and cu_q disagree about the number of sequences")
    if n > 0xffffff or width > 0xffffffff or page_table.stride(0) > 0xffffffff:
        raise ValueError("at most 2^24 - 1 sequences, and 2^32 - 1 entries to a row of page_table")
    return _cabi.KvBatch(page_table.data_ptr(), seq_lens.data_ptr(), cu_q.data_ptr(), n, width, page_table.stride(0), tokens)


_records = torch.is_grad_enabled


def _refuse_gradients(call: str) -> None:
    raise ValueError(f"{call} has no backward pass: call it under torch.no_grad(), or detach what requires a gradient")


def _dtype(t: torch.Tensor, call: str) -> int:
    if t.device.type != "cuda":
        raise ValueError(f"{call} needs CUDA tensors: there is no CPU path")
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{call} takes float16 or bfloat16")
    return code


# torch is told what was written behind its back: a graph that has kept one of these for its backward pass then says so
# instead of using the new values.
_written = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)      # the second wraps the first

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)      # without a Stream object around it


def _stream(device) -> int:
    return _raw_stream(device.index) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def kv_append(k_cache: torch.Tensor, v_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
              seq_lens: torch.Tensor, cu_q: torch.Tensor, *, inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
              position_offset: int = 0, q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write the new tokens' keys and values into the pages of their sequences; returns the rotated
    queries (``q_out``, made here when not given; it may be ``q``), or None without ``q``.

    ``k_cache``, ``v_cache``: [pages, page_size, kv_heads, head_dim], float16 or bfloat16, any strides with contiguous
    heads.  ``k``, ``v``: [tokens, kv_heads, head_dim]; ``q``: [tokens, q_heads, head_dim].  Rows
    ``cu_q[b]`` .. ``cu_q[b + 1] - 1`` are the last tokens of sequence b, which has ``seq_lens[b]`` own tokens with
    them; own token j goes to page ``page_table[b, j // page_size]``.  ``inv_freq`` (float64, one per pair;
    ``rope_frequencies``) rotates the first ``2 * len(inv_freq)`` elements of each key and query head by
    ``(position_offset + j) * inv_freq``; ``interleaved`` pairs elements (2c, 2c + 1) instead of halves."""
    if _records() and (k_cache.requires_grad or v_cache.requires_grad or k.requires_grad or v.requires_grad or (q is not None and q.requires_grad) or
                       (q_out is not None and q_out.requires_grad) or (inv_freq is not None and inv_freq.requires_grad)):
        _refuse_gradients("kv_append")
    code = _dtype(k, "kv_append")
    device, dtype = k.device, k.dtype
    a = _cabi.KvAppendArgs()
    a.cache = _pages(k_cache, v_cache, dtype, device, "cache")
    a.k, a.k_token_stride, a.k_head_stride, shape = _rows("k", k, dtype, device)
    a.v, a.v_token_stride, a.v_head_stride, v_shape = _rows("v", v, dtype, device)
    tokens, heads, dim = shape
    if shape != v_shape or (heads, dim) != tuple(k_cache.shape[2:]):
        raise ValueError("k, v and the cache disagree about heads or head_dim")
    if not 0 <= position_offset < 1 << 32:
        raise ValueError("position_offset must be 0 to 2^32 - 1")
    a.batch = _batch(page_table, seq_lens, cu_q, tokens, device)
    if q is not None:
        a.q, a.q_token_stride, a.q_head_stride, q_shape = _rows("q", q, dtype, device)
        if q_shape[0] != tokens or q_shape[2] != dim:
            raise ValueError("q and k disagree about tokens or head_dim")
        if q_out is None:
            q_out = torch.empty(q_shape, dtype=dtype, device=device)
        a.q_out, a.q_out_token_stride, a.q_out_head_stride, out_shape = _rows("q_out", q_out, dtype, device)
        if out_shape != q_shape:
            raise ValueError("q_out must have the shape of q")
        a.q_heads = q_shape[1]
    elif q_out is not None:
        raise ValueError("q_out without q")
    if inv_freq is not None:
        if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or inv_freq.device != device or not inv_freq.is_contiguous():
            raise ValueError(f"inv_freq must be a contiguous float64 vector on {device}")
        a.inv_freq, a.rotary_dim = inv_freq.data_ptr(), 2 * inv_freq.shape[0]
    a.position_offset, a.interleaved = position_offset, 1 if interleaved else 0
    a.dtype, a.kv_heads, a.head_dim = code, heads, dim
    if tokens:
        check(_cabi.lib().tsw_kv_append(device.index, C.byref(a), _stream(device)))
        _written((k_cache, v_cache) if q_out is None else (k_cache, v_cache, q_out))
    return q_out


def prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                     cu_q: torch.Tensor, *, max_q: Optional[int] = None, prefix_table: Optional[torch.Tensor] = None, prefix_len: int = 0,
                     prefix_k: Optional[torch.Tensor] = None, prefix_v: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                     causal: bool = True, out: Optional[torch.Tensor] = None, return_lse: bool = False,
                     workspace: Optional[torch.Tensor] = None):
    """Attention of ``q`` [tokens, q_heads, head_dim] over a prefix that all sequences share and each
    sequence's own pages; returns ``out``, or ``(out, lse)`` with ``return_lse``.

    The prefix is ``prefix_len`` tokens in the pages ``prefix_table`` (int32) of ``prefix_k`` / ``prefix_v`` (default: the cache
    itself); it is read once for the whole batch.  Rows, tables and cache are those of ``kv_append``.  A
    row sees the prefix and, with ``causal``, the own tokens up to itself; without, all own tokens of its
    sequence (queries on an encoder's states, for one).  ``max_q`` is the most new tokens any sequence has, or more (default:
    the number of rows).  Give it while generating: where the rows of a key head pass 128, a bound of 1 is up to a
    quarter faster than the default (200 sequences behind 2048 tokens 198 for 245 us).  ``scale`` defaults to ``head_dim ** -0.5``.  ``lse`` is the
    natural logarithm of the sum of exponentials, float32 [tokens, q_heads].  Rows that see nothing get zeros
    and -inf; rows that belong to no sequence are left as they were (undefined where the result is made here).
    ``workspace``: a uint8 tensor of at least ``prefix_attention_workspace`` bytes, 256-byte aligned; default: taken from torch's
    allocator for this call."""
    if _records() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad or (prefix_k is not None and prefix_k.requires_grad) or
                       (prefix_v is not None and prefix_v.requires_grad) or (out is not None and out.requires_grad)):
        _refuse_gradients("prefix_attention")
    code = _dtype(q, "prefix_attention")
    device, dtype = q.device, q.dtype
    a = _cabi.PrefixAttentionArgs()
    a.q, a.q_token_stride, a.q_head_stride, shape = _rows("q", q, dtype, device)
    tokens, heads, dim = shape
    a.cache = _pages(k_cache, v_cache, dtype, device, "cache")
    kv_shape = k_cache.shape
    if kv_shape[3] != dim:
        raise ValueError("q and the cache disagree about head_dim")
    a.batch = _batch(page_table, seq_lens, cu_q, tokens, device)
    if not 0 <= prefix_len <= _MAX_KEYS:
        raise ValueError("prefix_len must be 0 to 2^31 - 256")
    if prefix_len:
        if prefix_table is None:
            raise ValueError("a prefix needs its prefix_table")
        _int_table("prefix_table", prefix_table, 1, device)
        if (prefix_k is None) != (prefix_v is None):
            raise ValueError("prefix_k and prefix_v go together")
        if prefix_k is None:
            a.prefix = a.cache
        else:
            a.prefix = _pages(prefix_k, prefix_v, dtype, device, "prefix")
            if prefix_k.shape[2:] != kv_shape[2:]:
                raise ValueError("the prefix and the cache disagree about heads or head_dim")
        if prefix_table.shape[0] * a.prefix.page_size < prefix_len:
            raise ValueError("prefix_table is shorter than prefix_len")
        a.prefix_table, a.prefix_len = prefix_table.data_ptr(), prefix_len
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=device)
    a.out, a.out_token_stride, a.out_head_stride, out_shape = _rows("out", out, dtype, device)
    if out_shape != shape:
        raise ValueError("out must have the shape of q")
    lse = None
    if return_lse:
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=device)
        a.lse = lse.data_ptr()
    if max_q is not None and max_q < 0:
        raise ValueError("max_q must not be negative")
    a.max_q = tokens if max_q is None else min(max_q, tokens)
    a.dtype, a.q_heads, a.kv_heads, a.head_dim, a.causal = code, heads, kv_shape[2], dim, 1 if causal else 0
    a.scale = dim ** -0.5 if scale is None else scale
    if tokens and heads:
        L = _cabi.lib()
        need = C.c_uint64()
        check(L.tsw_prefix_attention_workspace(C.byref(a), C.byref(need)))
        if workspace is None:
            if need.value:
                workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
        elif workspace.dtype is not torch.uint8 or workspace.device != device or not workspace.is_contiguous() or workspace.numel() < need.value:
            raise ValueError(f"workspace must be {need.value} contiguous bytes on {device}")
        if workspace is not None:
            a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
        check(L.tsw_prefix_attention(device.index, C.byref(a), _stream(device)))
        _written((out,))
    return (out, lse) if return_lse else out


BAD_PAGE, BAD_LENGTH, BAD_ROWS, WAIT_GAVE_UP = 1, 2, 4, 8


def kv_status(device: int = 0, stream: int = 0, clear: bool = False) -> int:
    """What the operators found wrong in device tables since the word was last cleared: a sum of
    ``BAD_PAGE``, ``BAD_LENGTH``, ``BAD_ROWS``, ``WAIT_GAVE_UP``; 0 = nothing.  Synchronises ``stream``.  (``tsw_kv_status``)"""
    word = C.c_uint32()
    check(_cabi.lib().tsw_kv_status(device, stream, C.byref(word), 1 if clear else 0))
    return word.value
