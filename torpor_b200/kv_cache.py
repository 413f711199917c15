"""Key/value cache operators on device tensors, over the C ABI (``tsw_kv_append``,
``tsw_prefix_attention``).

A served language-model function needs, beside its weights, the keys and values of the tokens it has
read.  They lie in pages; a function's own prompt, which all its requests share, is one more list of
pages, often among the function's parameters, so that a swap-in brings it along with the weights.

* ``kv_append``        -- rotate the new keys and queries by position, write keys and values into pages
* ``prefix_attention`` -- attention of the new tokens over the shared prefix and their sequence's pages

Tensors are torch tensors on one CUDA device; the calls run on that device's current stream, allocate only
what they return (and a workspace, from torch's allocator), and may be captured into a graph.
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


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _int_table(name: str, t: torch.Tensor, dim: int, device) -> None:
    _need(t.dtype is torch.int32 and t.dim() == dim and t.device == device and (t.numel() == 0 or t.stride(-1) == 1),
          f"{name} must be an int32 tensor of {dim} dimension(s) on {device}, contiguous along the last")


def _rows(name: str, t: torch.Tensor, dtype, device) -> None:
    _need(t.dim() == 3 and t.dtype is dtype and t.device == device, f"{name} must be [tokens, heads, head_dim], {dtype}, on {device}")
    _need(t.stride(2) == 1 or t.shape[2] == 1, f"{name}: the elements of a head must be contiguous")


def _pages(p: _cabi.KvPages, k: torch.Tensor, v: torch.Tensor, dtype, device, name: str) -> None:
    _need(k.dim() == 4 and k.shape == v.shape and k.dtype is dtype and v.dtype is dtype and k.device == device and v.device == device,
          f"{name}: keys and values must be [pages, page_size, kv_heads, head_dim], {dtype}, on {device}")
    ks, vs = k.stride(), v.stride()
    _need((ks[3] == 1 and vs[3] == 1) or k.shape[3] == 1, f"{name}: the elements of a head must be contiguous")
    p.k, p.v = k.data_ptr(), v.data_ptr()
    p.k_page_stride, p.k_token_stride, p.k_head_stride = 2 * ks[0], 2 * ks[1], 2 * ks[2]
    p.v_page_stride, p.v_token_stride, p.v_head_stride = 2 * vs[0], 2 * vs[1], 2 * vs[2]
    p.pages, p.page_size = k.shape[0], k.shape[1]


def _batch(b: _cabi.KvBatch, page_table, seq_lens, cu_q, tokens: int, device) -> None:
    _int_table("page_table", page_table, 2, device)
    _int_table("seq_lens", seq_lens, 1, device)
    _int_table("cu_q", cu_q, 1, device)
    n = seq_lens.shape[0]
    _need(cu_q.shape[0] == n + 1 and page_table.shape[0] == n, "page_table, seq_lens and cu_q disagree about the number of sequences")
    b.page_table, b.seq_lens, b.cu_q = page_table.data_ptr(), seq_lens.data_ptr(), cu_q.data_ptr()
    b.batch, b.table_width, b.table_stride, b.tokens = n, page_table.shape[1], page_table.stride(0), tokens


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


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
    device, dtype = k.device, k.dtype
    _need(device.type == "cuda", "kv_append needs CUDA tensors: there is no CPU path")
    _need(dtype in _DTYPES, "keys and values must be float16 or bfloat16")
    a = _cabi.KvAppendArgs()
    _pages(a.cache, k_cache, v_cache, dtype, device, "cache")
    _rows("k", k, dtype, device)
    _rows("v", v, dtype, device)
    _need(k.shape == v.shape and k.shape[1:] == k_cache.shape[2:], "k, v and the cache disagree about heads or head_dim")
    _need(position_offset >= 0, "position_offset must not be negative")
    _batch(a.batch, page_table, seq_lens, cu_q, k.shape[0], device)
    a.k, a.v = k.data_ptr(), v.data_ptr()
    a.k_token_stride, a.k_head_stride = 2 * k.stride(0), 2 * k.stride(1)
    a.v_token_stride, a.v_head_stride = 2 * v.stride(0), 2 * v.stride(1)
    if q is not None:
        _rows("q", q, dtype, device)
        _need(q.shape[0] == k.shape[0] and q.shape[2] == k.shape[2], "q and k disagree about tokens or head_dim")
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=dtype, device=device)
        _rows("q_out", q_out, dtype, device)
        _need(q_out.shape == q.shape, "q_out must have the shape of q")
        a.q, a.q_out, a.q_heads = q.data_ptr(), q_out.data_ptr(), q.shape[1]
        a.q_token_stride, a.q_head_stride = 2 * q.stride(0), 2 * q.stride(1)
        a.q_out_token_stride, a.q_out_head_stride = 2 * q_out.stride(0), 2 * q_out.stride(1)
    else:
        _need(q_out is None, "q_out without q")
    if inv_freq is not None:
        _need(inv_freq.dtype is torch.float64 and inv_freq.dim() == 1 and inv_freq.device == device and inv_freq.is_contiguous(),
              f"inv_freq must be a contiguous float64 vector on {device}")
        a.inv_freq, a.rotary_dim = inv_freq.data_ptr(), 2 * inv_freq.shape[0]
    a.position_offset, a.interleaved = position_offset, 1 if interleaved else 0
    a.dtype, a.kv_heads, a.head_dim = _DTYPES[dtype], k.shape[1], k.shape[2]
    if k.shape[0]:
        check(_cabi.lib().tsw_kv_append(device.index, C.byref(a), _stream(device)))
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
    sequence (queries on an encoder's states, for one).  ``max_q`` is the most new tokens any sequence has (default:
    the number of rows; 1 while generating).  ``scale`` defaults to ``head_dim ** -0.5``.  ``lse`` is the
    natural logarithm of the sum of exponentials, float32 [tokens, q_heads].  Rows that see nothing get zeros
    and -inf; rows that belong to no sequence are left as they were (undefined where the result is made here).
    ``workspace``: a uint8 tensor of at least ``prefix_attention_workspace`` bytes, 256-byte aligned; default: taken from torch's
    allocator for this call."""
    device, dtype = q.device, q.dtype
    _need(device.type == "cuda", "prefix_attention needs CUDA tensors: there is no CPU path")
    _need(dtype in _DTYPES, "queries must be float16 or bfloat16")
    a = _cabi.PrefixAttentionArgs()
    _rows("q", q, dtype, device)
    _pages(a.cache, k_cache, v_cache, dtype, device, "cache")
    tokens, heads, dim = q.shape
    _need(k_cache.shape[3] == dim, "q and the cache disagree about head_dim")
    _batch(a.batch, page_table, seq_lens, cu_q, tokens, device)
    _need(prefix_len >= 0, "prefix_len must not be negative")
    if prefix_len:
        _need(prefix_table is not None, "a prefix needs its prefix_table")
        _int_table("prefix_table", prefix_table, 1, device)
        _need((prefix_k is None) == (prefix_v is None), "prefix_k and prefix_v go together")
        if prefix_k is None:
            a.prefix = a.cache
        else:
            _pages(a.prefix, prefix_k, prefix_v, dtype, device, "prefix")
            _need(prefix_k.shape[2:] == k_cache.shape[2:], "the prefix and the cache disagree about heads or head_dim")
        _need(prefix_table.shape[0] * a.prefix.page_size >= prefix_len, "prefix_table is shorter than prefix_len")
        a.prefix_table, a.prefix_len = prefix_table.data_ptr(), prefix_len
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=dtype, device=device)
    _rows("out", out, dtype, device)
    _need(out.shape == q.shape, "out must have the shape of q")
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=device) if return_lse else None
    a.q, a.out = q.data_ptr(), out.data_ptr()
    a.q_token_stride, a.q_head_stride = 2 * q.stride(0), 2 * q.stride(1)
    a.out_token_stride, a.out_head_stride = 2 * out.stride(0), 2 * out.stride(1)
    a.lse = lse.data_ptr() if lse is not None else 0
    _need(max_q is None or max_q >= 0, "max_q must not be negative")
    a.max_q = tokens if max_q is None else min(max_q, tokens)
    a.dtype, a.q_heads, a.kv_heads, a.head_dim, a.causal = _DTYPES[dtype], heads, k_cache.shape[2], dim, 1 if causal else 0
    a.scale = dim ** -0.5 if scale is None else scale
    if tokens and heads:
        L = _cabi.lib()
        need = C.c_uint64()
        check(L.tsw_prefix_attention_workspace(C.byref(a), C.byref(need)))
        if workspace is None:
            workspace = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
        else:
            _need(workspace.dtype is torch.uint8 and workspace.device == device and workspace.is_contiguous() and
                  workspace.numel() >= need.value, f"workspace must be {need.value} contiguous bytes on {device}")
        if workspace is not None:
            a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
        check(L.tsw_prefix_attention(device.index, C.byref(a), _stream(device)))
    return (out, lse) if return_lse else out


BAD_PAGE, BAD_LENGTH, BAD_ROWS, WAIT_GAVE_UP = 1, 2, 4, 8


def kv_status(device: int = 0, stream: int = 0, clear: bool = False) -> int:
    """What the operators found wrong in device tables since the word was last cleared: a sum of
    ``BAD_PAGE``, ``BAD_LENGTH``, ``BAD_ROWS``, ``WAIT_GAVE_UP``; 0 = nothing.  Synchronises ``stream``.  (``tsw_kv_status``)"""
    word = C.c_uint32()
    check(_cabi.lib().tsw_kv_status(device, stream, C.byref(word), 1 if clear else 0))
    return word.value
