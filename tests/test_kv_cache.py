"""Key/value cache operators without a GPU: layouts, refusals, and what a plan-only engine answers."""
import ctypes as C
import os
import re

import pytest
import torch

from torpor_b200 import _cabi
from torpor_b200.memory_manager import MemoryManager, repo_reset

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def fields(name):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "torpor_swap.h")).read(), flags=re.S)
    body = re.search(r"typedef\s+struct\s*\{([^}]*)\}\s*" + name + r"\s*;", text).group(1)
    out = []
    for decl in body.split(";"):
        decl = " ".join(decl.split())
        if decl:
            ctype, names = decl.split(" ", 1)
            out += [(n.strip(), ctype) for n in names.split(",")]
    return out


@pytest.mark.parametrize("c_name,binding", [("tsw_kv_pages", "KvPages"), ("tsw_kv_batch", "KvBatch"),
                                            ("tsw_kv_append_args", "KvAppendArgs"), ("tsw_prefix_attention_args", "PrefixAttentionArgs")])
def test_layouts_of_header_and_binding_agree(c_name, binding):
    width = {"uint32_t": 4, "uint64_t": 8, "float": 4, "tsw_kv_pages": C.sizeof(_cabi.KvPages), "tsw_kv_batch": C.sizeof(_cabi.KvBatch)}
    cls = getattr(_cabi, binding)
    have = fields(c_name)
    assert [n for n, _ in have] == [f[0] for f in cls._fields_]
    for (name, ctype), bound in zip(have, cls._fields_):
        assert width[ctype] == C.sizeof(bound[1]), name


def pages(n=8, ps=16, heads=2, dim=64):
    row = 2 * dim
    return _cabi.KvPages(1 << 40, 1 << 41, ps * heads * row, heads * row, row, ps * heads * row, heads * row, row, n, ps)


def batch(tokens=4, n=2, width=4):
    return _cabi.KvBatch(4096, 8192, 12288, n, width, width, tokens)


def append_args(**kw):
    a = _cabi.KvAppendArgs()
    a.cache, a.batch = pages(), batch()
    a.q, a.q_out, a.k, a.v = 1 << 42, 1 << 43, 1 << 44, 1 << 45
    for f in ("q", "q_out"):
        setattr(a, f + "_token_stride", 512)
        setattr(a, f + "_head_stride", 128)
    for f in ("k", "v"):
        setattr(a, f + "_token_stride", 256)
        setattr(a, f + "_head_stride", 128)
    a.inv_freq, a.rotary_dim, a.q_heads, a.kv_heads, a.head_dim = 1 << 46, 64, 4, 2, 64
    return change(a, kw)


def attention_args(**kw):
    a = _cabi.PrefixAttentionArgs()
    a.cache, a.prefix, a.batch = pages(), pages(), batch()
    a.prefix_table, a.prefix_len, a.max_q = 1 << 20, 20, 2
    a.q, a.out, a.q_token_stride, a.q_head_stride, a.out_token_stride, a.out_head_stride = 1 << 42, 1 << 43, 512, 128, 512, 128
    a.q_heads, a.kv_heads, a.head_dim, a.causal, a.scale = 4, 2, 64, 1, 0.125
    need = C.c_uint64()
    if _cabi.lib().tsw_prefix_attention_workspace(C.byref(a), C.byref(need)) == 0:
        a.workspace, a.workspace_bytes = 1 << 47, need.value
    return change(a, kw)


def change(a, kw):
    for k, v in kw.items():
        obj, names = a, k.split("__")
        for n in names[:-1]:
            obj = getattr(obj, n)
        setattr(obj, names[-1], v)
    return a


APPEND_REFUSED = [
    dict(dtype=2), dict(head_dim=0), dict(head_dim=63), dict(head_dim=514), dict(rotary_dim=66), dict(rotary_dim=3),
    dict(inv_freq=0), dict(inv_freq=(1 << 46) + 4), dict(kv_heads=0), dict(kv_heads=5000), dict(q_heads=70000), dict(q=0), dict(q_out=0),
    dict(k=0), dict(v=0), dict(k=1), dict(q_head_stride=127), dict(q_out_head_stride=64), dict(q_out_token_stride=0),
    dict(position_offset=1 << 32), dict(k_token_stride=1 << 41), dict(cache__page_size=0), dict(cache__page_size=1 << 21), dict(cache__k=0),
    dict(cache__k_head_stride=0), dict(cache__v_token_stride=64), dict(cache__k_page_stride=2), dict(cache__v=(1 << 41) + 1),
    dict(batch__seq_lens=0), dict(batch__cu_q=0), dict(batch__page_table=0), dict(batch__table_stride=3), dict(batch__page_table=4098),
    dict(batch__tokens=1 << 31), dict(batch__tokens=(1 << 28) + 1), dict(batch__batch=1 << 24), dict(q_out=1 << 42, q_out_head_stride=256, q_out_token_stride=1024),
]
ATTENTION_REFUSED = [
    dict(dtype=2), dict(head_dim=0), dict(head_dim=513), dict(q_heads=0), dict(q_heads=5), dict(kv_heads=0), dict(q=0), dict(out=0),
    dict(out_head_stride=64), dict(out_token_stride=0), dict(out=(1 << 43) + 1), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(prefix_table=0), dict(prefix_table=2), dict(prefix_len=0x7fffff01), dict(prefix__k=0), dict(prefix__page_size=0), dict(lse=2),
    dict(max_q=1 << 31), dict(out=1 << 42), dict(batch__tokens=(1 << 28) + 1), dict(batch__tokens=1 << 28, q_heads=64), dict(cache__v=0), dict(cache__k_page_stride=1 << 41), dict(batch__cu_q=0), dict(batch__table_stride=2),
]


@pytest.mark.parametrize("wrong", APPEND_REFUSED, ids=lambda w: "-".join(f"{k}={v}" for k, v in w.items()))
def test_append_refuses(built, wrong):
    L = _cabi.lib()
    assert L.tsw_kv_append(0, C.byref(append_args(**wrong)), None) == _cabi.ERR_INVALID
    assert L.tsw_last_error()


@pytest.mark.parametrize("wrong", ATTENTION_REFUSED, ids=lambda w: "-".join(f"{k}={v}" for k, v in w.items()))
def test_attention_refuses(built, wrong):
    L = _cabi.lib()
    assert L.tsw_prefix_attention(0, C.byref(attention_args(**wrong)), None) == _cabi.ERR_INVALID
    need = C.c_uint64()
    assert L.tsw_prefix_attention_workspace(C.byref(attention_args(**wrong)), C.byref(need)) == _cabi.ERR_INVALID


# Each stride alone steps over a row, together they do not.
OVERLAPPING = [
    ("append", dict(q_out_token_stride=128)), ("append", dict(q_out_token_stride=256)), ("append", dict(q_out_head_stride=640)),
    ("append", dict(cache__k_token_stride=128)), ("append", dict(cache__v_head_stride=256)), ("append", dict(cache__k_page_stride=256)),
    ("append", dict(cache__v_page_stride=15 * 256 + 128)), ("append", dict(cache__k=1 << 41)),
    ("attend", dict(out_token_stride=128)), ("attend", dict(out_token_stride=384)), ("attend", dict(out_head_stride=256)),
]


@pytest.mark.parametrize("call,wrong", OVERLAPPING, ids=lambda w: w if isinstance(w, str) else "-".join(f"{k}={v}" for k, v in w.items()))
def test_overlapping_results_are_refused(built, call, wrong):
    L = _cabi.lib()
    if call == "append":
        assert L.tsw_kv_append(0, C.byref(append_args(**wrong)), None) == _cabi.ERR_INVALID
    else:
        assert L.tsw_prefix_attention(0, C.byref(attention_args(**wrong)), None) == _cabi.ERR_INVALID


@pytest.mark.parametrize("order", [(0, 1, 2), (0, 2, 1), (1, 0, 2), (1, 2, 0), (2, 0, 1), (2, 1, 0)])
@pytest.mark.parametrize("pad", [0, 16])
def test_layouts_with_dimensions_in_any_order_are_taken(built, order, pad):
    """Refused for want of a device at most, and not at all without rows."""
    a, counts, strides, covered = append_args(batch__tokens=0), (8, 16, 2), [0, 0, 0], 128
    for d in order:
        strides[d] = covered + pad
        covered += (counts[d] - 1) * strides[d]
    for side in "kv":
        for d, name in enumerate(("page", "token", "head")):
            setattr(a.cache, f"{side}_{name}_stride", strides[d])
    assert _cabi.lib().tsw_kv_append(0, C.byref(a), None) == 0


@pytest.mark.parametrize("device", [-1, 64, 1 << 30])
def test_device_ordinals_out_of_range(built, device):
    L = _cabi.lib()
    word = C.c_uint32()
    assert L.tsw_kv_append(device, C.byref(append_args()), None) == _cabi.ERR_INVALID
    assert L.tsw_prefix_attention(device, C.byref(attention_args()), None) == _cabi.ERR_INVALID
    assert L.tsw_kv_status(device, None, C.byref(word), 0) == _cabi.ERR_INVALID


def test_good_arguments_without_a_device_fail_loudly(built):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: these addresses are not memory")
    L = _cabi.lib()
    assert L.tsw_kv_append(0, C.byref(append_args()), None) in (_cabi.ERR_NO_DEVICE, _cabi.ERR_CUDA)
    assert L.tsw_prefix_attention(0, C.byref(attention_args()), None) in (_cabi.ERR_NO_DEVICE, _cabi.ERR_CUDA)
    # a call without rows or without sequences has nothing to do
    for kw in (dict(batch__tokens=0), dict(batch__batch=0)):
        assert L.tsw_kv_append(0, C.byref(append_args(**kw)), None) == 0
        assert L.tsw_prefix_attention(0, C.byref(attention_args(**kw)), None) == 0


def test_plan_only_engine_runs_no_kernels(built):
    repo_reset()
    with MemoryManager(0, device=-1) as mm:
        L = _cabi.lib()
        assert L.tsw_func_kv_append(mm.h, b"f", C.byref(append_args()), None) == _cabi.ERR_NO_DEVICE
        assert L.tsw_func_prefix_attention(mm.h, b"f", C.byref(attention_args()), None) == _cabi.ERR_NO_DEVICE
    repo_reset()


def test_cpu_tensors_are_refused(built):
    from torpor_b200 import kv_cache
    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    cache = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CPU"):
        kv_cache.kv_append(cache, cache.clone(), x, x, i.view(1, 1), i, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CPU"):
        kv_cache.prefix_attention(x, cache, cache.clone(), i.view(1, 1), i, torch.zeros(2, dtype=torch.int32))


def test_frequencies():
    from torpor_b200 import kv_cache
    f = kv_cache.rope_frequencies(8, 10000.0, device="cpu")
    assert f.dtype is torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    assert kv_cache.rope_frequencies(0, device="cpu").numel() == 0
    with pytest.raises(ValueError):
        kv_cache.rope_frequencies(7, device="cpu")


def test_sizes_that_the_c_structures_would_cut_are_refused():
    """Expanded tensors have such sizes without the memory."""
    from torpor_b200 import kv_cache
    cpu, half = torch.device("cpu"), torch.float16
    x = torch.zeros(1, 1, 8, dtype=half)
    for shape in ((2 ** 28 + 1, 1, 8), (2 ** 32 + 1, 1, 8), (1, 65537, 8), (1, 2 ** 32 + 1, 8)):
        with pytest.raises(ValueError, match="at most"):
            kv_cache._rows("q", x.expand(shape), half, cpu)
    with pytest.raises(ValueError, match="at most"):
        kv_cache._rows("q", torch.zeros(1, 1, 513, dtype=half), half, cpu)
    for shape in ((2 ** 31, 1, 1, 8), (2 ** 32 + 1, 1, 1, 8), (1, 2 ** 20 + 1, 1, 8), (1, 2 ** 32 + 1, 1, 8), (1, 1, 4097, 8)):
        with pytest.raises(ValueError, match="at most"):
            kv_cache._pages(x[None].expand(shape), x[None].expand(shape), half, cpu, "cache")
    i = torch.zeros(1, dtype=torch.int32)
    many = torch.zeros(2 ** 24 + 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="at most"):
        kv_cache._batch(i[None].expand(2 ** 24, 1), many[:-1], many, 1, cpu)
