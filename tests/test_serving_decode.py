"""Functions that decode: what their weight sets, blocks and calls look like, without a GPU."""
import ctypes as C

import numpy as np
import pytest

from torpor_b200 import _cabi, serving
from torpor_b200 import workloads as W
from torpor_b200.memory_manager import MemoryManager, SizeOnly, repo_reset


def test_prompt_is_part_of_the_weight_set():
    ws = W.weight_set("llama_tiny")
    both = W.with_prompt(ws, "llama_tiny", 100)
    assert both.tensors[:len(ws.tensors)] == ws.tensors and both.seed == ws.seed
    extra = both.tensors[len(ws.tensors):]
    assert [t.name for t in extra] == [f"model.layers.{l}.prompt.{w}" for l in range(2) for w in ("keys", "values")]
    assert all(t.shape == (7, 16, 8, 128) and t.dtype == "float16" for t in extra)
    assert np.array_equal(W.tensor_bytes(both, 0), W.tensor_bytes(ws, 0))
    for name, a in W.ATTENTION.items():
        q = next(t for t in W.weight_set(name).tensors if t.name.endswith("q_proj.weight"))
        assert q.shape[0] == a.heads * a.head_dim
        assert sum(t.name.endswith("q_proj.weight") for t in W.weight_set(name).tensors) == a.layers


@pytest.mark.parametrize("arch,prompt,steps", [("llama_tiny", 1, 1), ("llama_mid", 333, 40), ("llama2_7b", 2048, 16)])
def test_block_of_a_request_holds_its_operands_apart(built, arch, prompt, steps):
    d = serving.PromptDecode(arch, prompt, steps)
    a = d.shape
    base = 1 << 40
    spans = []
    for n, t in d.tables.items():
        spans.append((d.offset[n], t.nbytes))
        assert np.array_equal(d.image[d.offset[n]:d.offset[n] + t.nbytes], t.view(np.uint8))
    pages = d.own_pages * d.page_size * a.kv_heads * a.head_dim * 2
    assert d.own_pages * d.page_size >= steps and d.prompt_pages * d.page_size >= prompt
    spans += [(d.offset[n], a.heads * a.head_dim * 2) for n in ("q_out", "out")]
    spans += [(d.offset[n, l], pages) for l in range(a.layers) for n in ("keys", "values")]
    spans.append((d.offset["workspace"], d.workspace_bytes))
    spans.sort()
    for (x, n), (y, _) in zip(spans, spans[1:]):
        assert x + n <= y and y % 256 == 0
    assert spans[-1][0] + spans[-1][1] <= d.block_bytes and d.workspace_bytes > 0
    x, y = d._append(base, a.layers - 1, steps - 1), d._attention(base, lambda l, w: 1 << 41, a.layers - 1, steps - 1)
    assert d.tables["lens"][(x.batch.seq_lens - base - d.offset["lens"]) // 4] == steps
    need = C.c_uint64()
    assert _cabi.lib().tsw_prefix_attention_workspace(C.byref(y), C.byref(need)) == 0 and need.value == d.workspace_bytes
    # a plan-only engine gets as far as saying that it has no device
    repo_reset()
    with MemoryManager(0, device=-1) as mm:
        assert _cabi.lib().tsw_func_kv_append(mm.h, b"f", C.byref(x), None) == _cabi.ERR_NO_DEVICE
        assert _cabi.lib().tsw_func_prefix_attention(mm.h, b"f", C.byref(y), None) == _cabi.ERR_NO_DEVICE
    repo_reset()


def test_refusals(built):
    for bad in ((0, 1), (1, 0)):
        with pytest.raises(ValueError):
            serving.PromptDecode("llama_tiny", *bad)
    with pytest.raises(KeyError):
        serving.PromptDecode("resnet50", 16, 1)
    repo_reset()
    with pytest.raises(ValueError, match="GPU"):
        serving.SwapServer(1, 1 << 30, devices=[-1], decode_tokens=4)
    repo_reset()


@pytest.mark.parametrize("wrong", [dict(decode_tokens=-1), dict(decode_tokens=4, prompt_tokens=0), dict(decode_tokens=4)])
def test_a_server_that_refuses_has_made_no_engine(built, monkeypatch, wrong):
    made = []
    monkeypatch.setattr(serving, "MemoryManager", lambda *a, **kw: made.append(a))
    with pytest.raises(ValueError):
        serving.SwapServer(1, 1 << 30, devices=[-1], **wrong)
    assert not made
