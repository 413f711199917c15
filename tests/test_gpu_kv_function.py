"""The key/value cache operators on a function's own memory: the prompt swapped in with the weights, client addresses
translated, the stream (not the host) waiting for what is still on its way."""
import numpy as np
import pytest
import torch

from kv_cases import Batch, UNIT, rotated
from torpor_b200 import _cabi, kv_cache, serving
from torpor_b200 import workloads as W
from torpor_b200.memory_manager import MemoryManager, SwapError, repo_reset

pytestmark = pytest.mark.gpu
PROMPT, STEPS = 75, 20


@pytest.fixture()
def function(built):
    assert torch.cuda.is_available(), "this test needs a CUDA device"
    repo_reset()
    kv_cache.kv_status(0, clear=True)
    ws = W.with_prompt(W.weight_set("llama_tiny", seed=5), "llama_tiny", PROMPT)
    decode = serving.PromptDecode("llama_tiny", PROMPT, STEPS)
    eng = MemoryManager(0, device=0)
    # prompt values of the size that keys and values have, not of weights
    data = lambda i: (W.tensor_values(ws, i).astype(np.float32) * (25 if ".prompt." in ws.tensors[i].name else 1)).astype(np.float16).view(np.uint8).reshape(-1)
    model = W.cold_start(eng, "f", ws, tensor_data=data, workspace_blocks=(W.SMALL_BLOCK, decode.block_bytes))
    yield eng, decode, model, model.workspace_vaddr[1], data
    eng.close()
    repo_reset()
    assert kv_cache.kv_status(0, clear=True) == 0


def read(eng, block, offset, nbytes, dtype):
    # the block's own address is what the engine translates; what lies in it is read from there
    base = eng.get_cuda_addr("f", block)
    return torch.from_numpy(eng.read_phys(base + offset, nbytes).view(dtype).copy()).cuda()


def expected(decode, data, ws, layer, step):
    """The last layer's result of one step in 64 bits, and its bound."""
    a = decode.shape
    names = {t.name: i for i, t in enumerate(ws.tensors)}
    prompt = [torch.from_numpy(data(names[f"model.layers.{layer}.prompt.{w}"]).view(np.float16).copy()).view(-1, a.kv_heads, a.head_dim)[:PROMPT].cuda()
              for w in ("keys", "values")]
    freq = torch.from_numpy(decode.tables["inv_freq"]).cuda()
    q, k, v = (torch.from_numpy(decode.tables[n]).cuda().view(-1, a.head_dim) for n in ("q", "k", "v"))
    own_k = torch.stack([rotated(k, PROMPT + j, freq, False)[0] for j in range(step + 1)]).half()
    return rotated(q, PROMPT + step, freq, False)[0].half(), torch.cat((prompt[0], own_k)), torch.cat((prompt[1], v[None].expand(step + 1, -1, -1)))


def check_last_layer(eng, decode, block, data, ws):
    a, n = decode.shape, decode.shape.heads * decode.shape.head_dim * 2
    layer, step = a.layers - 1, STEPS - 1
    q, keys, vals = expected(decode, data, ws, layer, step)
    got_q = read(eng, block, decode.offset["q_out"], n, np.float16).view(a.heads, a.head_dim)
    assert ((got_q.double() - q.double()).abs() <= 2 * UNIT[torch.float16] * q.double().abs() + 2.0 ** -18).all()
    # attend with what the kernels themselves stored: the queries and the own keys are roundings of their own
    own = read(eng, block, decode.offset["keys", layer], decode.own_pages * decode.page_size * n, np.float16).view(-1, a.kv_heads, a.head_dim)[:STEPS]
    assert ((own.double() - keys[PROMPT:].double()).abs() <= 2 * UNIT[torch.float16] * own.double().abs() + 2.0 ** -18).all()
    c = Batch([1], [0], q_heads=a.heads, kv_heads=a.kv_heads, dim=a.head_dim, prefix=0)
    keys = torch.cat((keys[:PROMPT], own))
    c.own, c.prefix, c.page_size = [PROMPT + STEPS], 0, PROMPT + STEPS
    c.table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    out = read(eng, block, decode.offset["out"], n, np.float16).view(1, a.heads, a.head_dim)
    c.check(out, q=got_q[None], k_cache=keys[None], v_cache=vals[None])


def test_decode_behind_a_swapped_in_prompt(function):
    eng, decode, model, block, data = function
    stream = torch.cuda.Stream()
    decode.enqueue(eng, "f", model, block, stream.cuda_stream)      # where the cold start put it
    stream.synchronize()
    check_last_layer(eng, decode, block, data, model.ws)
    # other functions come and go, so that the blocks lie elsewhere at every swap-in; the calls are enqueued while the
    # prompt is still on its way
    before = eng.get_cuda_addr("f", block)
    moved = False
    for cycle in range(3):
        eng.evict("f")
        W.cold_start(eng, f"other{cycle}", W.weight_set("bert_tiny", seed=cycle))
        eng.swap_in("f")
        decode.enqueue(eng, "f", model, block, stream.cuda_stream)
        stream.synchronize()
        eng.wait_ready("f")
        moved = moved or eng.get_cuda_addr("f", block) != before
        check_last_layer(eng, decode, block, data, model.ws)
    assert moved, "the blocks were never placed elsewhere"


def test_operands_have_to_be_the_functions(function):
    eng, decode, model, block, _ = function
    at = {t.name: model.tensor_vaddr[i] for i, t in enumerate(model.ws.tensors) if ".prompt." in t.name}
    prompt = lambda l, what: at[f"model.layers.{l}.prompt.{what}"]

    def refused(code, call, change):
        args = decode._append(block, 0, 0) if call == "kv_append" else decode._attention(block, prompt, 0, 0)
        change(args)
        with pytest.raises(SwapError) as e:
            getattr(eng, call)("f", args)
        assert e.value.code == code, e.value

    def at_end(field):
        def change(a):
            setattr(a, field, block + decode.block_bytes - 128)
        return change

    own = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda").data_ptr()
    for call, fields in (("kv_append", ("q", "q_out", "k", "v", "inv_freq")), ("prefix_attention", ("q", "out", "prefix_table", "workspace"))):
        for f in fields:
            refused(_cabi.ERR_NOT_FOUND, call, lambda a: setattr(a, f, own))
            if f != "prefix_table":
                refused(_cabi.ERR_NOT_FOUND, call, at_end(f))
    refused(_cabi.ERR_NOT_FOUND, "prefix_attention", lambda a: setattr(a.prefix, "pages", 1 << 20))
    refused(_cabi.ERR_NOT_FOUND, "kv_append", lambda a: setattr(a.batch, "seq_lens", own))
    refused(_cabi.ERR_BUFFER, "prefix_attention", lambda a: setattr(a, "workspace_bytes", 256))
    refused(_cabi.ERR_INVALID, "prefix_attention", lambda a: setattr(a, "workspace", 0))
    args = decode._append(block, 0, 0)
    with pytest.raises(SwapError) as e:
        eng.kv_append("nobody", args)
    assert e.value.code == _cabi.ERR_UNKNOWN_MODEL
    eng.evict("f")
    with pytest.raises(SwapError) as e:
        eng.kv_append("f", args)
    assert e.value.code == _cabi.ERR_STATE
    eng.swap_in("f")
    eng.wait_ready("f")
    eng.kv_append("f", args)
    torch.cuda.synchronize()


def test_launches_are_counted(function):
    eng, decode, model, block, _ = function
    at = {t.name: model.tensor_vaddr[i] for i, t in enumerate(model.ws.tensors) if ".prompt." in t.name}
    prompt = lambda l, what: at[f"model.layers.{l}.prompt.{what}"]
    append, attention = decode._append(block, 0, 0), decode._attention(block, prompt, 0, 0)
    rows = decode._attention(block, prompt, 0, 0)
    rows.scale = 0.0                                # not for the tiles
    for call, args, launches in ((eng.kv_append, append, 1), (eng.prefix_attention, attention, 2), (eng.prefix_attention, rows, 1)):
        before = eng.stats()["kernel_launches"]
        call("f", args)
        assert eng.stats()["kernel_launches"] - before == launches
        args.batch.tokens = 0
        call("f", args)
        assert eng.stats()["kernel_launches"] - before == launches
    torch.cuda.synchronize()


@pytest.mark.parametrize("call,side", [("kv_append", "cache"), ("prefix_attention", "cache"), ("prefix_attention", "prefix")])
@pytest.mark.parametrize("field", ["k_page_stride", "v_page_stride"])
def test_pages_that_pass_64_bits_leave_their_block(function, call, side, field):
    """2^25 strides of 2^39 bytes are 0 modulo 2^64: no reason to take them for a short operand."""
    eng, decode, model, block, _ = function
    at = {t.name: model.tensor_vaddr[i] for i, t in enumerate(model.ws.tensors) if ".prompt." in t.name}
    args = decode._append(block, 0, 0) if call == "kv_append" else decode._attention(block, lambda l, what: at[f"model.layers.{l}.prompt.{what}"], 0, 0)
    pages = getattr(args, side)
    pages.pages = (1 << 25) + 1
    setattr(pages, field, 1 << 39)
    with pytest.raises(SwapError) as e:
        getattr(eng, call)("f", args)
    assert e.value.code == _cabi.ERR_NOT_FOUND, e.value


def test_request_stream_with_decoding_functions(built):
    repo_reset()
    out = serving.run_stream(n_gpus=1, n_models=4, rate=40.0, duration_s=1.0, cap_bytes=300 << 20, seed=4, archs=("llama_tiny",),
                             devices=[0], decode_tokens=6, prompt_tokens=200)
    assert out["completed"] == out["requests"] > 20
    assert out["requests_decoded"] == out["requests"] and out["swaps"] > 0
    assert kv_cache.kv_status(0, clear=True) == 0
