"""Key/value cache operators and autograd: no gradient is dropped in silence."""
import pytest
import torch


def operands(device):
    half = dict(dtype=torch.float16, device=device)
    i = dict(dtype=torch.int32, device=device)
    return dict(k_cache=torch.zeros(4, 16, 2, 64, **half), v_cache=torch.zeros(4, 16, 2, 64, **half), k=torch.ones(1, 2, 64, **half),
                v=torch.ones(1, 2, 64, **half), q=torch.ones(1, 2, 64, **half), q_out=torch.zeros(1, 2, 64, **half),
                inv_freq=torch.ones(32, dtype=torch.float64, device=device), page_table=torch.zeros(1, 1, **i), seq_lens=torch.ones(1, **i),
                cu_q=torch.tensor([0, 1], **i), out=torch.zeros(1, 2, 64, **half), prefix_k=torch.zeros(4, 16, 2, 64, **half),
                prefix_v=torch.zeros(4, 16, 2, 64, **half), prefix_table=torch.zeros(1, **i))


def append(o):
    from torpor_b200 import kv_cache
    return kv_cache.kv_append(*(o[n] for n in ("k_cache", "v_cache", "k", "v", "page_table", "seq_lens", "cu_q")), inv_freq=o["inv_freq"], q=o["q"],
                              q_out=o["q_out"])


def attend(o):
    from torpor_b200 import kv_cache
    return kv_cache.prefix_attention(*(o[n] for n in ("q", "k_cache", "v_cache", "page_table", "seq_lens", "cu_q")), prefix_table=o["prefix_table"],
                                     prefix_len=9, prefix_k=o["prefix_k"], prefix_v=o["prefix_v"], out=o["out"])


CALLS = [(append, n) for n in ("k_cache", "v_cache", "k", "v", "q", "q_out", "inv_freq")] + \
        [(attend, n) for n in ("q", "k_cache", "v_cache", "prefix_k", "prefix_v", "out")]


@pytest.mark.parametrize("call,name", CALLS, ids=lambda x: x if isinstance(x, str) else x.__name__)
def test_operands_that_require_a_gradient_are_refused(built, call, name):
    o = operands("cpu")
    o[name].requires_grad_()
    with pytest.raises(ValueError, match="no backward pass"):
        call(o)
    for quiet in (torch.no_grad, torch.inference_mode):
        with quiet(), pytest.raises(ValueError, match="CPU"):         # as far as the next check
            call(o)


@pytest.mark.gpu
@pytest.mark.parametrize("call,name", CALLS, ids=lambda x: x if isinstance(x, str) else x.__name__)
def test_they_are_taken_where_no_gradient_is_recorded(built, call, name):
    o = operands("cuda")
    want = call(operands("cuda"))
    o[name].requires_grad_()
    with pytest.raises(ValueError, match="no backward pass"):
        call(o)
    with torch.no_grad():
        assert torch.equal(call(o), want)


@pytest.mark.gpu
def test_what_is_written_is_seen_by_graphs_that_kept_it(built):
    w = torch.ones(1, 2, 64, dtype=torch.float16, device="cuda", requires_grad=True)
    for call, name in ((append, "k_cache"), (append, "v_cache"), (append, "q_out"), (attend, "out")):
        o = operands("cuda")
        before = {n: t._version for n, t in o.items()}
        loss = (o[name][:1].reshape(-1, 2, 64)[:1] * w).sum()
        call(o)
        written = {"k_cache", "v_cache", "q_out"} if call is append else {"out"}
        assert {n for n, t in o.items() if t._version != before[n]} == written
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        o = operands("cuda")
        append(o), attend(o)                                          # tensors without a version
