"""Key/value cache operators on a GPU: legal calls at the edges of what the arguments allow."""
import ctypes as C

import pytest
import torch

from kv_cases import Batch
from torpor_b200 import _cabi, kv_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status(built):
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    kv_cache.kv_status(0, clear=True)
    yield
    assert kv_cache.kv_status(0, clear=True) == 0


def pages(k, v):
    return _cabi.KvPages(k.data_ptr(), v.data_ptr(), *(2 * s for s in k.stride()[:3]), *(2 * s for s in v.stride()[:3]), k.shape[0], k.shape[1])


class Call:
    """An attention call over the C ABI, whose arguments the tensor API would fit to the tensors."""

    def __init__(self, c, max_q, causal=True):
        self.c, self.out = c, torch.full_like(c.q, 5.0)
        self.lse = torch.full((c.tokens, c.q_heads), 5.0, device="cuda")
        a = self.a = _cabi.PrefixAttentionArgs()
        a.cache = a.prefix = pages(c.k_cache, c.v_cache)
        a.batch = _cabi.KvBatch(c.table.data_ptr(), c.lens.data_ptr(), c.cu_q.data_ptr(), c.batch, c.table.shape[1], c.table.stride(0), c.tokens)
        a.prefix_table, a.prefix_len, a.max_q = c.prefix_table.data_ptr(), c.prefix, max_q
        a.q, a.out, a.lse = c.q.data_ptr(), self.out.data_ptr(), self.lse.data_ptr()
        a.q_token_stride, a.q_head_stride, _ = (2 * s for s in c.q.stride())
        a.out_token_stride, a.out_head_stride, _ = (2 * s for s in self.out.stride())
        a.dtype, a.q_heads, a.kv_heads, a.head_dim = (_cabi.F16 if c.dtype is torch.float16 else _cabi.BF16), c.q_heads, c.kv_heads, c.dim
        a.causal, a.scale = int(causal), c.dim ** -0.5
        need = C.c_uint64()
        assert _cabi.lib().tsw_prefix_attention_workspace(C.byref(a), C.byref(need)) == 0
        self.workspace = torch.full((max(1, need.value),), 0xFF, dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = self.workspace.data_ptr(), need.value

    def __call__(self):
        assert _cabi.lib().tsw_prefix_attention(0, C.byref(self.a), torch.cuda.current_stream().cuda_stream) == 0, _cabi.lib().tsw_last_error()
        return self.out, self.lse


@pytest.mark.parametrize("q_lens,own,q_heads,kv_heads,dim,prefix", [
    ([1], [2000], 32, 32, 128, 5000), ([1], [2000], 32, 32, 64, 5000), ([1, 1, 1], [700, 0, 90], 32, 4, 128, 3000), ([2, 5], [400, 5], 16, 16, 64, 700),
    ([1], [900], 8, 2, 128, 0)])
def test_max_q_may_be_any_upper_bound(q_lens, own, q_heads, kv_heads, dim, prefix):
    """More than the rows of the batch is a bound like any other: a captured step keeps one for all its batches."""
    c = Batch(q_lens, own, q_heads=q_heads, kv_heads=kv_heads, dim=dim, prefix=prefix, seed=q_heads + dim)
    c.check(*Call(c, max(q_lens))())
    want = [t.clone() for t in Call(c, c.tokens)()]
    c.check(*want)
    for max_q in (c.tokens + 1, 16, 64, 200, 0x7fffffff):
        got = Call(c, max_q)()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), max_q
