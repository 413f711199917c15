"""Key/value cache operators on a GPU: legal calls at the edges of what the arguments allow."""
import ctypes as C
import math

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


BROKEN = [[0, 10, 12, 5], [0, 10, 12, 0], [0, 12, 10, 12], [9, 10, 12, 3]]


@pytest.mark.parametrize("cu", BROKEN)
def test_append_follows_no_row_into_a_sequence_that_does_not_have_it(cu):
    """A row is appended to a sequence whose rows contain it, or not at all."""
    c = Batch([10, 2, 0], [40, 30, 20], seed=3)
    c.cu_q.copy_(torch.tensor(cu, dtype=torch.int32))
    want_k, want_v = c.k_cache.clone(), c.v_cache.clone()
    other_k, other_v = want_k.clone(), want_v.clone()
    for tok in range(c.tokens):
        for b in range(3):
            if not cu[b] <= tok < cu[b + 1]:
                continue
            j = c.own[b] - (cu[b + 1] - cu[b]) + tok - cu[b]
            want_k[int(c.table[b, j // 16]), j % 16], want_v[int(c.table[b, j // 16]), j % 16] = c.k[tok], c.v[tok]
            break
    kv_cache.kv_append(c.k_cache, c.v_cache, c.k, c.v, c.table, c.lens, c.cu_q)
    assert kv_cache.kv_status(0, clear=True) in (0, kv_cache.BAD_ROWS)
    # a row that two overlapping sequences claim may be found in either
    changed = (c.k_cache != other_k).flatten(2).any(-1)
    assert (changed <= (want_k != other_k).flatten(2).any(-1)).all()
    if cu == BROKEN[0]:
        assert torch.equal(c.k_cache, want_k) and torch.equal(c.v_cache, want_v)


@pytest.mark.parametrize("cu", BROKEN)
@pytest.mark.parametrize("prefix,dim,causal", [(0, 64, True), (300, 128, True), (300, 64, False), (20, 200, True)])
def test_attention_with_rows_out_of_order_is_recorded_and_stays_in_bounds(cu, prefix, dim, causal):
    c = Batch([10, 2, 0], [400, 300, 200], dim=dim, prefix=prefix, seed=4, pad=2)
    c.cu_q.copy_(torch.tensor(cu, dtype=torch.int32))
    kv_cache.prefix_attention(c.q, c.k_cache, c.v_cache, c.table, c.lens, c.cu_q, max_q=12, causal=causal, prefix_len=prefix,
                              prefix_table=c.prefix_table if prefix else None)
    # the tile kernel looks at every sequence, the row kernel (wide heads) at those that it finds rows in
    assert kv_cache.kv_status(0, clear=True) in ((0, kv_cache.BAD_ROWS) if dim > 128 else (kv_cache.BAD_ROWS,))


def test_rows_claimed_by_very_many_sequences_are_recorded_and_not_dealt_out():
    """131072 sequences that all name the same 8192 rows: more tiles than 32 bits count."""
    tokens, heads, batch, keys = 8192, 32, 131072, 32768
    q = torch.randn(tokens, heads, 8, device="cuda").half()
    k, v = torch.randn(2, 4, 128, heads, 8, device="cuda").half()
    cu = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    cu[1::2] = tokens
    table = torch.zeros(batch, keys // 128, dtype=torch.int32, device="cuda")
    lens = torch.full((batch,), keys, dtype=torch.int32, device="cuda")
    kv_cache.prefix_attention(q, k, v, table, lens, cu, max_q=tokens, causal=False)
    assert kv_cache.kv_status(0, clear=True) == kv_cache.BAD_ROWS


@pytest.mark.parametrize("q_lens,max_q,pad", [([5], 3, 0), ([200], 100, 40)])
def test_what_follows_on_the_stream_comes_after_both_kernels(q_lens, max_q, pad):
    """No row has anything to join (its sequence has more rows than max_q), while the tile kernel walks a long prefix for them: its
    workspace and its report are complete for whatever the stream does next."""
    c = Batch(q_lens, [400], q_heads=32, kv_heads=32, dim=128, prefix=40000, page_size=64, pad=pad, seed=6)
    c.prefix_table[-1] = c.pages                       # seen last, in the range that ends the list
    call = Call(c, max_q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            call.workspace.fill_(0xFF)
            call()
            behind = call.workspace.clone()
            word = kv_cache.kv_status(0, side.cuda_stream, clear=True)
        torch.cuda.synchronize()
        assert word == kv_cache.BAD_ROWS | kv_cache.BAD_PAGE
        assert kv_cache.kv_status(0) == 0
        assert torch.equal(behind, call.workspace)
        assert (call.out == 5.0).all()


def long_list(n, page_size):
    """``n`` keys that name two pages over and over, values 0 in the first half of the list and 1 in the second: (table, keys, values)."""
    pages_ = -(-n // page_size)
    table = torch.zeros(pages_, dtype=torch.int32, device="cuda")
    table[pages_ // 2:] = 1
    k = torch.zeros(2, page_size, 1, 8, dtype=torch.float16, device="cuda")
    v = torch.stack((torch.zeros_like(k[0]), torch.ones_like(k[0])))
    return table, k, v


@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("n", [0x7fffff00, (1 << 30) + (1 << 29) + 77])
def test_lists_longer_than_two_to_the_thirtieth(where, n):
    """Equal scores, so the result is the share of the second half and the log-sum is ln n.  Sums of equal powers of two are exact in
    32 bits up to 2^24 of them; joining up to 300 of them rounds each time by 2^-24 at most, the result once."""
    ps = 1 << 20
    table, k, v = long_list(n, ps)
    q = torch.randn(3, 1, 8, device="cuda").half()
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    if where == "prefix":
        out, lse = kv_cache.prefix_attention(q, k, v, torch.zeros(1, 0, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"),
                                             cu, prefix_table=table, prefix_len=n, return_lse=True)
    else:
        out, lse = kv_cache.prefix_attention(q, k, v, table[None], torch.tensor([n], dtype=torch.int32, device="cuda"), cu, causal=False, return_lse=True)
    want = (n - len(table) // 2 * ps) / n
    assert (out.double() - want).abs().max() <= want * (2.0 ** -11 + 300 * 2.0 ** -23)
    assert (lse.double() - torch.tensor(float(n)).double().log().cuda()).abs().max() <= 300 * 2.0 ** -24 + 2.0 ** -22 * 23


def one_key_and_a_tail(n, share, dtype, where, heads=1, dim=64):
    """Key 7 takes ``share`` of the weight, the others an equal part of the rest each; its value is 0, theirs 1.
    Returns the call's results and what they are in 64 bits."""
    u = 8.0
    score = math.log(share / (1 - share) * (n - 1))
    q = torch.zeros(1, heads, dim, device="cuda", dtype=dtype)
    q[..., 0] = u
    pages_ = -(-n // 256)
    k = torch.zeros(pages_ + 1, 256, heads, dim, device="cuda", dtype=dtype)
    v = torch.ones_like(k)
    k[0, 7, :, 0], v[0, 7] = score / u, 0.0
    score = u * k[0, 7, 0, 0].double().item()
    table, cu = torch.arange(pages_, dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n if where == "own" else 0], dtype=torch.int32, device="cuda")
    out, lse = kv_cache.prefix_attention(q, k, v, table[None], lens, cu, max_q=1, scale=1.0, return_lse=True,
                                         **(dict(prefix_table=table, prefix_len=n) if where == "prefix" else {}))
    w = math.exp(score)
    return out, lse, (n - 1) / (w + n - 1), math.log(w + n - 1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("where", ["prefix", "own"])
@pytest.mark.parametrize("n", [1 << 15, 1 << 18, 1 << 20, (1 << 22) + 5])
@pytest.mark.parametrize("share", [0.9, 0.99])
def test_a_flat_tail_behind_one_key_counts(dtype, where, n, share):
    """Weights far below the largest add up.  Each is rounded once (to 16 bits, half a step relative; in fp16 to 2^-36 of the largest
    at worst, where its steps are equal), the result once more; the exponential and its argument (up to 21, in 32 bits)
    take 2^-18, the sums of n / 64 / 148 units and 148 ranges 2^-13 at most."""
    out, lse, want, want_lse = one_key_and_a_tail(n, share, dtype, where)
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    tol = want * (2.01 * u + 2.0 ** -18 + 2.0 ** -13) + (n * share * 2.0 ** -36 if dtype is torch.float16 else 0.0)
    assert (out.double() - want).abs().max().item() <= tol, (out.double().flatten()[0].item(), want)
    assert abs(lse.item() - want_lse) <= 2.0 ** -13 + 2.0 ** -18


@pytest.mark.parametrize("lens", [[65, 33], [66, 33], [2**31 - 1, 33], [-1, 33]])
def test_append_beyond_the_table_overwrites_nothing(lens):
    """A sequence that has outgrown its table: the new token has no place, and the last cached one keeps its own."""
    c = Batch([1, 2], [64, 33], seed=12)
    c.table = c.table[:, :4].contiguous()
    c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    k0, v0 = c.k_cache.clone(), c.v_cache.clone()
    q_out = torch.full_like(c.q, 7.0)
    kv_cache.kv_append(c.k_cache, c.v_cache, c.k, c.v, c.table, c.lens, c.cu_q, q=c.q, q_out=q_out)
    assert kv_cache.kv_status(0, clear=True) == kv_cache.BAD_LENGTH
    assert (q_out[0] == 7.0).all() and torch.equal(q_out[1:], c.q[1:])
    for j in (31, 32):
        k0[int(c.table[1, j // 16]), j % 16], v0[int(c.table[1, j // 16]), j % 16] = c.k[j - 30], c.v[j - 30]
    assert torch.equal(c.k_cache, k0) and torch.equal(c.v_cache, v0)


@pytest.mark.parametrize("where", ["prefix", "own"])
def test_the_row_kernel_sums_more_keys_than_32_bits_count_one_by_one(where):
    """2^24 + 2^20 equal scores, values 1: the result is 1.  Sums of up to 2^15 ones are exact, and so are those of their sums."""
    n, ps = (1 << 24) + (1 << 20) + 5, 1 << 20
    table = torch.zeros(-(-n // ps), dtype=torch.int32, device="cuda")
    k, v = torch.zeros(1, ps, 1, 2, dtype=torch.float16, device="cuda"), torch.ones(1, ps, 1, 2, dtype=torch.float16, device="cuda")
    q, cu = torch.randn(1, 1, 2, device="cuda").half(), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    if where == "prefix":
        none = torch.zeros(1, 0, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        out, lse = kv_cache.prefix_attention(q, k, v, *none, cu, prefix_table=table, prefix_len=n, return_lse=True)
    else:
        out, lse = kv_cache.prefix_attention(q, k, v, table[None], torch.tensor([n], dtype=torch.int32, device="cuda"), cu, return_lse=True)
    assert (out == 1.0).all()
    assert abs(lse.item() - math.log(n)) <= 2.0 ** -22 * 17


@pytest.mark.parametrize("dim", [200, 512, 50])
def test_the_row_kernel_joins_its_sums(dim):
    """Over the borders of its partial sums, with maxima that move on both sides of them."""
    c = Batch([1, 2], [40000, 33000], dim=dim, prefix=32768 * 2 + 17, seed=15, page_size=512)
    out, lse = kv_cache.prefix_attention(c.q, c.k_cache, c.v_cache, c.table, c.lens, c.cu_q, max_q=2, prefix_table=c.prefix_table, prefix_len=c.prefix,
                                         return_lse=True)
    c.check(out, lse)


def test_calls_on_a_functions_memory_cannot_be_captured(built):
    """Its blocks move with every swap-in; a replay would go to where they lay."""
    from torpor_b200 import serving
    from torpor_b200 import workloads as W
    from torpor_b200.memory_manager import MemoryManager, SwapError, repo_reset
    repo_reset()
    ws = W.with_prompt(W.weight_set("llama_tiny", seed=5), "llama_tiny", 20)
    decode = serving.PromptDecode("llama_tiny", 20, 2)
    with MemoryManager(0, device=0) as eng:
        model = W.cold_start(eng, "f", ws, workspace_blocks=(W.SMALL_BLOCK, decode.block_bytes))
        block = model.workspace_vaddr[1]
        at = {t.name: model.tensor_vaddr[i] for i, t in enumerate(ws.tensors)}
        append = decode._append(block, 0, 0)
        attention = decode._attention(block, lambda l, what: at[f"model.layers.{l}.prompt.{what}"], 0, 0)
        stream = torch.cuda.Stream()
        decode.enqueue(eng, "f", model, block, stream.cuda_stream)
        stream.synchronize()
        for call, args in ((eng.kv_append, append), (eng.prefix_attention, attention)):
            graph, x = torch.cuda.CUDAGraph(), torch.zeros(1, device="cuda")
            with torch.cuda.graph(graph, stream=stream):
                with pytest.raises(SwapError) as e:
                    call("f", args, stream.cuda_stream)
                x += 1
            assert e.value.code == _cabi.ERR_STATE
            graph.replay()
            torch.cuda.synchronize()
            assert x.item() == 1
            call("f", args, stream.cuda_stream)
        stream.synchronize()
    repo_reset()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, 0.7, 5.3])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_scores_of_any_size_leave_finite_results(dtype, scale, where):
    """Every 5th key has the largest score, exactly, the others one that is 2^-7 smaller (or larger, where scores are negative): sums of one
    product, so scores are exact before the scale.  Rows whose scores lie 40 or more apart are the average of the
    largest keys' values; all rows are averages of values between 1 and 2.  Weights rounded once, the result once: 2.01 half steps,
    2^-12 for sums and their joining; where scores lie apart, what the others add is below e^-40 * 5."""
    n, ps, dim, heads = 3000, 64, 64, 46
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.zeros(-(-n // ps), ps, 1, dim, dtype=dtype, device="cuda")
    v = torch.rand(k.shape, generator=g, device="cuda").add(1).to(dtype)
    at = torch.arange(k.shape[0] * ps, device="cuda").view(k.shape[:2])
    big = 2.0 ** 15 if dtype is torch.float16 else 2.0 ** 60
    k[..., 0, 0] = torch.where(at % 5 == 3, big, big * (1 - 2.0 ** -7)).to(dtype)
    k[..., 0, 1] = torch.where(at % 5 == 3, big * (1 - 2.0 ** -7), big).to(dtype)
    q = torch.zeros(1, heads, dim, dtype=dtype, device="cuda")
    half = heads // 2
    sizes = [2.0 ** (15 - i) if dtype is torch.float16 else 2.0 ** (55 - 5 * i) for i in range(half)]
    for i, s in enumerate(sizes):
        q[0, i, 0] = s                       # positive scores
        q[0, half + i, 1] = -s               # negative ones: the smallest in size is the largest
    table, cu = torch.arange(k.shape[0], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n if where == "own" else 0], dtype=torch.int32, device="cuda")
    out, lse = kv_cache.prefix_attention(q, k, v, table[None], lens, cu, max_q=1, scale=scale, return_lse=True,
                                         **(dict(prefix_table=table, prefix_len=n) if where == "prefix" else {}))
    out = out.double()[0]
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    assert (out >= 1 - 4 * u).all() and (out <= 2 + 8 * u).all()
    vals = v.view(-1, dim)[:n].double()
    want = vals[torch.arange(n, device="cuda") % 5 == 3].mean(0)
    apart = torch.tensor([s * big * scale * 2.0 ** -7 >= 40 for s in sizes] * 2, device="cuda")
    assert apart.sum() >= 10
    assert ((out - want).abs()[apart] <= want * (2.01 * u + 2.0 ** -12) + 5 * math.exp(-40)).all()
