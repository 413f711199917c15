"""Key/value cache operators on a GPU: against 64-bit references, at the sizes and masks where they can go wrong."""
import itertools
import math
import os
import subprocess
import sys

import pytest
import torch

from kv_cases import Batch, rotated
from torpor_b200 import _cabi, kv_cache
from torpor_b200.memory_manager import SwapError

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def clean_status(built):
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    kv_cache.kv_status(0, clear=True)
    yield
    assert kv_cache.kv_status(0, clear=True) == 0


def attend(c, **kw):
    kw.setdefault("max_q", max(c.q_lens + [0]))
    return kv_cache.prefix_attention(c.q, c.k_cache, c.v_cache, c.table, c.lens, c.cu_q,
                                     prefix_table=c.prefix_table if c.prefix else None, prefix_len=c.prefix, **kw)


# ------------------------------------------------------------------------------- append

def append_and_check(c, rotary, interleaved=False, offset=0, queries=True, in_place=False, theta=10000.0):
    freq = kv_cache.rope_frequencies(rotary, theta) if rotary else None
    k0, v0, q0 = c.k_cache.clone(), c.v_cache.clone(), c.q.clone()
    q_out = c.q if in_place else torch.full_like(c.q, 7.0) if queries else None
    got = kv_cache.kv_append(c.k_cache, c.v_cache, c.k, c.v, c.table, c.lens, c.cu_q, inv_freq=freq, interleaved=interleaved,
                             position_offset=offset, q=c.q if queries else None, q_out=q_out)
    freq = freq if rotary else torch.zeros(0, dtype=torch.float64, device="cuda")
    want_q = q0.clone() if in_place else torch.full_like(q0, 7.0)
    touched = torch.zeros(c.k_cache.shape[:2], dtype=torch.bool, device="cuda")
    for b, at, n, length in c.rows():
        for i in range(n):
            j = length - n + i
            if j < 0:
                continue
            page, place = int(c.table[b, j // c.page_size]), j % c.page_size
            touched[page, place] = True
            ref, tol = rotated(c.k[at + i], offset + j, freq, interleaved)
            assert ((c.k_cache[page, place].double() - ref).abs() <= tol).all()
            assert torch.equal(c.v_cache[page, place], c.v[at + i])
            if queries:
                ref, tol = rotated(q0[at + i], offset + j, freq, interleaved)
                assert ((got[at + i].double() - ref).abs() <= tol).all()
                want_q[at + i] = got[at + i]
    assert torch.equal(c.k_cache[~touched], k0[~touched]) and torch.equal(c.v_cache[~touched], v0[~touched])
    if queries:
        assert torch.equal(got, want_q), "rows of nobody were written"
    else:
        assert got is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rotary,interleaved", [(64, 64, False), (128, 128, True), (128, 64, False), (80, 40, False), (96, 96, False),
                                                     (64, 0, False), (34, 10, False), (34, 6, True), (256, 256, False), (2, 2, True)])
def test_append_rotates_and_places(dtype, dim, rotary, interleaved):
    c = Batch([1, 3, 0, 20, 7], [1, 40, 5, 33, 7], dim=dim, dtype=dtype, seed=dim + rotary, page_size=16, pad=3)
    append_and_check(c, rotary, interleaved, offset=11)


@pytest.mark.parametrize("q_heads,kv_heads,page_size,head_major,row_pad", [
    (1, 1, 1, False, 0), (32, 32, 16, True, 0), (28, 4, 24, False, 0), (8, 8, 100, True, 8), (4, 2, 16, False, 1), (3, 5, 7, False, 2)])
def test_append_layouts(q_heads, kv_heads, page_size, head_major, row_pad):
    c = Batch([5, 1, 31], [5, 300, 64], q_heads=q_heads, kv_heads=kv_heads, dim=64, page_size=page_size, head_major=head_major,
              row_pad=row_pad, seed=q_heads)
    append_and_check(c, 64)


@pytest.mark.parametrize("offset", [0, 1, 131071, (1 << 31) + 5, (1 << 32) - 1])
def test_append_far_positions(offset):
    append_and_check(Batch([2, 2], [9, 2], dim=128, dtype=torch.bfloat16, seed=3), 128, offset=offset)


def test_append_rows_of_nobody_and_rows_beyond_the_length():
    append_and_check(Batch([4, 2, 6], [2, 0, 6], first=3, pad=5, seed=4), 32)
    append_and_check(Batch([0, 0], [4, 0], pad=2, seed=5), 32)


def test_append_in_place_and_without_queries():
    append_and_check(Batch([3, 50], [17, 50], seed=6), 64, in_place=True)
    append_and_check(Batch([3, 50], [17, 50], seed=7), 64, queries=False)


def test_append_many_sequences():
    append_and_check(Batch([(i * 7) % 3 for i in range(1100)], [(i * 7) % 3 + i % 5 for i in range(1100)], q_heads=1, kv_heads=1, dim=32,
                           page_size=4, seed=8), 32)


def test_append_page_outside_the_cache_is_skipped_and_recorded():
    c = Batch([1, 1, 1], [5, 6, 7], seed=9)
    good = c.table.clone()
    for wrong in (c.pages, -1, 2**31 - 1, -2**31):
        c.table.copy_(good)
        c.table[1, 0] = wrong
        k0 = c.k_cache.clone()
        kv_cache.kv_append(c.k_cache, c.v_cache, c.k, c.v, c.table, c.lens, c.cu_q)
        assert kv_cache.kv_status(0, clear=True) == kv_cache.BAD_PAGE
        changed = (c.k_cache != k0).flatten(2).any(-1).sum().item()
        assert changed <= 2


def test_tables_out_of_order_are_recorded_not_followed():
    c = Batch([2, 2], [40, 33], seed=10)
    for name, values, want in [("cu_q", [0, 5, 4], kv_cache.BAD_ROWS), ("cu_q", [-3, 2, 4], kv_cache.BAD_ROWS),
                               ("cu_q", [0, 2, 2**31 - 1], kv_cache.BAD_ROWS),
                               ("lens", [2**31 - 1, 33], kv_cache.BAD_LENGTH), ("lens", [40, -7], kv_cache.BAD_LENGTH)]:
        old = getattr(c, name).clone()
        getattr(c, name).copy_(torch.tensor(values, dtype=torch.int32))
        kv_cache.kv_append(c.k_cache, c.v_cache, c.k, c.v, c.table, c.lens, c.cu_q)
        assert kv_cache.kv_status(0, clear=True) & want, (name, values)
        attend(c)
        assert kv_cache.kv_status(0, clear=True) & want, (name, values)
        getattr(c, name).copy_(old)


# ---------------------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,kv_heads,dim,page_size,head_major", [
    (4, 4, 64, 16, False), (8, 2, 128, 16, True), (28, 4, 128, 64, False), (7, 1, 96, 8, False), (16, 1, 80, 32, True),
    (3, 3, 128, 256, False), (32, 8, 64, 128, True), (5, 5, 40, 16, False), (2, 1, 72, 1, False), (2, 1, 8, 16, False), (6, 2, 120, 32, True),
    (128, 1, 64, 16, False), (96, 1, 128, 64, False), (130, 1, 64, 16, False), (4, 4, 256, 16, False), (4, 2, 50, 24, False)])
def test_attention_heads_and_pages(dtype, q_heads, kv_heads, dim, page_size, head_major):
    c = Batch([1, 1, 1, 1], [1, 37, 128, 300], q_heads=q_heads, kv_heads=kv_heads, dim=dim, page_size=page_size, head_major=head_major,
              dtype=dtype, prefix=150, seed=q_heads + dim)
    out, lse = attend(c, return_lse=True)
    c.check(out, lse)


@pytest.mark.parametrize("prefix", [0, 1, 15, 127, 128, 129, 255, 1000])
@pytest.mark.parametrize("q_lens,own", [([1, 1, 1], [1, 129, 0]), ([5, 0, 130], [127, 50, 130]), ([300], [300]), ([2, 3], [1, 2]),
                                         ([1] * 150, [(i * 13) % 70 for i in range(150)])])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_lengths_and_masks(prefix, q_lens, own, causal):
    c = Batch(q_lens, own, prefix=prefix, dim=64, seed=prefix + len(own), poison=True, pad=2, first=1)
    keep = torch.full_like(c.q, 5.0)
    out, lse = attend(c, causal=causal, out=keep, return_lse=True)
    c.check(out, lse, causal=causal)
    _, _, _, _, own_rows = c.attend(causal=causal)
    assert (out[~own_rows] == 5.0).all(), "rows of nobody were written"


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_more_sequences_than_threads(dtype):
    """Every CTA sums all sequences' tiles: some thread has several, many have none; empty sequences among them."""
    n = 900
    c = Batch([(i * 5) % 2 for i in range(n)], [(i * 7) % 9 for i in range(n)], q_heads=2, kv_heads=1, dim=64, prefix=40, page_size=8, dtype=dtype,
              seed=19)
    out, lse = attend(c, return_lse=True)
    c.check(out, lse)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_long(dtype):
    c = Batch([1, 1, 2], [5000, 3, 9000], q_heads=8, kv_heads=2, dim=128, prefix=7000, dtype=dtype, seed=20)
    out, lse = attend(c, return_lse=True)
    c.check(out, lse)


@pytest.mark.parametrize("q_heads,kv_heads,dim", [(6, 2, 64), (1, 1, 128)])
def test_attention_many_tokens_without_a_prefix(q_heads, kv_heads, dim):
    """Enough rows that the joining warps take a token each; rows that see nothing, rows of nobody, heads that are no
    multiple of four, texts that end inside a row tile."""
    c = Batch([3901, 0, 130, 70, 5], [3901, 9, 700, 33, 0], q_heads=q_heads, kv_heads=kv_heads, dim=dim, prefix=0, pad=3, first=2, seed=55)
    out = torch.full_like(c.q, 7.0)
    _, lse = attend(c, out=out, return_lse=True)
    assert c.tokens >= 4096 and (out[:2] == 7).all() and (out[-3:] == 7).all()
    c.check(out, lse)


def test_attention_wide_batches_behind_a_prefix():
    c = Batch([1] * 200, [(i * 7) % 40 + 1 for i in range(200)], q_heads=8, kv_heads=2, dim=128, prefix=600, dtype=torch.bfloat16, seed=21)
    c.check(attend(c))
    c = Batch([70, 129, 1, 256], [70, 200, 9, 300], q_heads=4, kv_heads=2, dim=128, prefix=520, seed=22)
    c.check(attend(c))


@pytest.mark.parametrize("spread", [0.0, 6.0, 40.0])
def test_attention_flat_and_sharp_scores(spread):
    """Equal scores; one key that takes everything; scores of thousands, whose maximum moves from tile to tile."""
    c = Batch([1, 40], [700, 400], prefix=500, dim=64, spread=spread, seed=23)
    out, lse = attend(c, return_lse=True)
    c.check(out, lse)


def test_attention_rising_scores():
    """Every tile holds a new maximum, so every tile's sums have to be taken to the new base."""
    c = Batch([1, 3], [900, 600], q_heads=2, kv_heads=1, prefix=800, dim=64, seed=24)
    c.q.fill_(1.0)
    ramp = torch.arange(c.pages * c.page_size, device="cuda").view(c.pages, c.page_size, 1, 1)
    c.prefix_table.copy_(torch.arange(len(c.prefix_table)))
    at = len(c.prefix_table)
    for b, n in enumerate(c.own):
        m = -(-n // c.page_size)
        c.table[b, :m] = torch.arange(at, at + m)
        at += m
    c.k_cache.copy_((ramp * 0.05).expand_as(c.k_cache))
    out, lse = attend(c, return_lse=True)
    c.check(out, lse)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_attention_scale(scale):
    c = Batch([3, 1], [60, 200], prefix=70, seed=25)
    c.check(attend(c, scale=scale), scale=scale)


def test_attention_strided_operands_and_separate_prefix():
    c = Batch([3, 1], [60, 200], prefix=70, seed=26, row_pad=8, dim=64)
    wide = torch.zeros(c.tokens, 3 * c.q_heads, 64, dtype=c.dtype, device="cuda")
    out = wide[:, c.q_heads:2 * c.q_heads]
    attend(c, out=out)
    c.check(out)
    assert (wide[:, :c.q_heads] == 0).all() and (wide[:, 2 * c.q_heads:] == 0).all()
    other = Batch([3, 1], [60, 200], prefix=70, seed=27, page_size=32)
    # the prefix in other memory, of another page size
    pk, pv = other.k_cache, other.v_cache
    got = kv_cache.prefix_attention(c.q, c.k_cache, c.v_cache, c.table, c.lens, c.cu_q, max_q=3, prefix_table=other.prefix_table,
                                    prefix_len=70, prefix_k=pk, prefix_v=pv)
    # the reference takes one page size: lay the prefix out again
    jp = torch.arange(70, device="cuda")
    flat_k = pk[other.prefix_table.long()[jp // 32], jp % 32]
    flat_v = pv[other.prefix_table.long()[jp // 32], jp % 32]
    k16, v16 = torch.zeros_like(c.k_cache), torch.zeros_like(c.v_cache)
    k16[c.prefix_table.long()[jp // 16], jp % 16] = flat_k
    v16[c.prefix_table.long()[jp // 16], jp % 16] = flat_v
    c.check(got, prefix_k=k16, prefix_v=v16)


@pytest.mark.parametrize("offset", [1, 2, 4])
def test_attention_unaligned_operands(offset):
    c = Batch([3, 1], [60, 200], prefix=70, seed=28, dim=64)
    n = c.q.numel()
    buf = torch.zeros(n + offset, dtype=c.dtype, device="cuda")
    q = buf[offset:].view(c.q.shape)
    q.copy_(c.q)
    c.q = q
    out = torch.zeros(n + offset, dtype=c.dtype, device="cuda")[offset:].view(q.shape)
    c.check(attend(c, out=out))


def test_attention_is_the_same_on_every_call():
    c = Batch([1] * 20 + [90], [400 + 3 * i for i in range(20)] + [500], prefix=1500, dim=128, q_heads=8, kv_heads=2, seed=29)
    first = attend(c)
    for _ in range(5):
        assert torch.equal(attend(c), first)


def test_attention_page_outside_the_cache_is_recorded():
    c = Batch([1, 1, 1], [50, 60, 70], prefix=40, seed=30)
    good = attend(c)
    for wrong in (c.pages, -1, 2**31 - 1, -2**31):
        table = c.table.clone()
        table[1, 1] = wrong
        got = kv_cache.prefix_attention(c.q, c.k_cache, c.v_cache, table, c.lens, c.cu_q, max_q=1, prefix_table=c.prefix_table, prefix_len=40)
        assert kv_cache.kv_status(0, clear=True) == kv_cache.BAD_PAGE
        assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
        prefix = c.prefix_table.clone()
        prefix[1] = wrong
        kv_cache.prefix_attention(c.q, c.k_cache, c.v_cache, c.table, c.lens, c.cu_q, max_q=1, prefix_table=prefix, prefix_len=40)
        assert kv_cache.kv_status(0, clear=True) == kv_cache.BAD_PAGE


def test_attention_more_rows_than_max_q_is_recorded():
    c = Batch([1, 4, 1], [50, 60, 70], prefix=40, seed=31)
    good = attend(c)
    got = attend(c, max_q=3)
    assert kv_cache.kv_status(0, clear=True) == kv_cache.BAD_ROWS
    assert torch.equal(got[0], good[0]) and torch.equal(got[5], good[5])


def test_nothing_to_do():
    c = Batch([], [], seed=32)
    assert attend(c).shape == (0, 4, 64)
    kv_cache.kv_append(c.k_cache, c.v_cache, c.k, c.v, c.table, c.lens, c.cu_q)
    c = Batch([0, 0], [0, 0], pad=4, seed=33, prefix=10)
    out = torch.full_like(c.q, 3.0)
    assert (attend(c, out=out) == 3.0).all()


def test_cache_beyond_32_bit_offsets():
    pages, ps, heads, dim = 36000, 64, 8, 128            # 4.7 GB each for keys and values
    c = Batch([1, 5], [100, 70], q_heads=8, kv_heads=heads, dim=dim, page_size=ps, prefix=200, dtype=torch.bfloat16, seed=34)
    k = torch.empty(pages, ps, heads, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    far = pages - c.pages
    k[far:], v[far:] = c.k_cache, c.v_cache
    c.k_cache, c.v_cache, c.pages = k, v, pages
    c.table = torch.where(c.table >= 0, c.table + far, c.table)
    c.prefix_table = c.prefix_table + far
    freq = kv_cache.rope_frequencies(128)
    kv_cache.kv_append(k, v, c.k, c.v, c.table, c.lens, c.cu_q, inv_freq=freq, position_offset=200)
    ref, tol = rotated(c.k[0], 200 + 99, freq, False)
    page = int(c.table[0, 1])
    assert page * ps * heads * dim * 2 > 1 << 32
    assert ((k[page, 35].double() - ref).abs() <= tol).all() and torch.equal(v[page, 35], c.v[0])
    c.check(attend(c))


# ------------------------------------------------------------------------------- a run

def test_generating_with_both_together():
    """A batch takes in a chunk and then generates, every step appending and attending; the reference keeps its
    own 64-bit copy of everything rotated so far."""
    prefix, heads, kvh, dim, ps = 83, 4, 2, 64, 16
    lens = [20, 1, 50]
    steps = [[20, 1, 50], [1, 1, 1], [1, 0, 1], [3, 2, 1], [1, 1, 1]]
    total = [sum(s[b] for s in steps) for b in range(3)]
    c = Batch([0, 0, 0], total, q_heads=heads, kv_heads=kvh, dim=dim, page_size=ps, prefix=prefix, seed=40, poison=True)
    c.v_cache[torch.isnan(c.v_cache) | torch.isinf(c.v_cache)] = 1.0
    freq = kv_cache.rope_frequencies(dim)
    have = [0, 0, 0]
    g = torch.Generator(device="cuda").manual_seed(41)
    for new in steps:
        have = [h + n for h, n in zip(have, new)]
        t = sum(new)
        c.q_lens, c.own, c.tokens, c.first = new, have, t, 0
        c.lens = torch.tensor(have, dtype=torch.int32, device="cuda")
        c.cu_q = torch.tensor([0] + list(itertools.accumulate(new)), dtype=torch.int32, device="cuda")
        qkv = torch.randn(t, heads + 2 * kvh, dim, generator=g, device="cuda").half()
        k, v = qkv[:, heads:heads + kvh], qkv[:, heads + kvh:]
        q = kv_cache.kv_append(c.k_cache, c.v_cache, k, v, c.table, c.lens, c.cu_q, inv_freq=freq, position_offset=prefix, q=qkv[:, :heads])
        out, lse = kv_cache.prefix_attention(q, c.k_cache, c.v_cache, c.table, c.lens, c.cu_q, max_q=max(new), prefix_table=c.prefix_table,
                                             prefix_len=prefix, return_lse=True)
        c.check(out, lse, q=q)


def test_captured_steps_follow_the_tables():
    c = Batch([1, 1, 1], [300, 300, 300], prefix=200, dim=128, q_heads=8, kv_heads=2, seed=42)
    freq = kv_cache.rope_frequencies(128)
    outs = []

    def step():
        q = kv_cache.kv_append(c.k_cache, c.v_cache, c.k, c.v, c.table, c.lens, c.cu_q, inv_freq=freq, position_offset=200, q=c.q,
                               q_out=torch.zeros_like(c.q))
        return q, kv_cache.prefix_attention(q, c.k_cache, c.v_cache, c.table, c.lens, c.cu_q, max_q=1, prefix_table=c.prefix_table,
                                            prefix_len=200)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(step())
    for own in ([1, 1, 1], [5, 299, 0], [300, 17, 128]):
        c.lens.copy_(torch.tensor(own, dtype=torch.int32))
        for gr, (q, out) in zip(graphs, outs):
            out.fill_(9.0)
            gr.replay()
            torch.cuda.synchronize()
            c.own = own
            ref = step()
            assert torch.equal(out, ref[1])
            c.check(out, q=q)


def test_whole_path_on_another_stream():
    """Tables, inputs and calls on a stream of the caller's, nothing on the default one."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c = Batch([1, 30, 1], [200, 30, 77], prefix=140, dim=128, q_heads=8, kv_heads=2, seed=43)
        q = kv_cache.kv_append(c.k_cache, c.v_cache, c.k, c.v, c.table, c.lens, c.cu_q, inv_freq=kv_cache.rope_frequencies(128),
                               position_offset=140, q=c.q)
        out, lse = kv_cache.prefix_attention(q, c.k_cache, c.v_cache, c.table, c.lens, c.cu_q, max_q=30, prefix_table=c.prefix_table,
                                             prefix_len=140, return_lse=True)
    side.synchronize()
    c.check(out, lse, q=q)


def test_given_workspace():
    c = Batch([1] * 5, [300 + i for i in range(5)], prefix=700, dim=128, q_heads=8, kv_heads=2, seed=44)
    want = attend(c)
    for size, ok in ((64 << 20, True), (256, False)):
        ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
        if ok:
            assert torch.equal(attend(c, workspace=ws), want)        # whatever it holds
            assert torch.equal(attend(c, workspace=ws), want)
            with pytest.raises(SwapError):
                attend(c, workspace=ws[64:])                          # not 256-byte aligned
        else:
            with pytest.raises(ValueError):
                attend(c, workspace=ws)


def test_not_a_number_in_a_visible_key_shows():
    """Nothing is swept under: a NaN or an infinity among the keys or values a row sees leaves that row not finite,
    and rows of other sequences as they were."""
    for what in ("k_cache", "v_cache"):
        for bad in (math.nan, math.inf):
            c = Batch([1, 1, 1], [200, 190, 77], prefix=140, dim=64, seed=45)
            good = attend(c)
            getattr(c, what)[int(c.table[1, 3]), 5] = bad
            out = attend(c)
            assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
            assert not torch.isfinite(out[1]).all()


def test_calls_on_two_streams_at_once():
    cases = [Batch([1] * 30, [200 + i for i in range(30)], prefix=900, dim=128, q_heads=8, kv_heads=2, seed=50 + i) for i in range(2)]
    want = [attend(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(attend(c))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_refusals_on_device_tensors():
    c = Batch([1, 1], [5, 6], seed=60, prefix=20)
    args = (c.k_cache, c.v_cache, c.k, c.v, c.table, c.lens, c.cu_q)
    for bad in [dict(q_out=c.q), dict(inv_freq=torch.zeros(4, device="cuda")), dict(position_offset=-1), dict(position_offset=1 << 32),
                dict(inv_freq=torch.zeros(40, dtype=torch.float64, device="cuda")), dict(q=c.q[:1]), dict(q=c.q.float())]:
        with pytest.raises((ValueError, SwapError)):
            kv_cache.kv_append(*args, **bad)
    for i, wrong in [(0, c.k_cache[..., :32]), (2, c.k.cpu()), (2, c.k.double()), (3, c.v[:1]), (4, c.table.long()), (5, c.lens[:1]),
                     (6, c.cu_q.cpu()), (0, c.k_cache.transpose(2, 3)), (0, c.k_cache[:, :, :1].expand_as(c.k_cache))]:
        with pytest.raises((ValueError, SwapError)):
            kv_cache.kv_append(*(wrong if j == i else a for j, a in enumerate(args)))
    for bad in [dict(prefix_len=-1), dict(prefix_len=20, prefix_table=None), dict(prefix_len=500, prefix_table=c.prefix_table),
                dict(scale=math.inf), dict(scale=math.nan), dict(out=c.q[:, :1]), dict(out=c.q[:1].expand_as(c.q)), dict(max_q=-1),
                dict(prefix_len=20, prefix_table=c.prefix_table, prefix_k=c.k_cache)]:
        with pytest.raises((ValueError, SwapError)):
            kv_cache.prefix_attention(c.q, c.k_cache, c.v_cache, c.table, c.lens, c.cu_q, **bad)
    with pytest.raises((ValueError, SwapError)):
        kv_cache.prefix_attention(c.q[:, :3], c.k_cache, c.v_cache, c.table, c.lens, c.cu_q)
    with pytest.raises((ValueError, SwapError)):
        kv_cache.prefix_attention(c.q.cpu(), c.k_cache.cpu(), c.v_cache.cpu(), c.table.cpu(), c.lens.cpu(), c.cu_q.cpu())
    a = _cabi.KvAppendArgs()
    a.dtype = 9
    assert _cabi.lib().tsw_kv_append(0, a, None) == _cabi.ERR_INVALID


def test_numbers_that_the_c_structures_would_cut_are_refused():
    c = Batch([1], [4], prefix=16)
    for offset in (-1, 1 << 32, (1 << 64) + 3):
        with pytest.raises(ValueError, match="position_offset"):
            kv_cache.kv_append(c.k_cache, c.v_cache, c.k, c.v, c.table, c.lens, c.cu_q, position_offset=offset)
    for length in (-1, 0x7fffff01, (1 << 32) + 16):
        with pytest.raises(ValueError, match="prefix_len"):
            kv_cache.prefix_attention(c.q, c.k_cache, c.v_cache, c.table, c.lens, c.cu_q, prefix_table=c.prefix_table, prefix_len=length)


FIRST_CALL = """
import sys
sys.path[:0] = [{tests!r}, {root!r}]
import torch
from kv_cases import Batch
from torpor_b200 import kv_cache
c = Batch([1, 3], [40, 200], prefix=130, dim={dim}, seed=77)
cache = c.k_cache.clone(), c.v_cache.clone()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    q = kv_cache.kv_append(*cache, c.k, c.v, c.table, c.lens, c.cu_q, q=c.q)
    out = kv_cache.prefix_attention(q, c.k_cache, c.v_cache, c.table, c.lens, c.cu_q, max_q=3, prefix_table=c.prefix_table, prefix_len=130)
graph.replay()
torch.cuda.synchronize()
c.check(out, q=q)
assert kv_cache.kv_status(0) == 0
print("captured")
"""


@pytest.mark.parametrize("dim", [64, 128, 200])
def test_a_process_may_capture_its_first_call(dim):
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(tests=here, root=os.path.dirname(here), dim=dim)], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "captured", r.stderr[-2000:]
