"""Timed cases of the key/value cache operators: appending to a paged cache, and attention over it.

Two operators.  ``append`` rotates the new keys (and queries) by their positions and writes keys and
values into the pages of their sequences.  ``attend`` is the attention of a batch whose sequences share
one prefix: every query sees the prefix and its own sequence's pages.  Sizes are those of the weight sets
in this repository (32 heads of 128 for the 4096-wide set, 16 heads of 64 for the 1024-wide one) or generic.
"""
import math
import random

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _append(name, **kw):
    case = dict(name=name, kind="append", dtype="float16", batch=1, q_heads=32, kv_heads=32, head_dim=128,
                page_size=16, offset=0, q_max=1, own_max=1, ragged=False, head_major=False, rotary=128,
                interleaved=False, fused=False, mix=1)
    case.update(kw)
    return case


def _attend(name, **kw):
    case = dict(name=name, kind="attend", dtype="float16", batch=1, q_heads=32, kv_heads=32, head_dim=128,
                page_size=16, prefix=0, q_max=1, own_max=1, ragged=False, head_major=False, causal=True,
                lse=False, mix=1)
    case.update(kw)
    return case


def listed():
    return [
        # one request generating its next token behind a 512-token prompt: all latency
        _append("append_one_token", offset=512, own_max=1000),
        # a served batch generating, grouped heads, every sequence at a length of its own
        _append("append_batch", dtype="bfloat16", batch=64, kv_heads=8, page_size=32, offset=8192, own_max=4096,
                ragged=True, mix=2),
        # chunks of several requests, heads of 64, pairs side by side, half of each head rotated,
        # queries, keys and values in one projection's output
        _append("append_chunks", dtype="bfloat16", batch=7, q_heads=16, kv_heads=16, head_dim=64, page_size=64,
                q_max=301, own_max=900, ragged=True, rotary=32, interleaved=True, fused=True, mix=3),
        # one long prompt at once, pages stored head by head
        _append("append_prompt", q_max=16384, own_max=16384, head_major=True, fused=True, mix=4),
        # two short requests behind a short prompt: all latency
        _attend("attend_small", dtype="bfloat16", batch=2, q_heads=16, kv_heads=16, head_dim=64, prefix=130,
                own_max=40, ragged=True, mix=5),
        # generating on the 7B set behind its function's prompt
        _attend("attend_decode", batch=32, prefix=2048, own_max=512, ragged=True, mix=6),
        # a large batch with grouped heads behind a long prompt: 512 rows to a key head
        _attend("attend_decode_grouped", dtype="bfloat16", batch=128, kv_heads=8, page_size=64, prefix=8192,
                own_max=1024, ragged=True, mix=7),
        # few requests with long texts of their own behind a short prompt of odd length
        _attend("attend_long_own", dtype="bfloat16", batch=8, kv_heads=8, prefix=777, own_max=32768, ragged=True,
                lse=True, mix=8),
        # ragged chunks of several requests behind a prompt of odd length
        _attend("attend_chunks", batch=6, prefix=4101, q_max=200, own_max=1500, ragged=True, page_size=32, mix=9),
        # queries on an encoder's states of other lengths: no prefix, no order
        _attend("attend_encoder", dtype="bfloat16", batch=16, q_heads=16, kv_heads=16, head_dim=64, page_size=128,
                q_max=60, own_max=512, ragged=True, causal=False, head_major=True, mix=10),
        # one prompt read from its start: causal, nothing shared
        _attend("attend_prompt", dtype="bfloat16", q_max=8192, own_max=8192, page_size=64, mix=11),
        # sixteen requests' first chunks behind a long shared document
        _attend("attend_shared_document", batch=16, prefix=16384, q_max=256, own_max=700, page_size=64,
                lse=True, mix=12),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    top = {"append": work(listed()[3]), "attend": work(listed()[11])}
    kind = rng.choice(["append", "attend"])
    while True:
        kv_heads, group = rng.choice([(32, 1), (16, 1), (8, 4), (8, 1), (4, 7), (2, 8), (1, 16), (12, 1), (6, 2)])
        dim = rng.choice([64, 128, 64, 128, 80, 96])
        q_max = rng.choice([1, 1, _spread(rng, 2, 2000)])
        common = dict(dtype=rng.choice(["float16", "bfloat16"]), batch=_spread(rng, 1, 160), q_heads=kv_heads * group,
                      kv_heads=kv_heads, head_dim=dim, page_size=rng.choice([8, 16, 32, 64, 128, 256]),
                      q_max=q_max, own_max=q_max + _spread(rng, 1, 20000) - 1, ragged=rng.random() < 0.75,
                      head_major=rng.random() < 0.4, mix=rng.randrange(1 << 30))
        if kind == "append":
            case = _append("", offset=_spread(rng, 1, 200000) - 1, rotary=rng.choice([dim, dim, dim // 2]),
                           interleaved=rng.random() < 0.4, fused=rng.random() < 0.5, **common)
        else:
            case = _attend("", prefix=rng.choice([0, _spread(rng, 1, 20000), _spread(rng, 1, 20000)]),
                           causal=rng.random() < 0.8, lse=rng.random() < 0.4, **common)
        del case["name"]
        w, t, b = work(case), top[kind], _cache_bytes(case)
        # keep the plain form's scores and the cache within what the largest listed case needs
        if w["flops"] <= t["flops"] and w["bytes"] <= t["bytes"] and b <= 3 << 30 and _scores(case) <= 3 << 30:
            return case


def _lengths(case):
    """New tokens and own lengths (new ones included) of every sequence: from the case alone."""
    rng = random.Random(case["mix"])
    q, n = [], []
    for _ in range(case["batch"]):
        ql = rng.randint(1, case["q_max"]) if case["ragged"] else case["q_max"]
        top = max(ql, case["own_max"])
        q.append(ql)
        n.append(rng.randint(ql, top) if case["ragged"] else top)
    return q, n


def _pages(case):
    q, n = _lengths(case)
    ps = case["page_size"]
    own_pages = [-(-x // ps) for x in n]
    prefix_pages = -(-case.get("prefix", 0) // ps)
    return own_pages, prefix_pages


def _cache_bytes(case):
    own_pages, prefix_pages = _pages(case)
    return 4 * (sum(own_pages) + prefix_pages) * case["page_size"] * case["kv_heads"] * case["head_dim"]


def _scores(case):
    q, n = _lengths(case)
    if case["kind"] == "append":
        return 0
    return 4 * case["q_heads"] * (sum(q) * case["prefix"] + case["batch"] * max(q) * max(n))


def work(case):
    q, n = _lengths(case)
    d, hq, hkv, t = case["head_dim"], case["q_heads"], case["kv_heads"], sum(q)
    own_pages, prefix_pages = _pages(case)
    tables = 4 * (sum(own_pages) + prefix_pages + 2 * case["batch"] + 1)
    if case["kind"] == "append":
        # queries read and written, keys and values read and written; six operations for each rotated pair
        return {"bytes": 2 * t * d * 2 * (hq + 2 * hkv) + tables + 4 * case["rotary"],
                "flops": 3 * t * case["rotary"] * (hq + hkv)}
    keys = sum(n) + case["prefix"]
    seen = t * case["prefix"]
    for ql, nl in zip(q, n):
        seen += ql * (nl - ql) + ql * (ql + 1) // 2 if case["causal"] else ql * nl
    return {"bytes": 2 * (2 * t * hq * d + 2 * keys * hkv * d) + tables + (4 * t * hq if case["lse"] else 0),
            "flops": 4 * d * hq * seen}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    q_lens, own = _lengths(case)
    own_pages, prefix_pages = _pages(case)
    ps, hq, hkv, d = case["page_size"], case["q_heads"], case["kv_heads"], case["head_dim"]
    n_pages = sum(own_pages) + prefix_pages + 3                      # three pages belong to nobody

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    shape = (n_pages, hkv, ps, d) if case["head_major"] else (n_pages, ps, hkv, d)
    k_cache, v_cache = normal(*shape), normal(*shape)
    if case["head_major"]:
        k_cache, v_cache = k_cache.transpose(1, 2), v_cache.transpose(1, 2)
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["batch"], max(own_pages)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, m in enumerate(own_pages):
        table[b, :m] = order[at:at + m]
        at += m
    cu_q = [0]
    for x in q_lens:
        cu_q.append(cu_q[-1] + x)
    state = {"case": case, "k_cache": k_cache, "v_cache": v_cache, "table": table,
             "lens": torch.tensor(own, dtype=torch.int32, device="cuda"),
             "cu_q": torch.tensor(cu_q, dtype=torch.int32, device="cuda"), "q_lens": q_lens, "own": own}
    t = cu_q[-1]
    if case["kind"] == "append":
        if case["fused"]:
            qkv = normal(t, hq + 2 * hkv, d)
            state["q"], state["k"], state["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        else:
            state["q"], state["k"], state["v"] = normal(t, hq, d), normal(t, hkv, d), normal(t, hkv, d)
        r = case["rotary"]
        state["inv_freq"] = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    else:
        state["q"] = normal(t, hq, d)
        state["prefix_table"] = order[at:at + prefix_pages].clone() if prefix_pages else None
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from torpor_b200 import kv_cache
    case = state["case"]
    if case["kind"] == "append":
        q_out = kv_cache.kv_append(state["k_cache"], state["v_cache"], state["k"], state["v"], state["table"],
                                   state["lens"], state["cu_q"], inv_freq=state["inv_freq"],
                                   interleaved=case["interleaved"], position_offset=case["offset"], q=state["q"])
        return q_out, state["k_cache"], state["v_cache"]
    return kv_cache.prefix_attention(state["q"], state["k_cache"], state["v_cache"], state["table"], state["lens"],
                                     state["cu_q"], max_q=max(state["q_lens"]), prefix_table=state["prefix_table"],
                                     prefix_len=case["prefix"], causal=case["causal"], return_lse=case["lse"])


def _token_index(state):
    """Sequence, own index of every new token."""
    cu = state["cu_q"].long()
    t = torch.arange(state["q"].shape[0], device="cuda")
    b = torch.bucketize(t, cu[1:], right=True)
    return b, state["lens"].long()[b] - (cu[b + 1] - t)


def _rotate(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    y = x.clone()
    c, s = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * c - b * s, a * s + b * c
    return y


def _run_plain(state):
    case = state["case"]
    if case["kind"] == "append":
        b, j = _token_index(state)
        angle = (j + case["offset"]).double()[:, None] * state["inv_freq"]     # far positions: 64 bits
        cos, sin = angle.cos().float(), angle.sin().float()
        q = _rotate(state["q"].float(), cos, sin, case["interleaved"])
        k = _rotate(state["k"].float(), cos, sin, case["interleaved"])
        page = state["table"][b, j // case["page_size"]].long()
        at = j % case["page_size"]
        state["k_cache"][page, at] = k.to(state["k_cache"].dtype)
        state["v_cache"][page, at] = state["v"].to(state["v_cache"].dtype)
        return q.to(state["q"].dtype), state["k_cache"], state["v_cache"]
    return _attend_plain(state)


def _attend_plain(state):
    case = state["case"]
    hkv, d, p = case["kv_heads"], case["head_dim"], case["prefix"]
    group = case["q_heads"] // hkv
    q = state["q"].float()
    t, batch, width = q.shape[0], case["batch"], max(state["q_lens"])
    b, j = _token_index(state)
    i = torch.arange(t, device="cuda") - state["cu_q"].long()[b]               # place among the sequence's new tokens
    q = q.view(t, hkv, group, d) / math.sqrt(d)
    n_max = max(state["own"])
    # own part: queries padded to the longest sequence's, keys gathered from the pages
    padded = q.new_zeros(batch, width, hkv, group, d)
    padded[b, i] = q
    table = state["table"].long().clamp(min=0)

    def gather(cache):
        return cache[table].reshape(batch, -1, hkv, d)[:, :n_max].permute(0, 2, 3, 1)   # sequence, head, dim, key

    rows = padded.permute(0, 2, 3, 1, 4).reshape(batch, hkv, group * width, d)
    s_own = torch.matmul(rows, gather(state["k_cache"]).float()).view(batch, hkv, group, width, n_max)
    key = torch.arange(n_max, device="cuda")
    lens, cu = state["lens"].long(), state["cu_q"].long()
    if case["causal"]:
        last = (lens - (cu[1:] - cu[:-1]))[:, None] + torch.arange(width, device="cuda")
        hidden = key > last.clamp(max=n_max)[:, :, None]
    else:
        hidden = (key >= lens[:, None])[:, None, :].expand(batch, width, n_max)
    s_own = s_own.masked_fill(hidden[:, None, None], float("-inf"))
    top = s_own.amax(-1)                                                        # sequence, head, group, place
    if p:
        pk = state["k_cache"][state["prefix_table"].long()].reshape(-1, hkv, d)[:p].permute(1, 2, 0).float()
        pv = state["v_cache"][state["prefix_table"].long()].reshape(-1, hkv, d)[:p].permute(1, 0, 2).float()
        s_pre = torch.matmul(q.permute(1, 0, 2, 3).reshape(hkv, t * group, d), pk).view(hkv, t, group, p)
        top_pre = s_pre.amax(-1)                                                # head, token, group
        top[b, :, :, i] = torch.maximum(top[b, :, :, i], top_pre.permute(1, 0, 2))
    top = top.clamp(min=torch.finfo(torch.float32).min)                         # padded places
    e = (s_own - top[..., None]).exp()
    del s_own
    total = e.sum(-1)
    out = torch.matmul(e.view(batch, hkv, group * width, n_max), gather(state["v_cache"]).float().transpose(-1, -2))
    out = out.view(batch, hkv, group, width, d)[b, :, :, i]                     # token, head, group, dim
    total, top = total[b, :, :, i], top[b, :, :, i]
    if p:
        e = (s_pre - top.permute(1, 0, 2)[..., None]).exp()
        del s_pre
        total = total + e.sum(-1).permute(1, 0, 2)
        out = out + torch.matmul(e.view(hkv, t * group, p), pv).view(hkv, t, group, d).permute(1, 0, 2, 3)
    out = (out / total[..., None]).reshape(t, case["q_heads"], d).to(state["q"].dtype)
    if case["lse"]:
        return out, (top + total.log()).reshape(t, case["q_heads"])
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_append(case, state) if case["kind"] == "append" else _exact_attend(case, state)


def _exact_append(case, state):
    ps, r, off = case["page_size"], case["rotary"], case["offset"]
    k_out, v_out = state["k_cache"].double(), state["v_cache"].double()
    q_out = torch.empty_like(state["q"], dtype=torch.float64)
    theta = [10000.0 ** (-2.0 * c / r) for c in range(r // 2)]
    theta = torch.tensor(theta, dtype=torch.float64, device="cuda")
    first = 0
    for b, (ql, nl) in enumerate(zip(state["q_lens"], state["own"])):
        j = torch.arange(nl - ql, nl, device="cuda")
        turn = torch.polar(torch.ones(ql, r // 2, dtype=torch.float64, device="cuda"), (j + off).double()[:, None] * theta)
        pages = state["table"][b].long()[j // ps]
        for src, dst in (("q", q_out), ("k", None)):
            x = state[src][first:first + ql].double()
            if case["interleaved"]:
                z = torch.complex(x[..., 0:r:2].contiguous(), x[..., 1:r:2].contiguous()) * turn[:, None]
                turned = torch.stack((z.real, z.imag), dim=-1).flatten(-2)
            else:
                z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn[:, None]
                turned = torch.cat((z.real, z.imag), dim=-1)
            x = torch.cat((turned, x[..., r:]), dim=-1)
            if dst is not None:
                dst[first:first + ql] = x
            else:
                k_out[pages, j % ps] = x
        v_out[pages, j % ps] = state["v"][first:first + ql].double()
        first += ql
    return q_out, k_out, v_out


def _exact_attend(case, state):
    ps, p, d = case["page_size"], case["prefix"], case["head_dim"]
    group = case["q_heads"] // case["kv_heads"]
    pre = torch.arange(p, device="cuda")
    outs, lses = [], []
    first = 0
    for b, (ql, nl) in enumerate(zip(state["q_lens"], state["own"])):
        j = torch.arange(nl, device="cuda")
        page, at = state["table"][b].long()[j // ps], j % ps
        if p:
            page = torch.cat((state["prefix_table"].long()[pre // ps], page))
            at = torch.cat((pre % ps, at))
        keys, values = state["k_cache"][page, at].double(), state["v_cache"][page, at].double()   # key, head, dim
        step = max(1, (1 << 28) // (case["q_heads"] * (p + nl)))
        for lo in range(0, ql, step):
            hi = min(ql, lo + step)
            q = state["q"][first + lo:first + hi].double().unflatten(1, (case["kv_heads"], group))
            s = torch.einsum("thgd,khd->thgk", q, keys) * (1.0 / math.sqrt(d))
            if case["causal"]:
                bound = p + nl - ql + torch.arange(lo, hi, device="cuda")
                s[(torch.arange(p + nl, device="cuda") > bound[:, None])[:, None, None].expand_as(s)] = -math.inf
            lse = s.logsumexp(-1, keepdim=True)
            outs.append(torch.einsum("thgk,khd->thgd", (s - lse).exp(), values).flatten(1, 2))
            lses.append(lse.squeeze(-1).flatten(1))
        first += ql
    out = torch.cat(outs)
    return (out, torch.cat(lses)) if case["lse"] else out
