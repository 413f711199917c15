"""Inputs and 64-bit reference of the key/value cache operators, for tests."""
import math

import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}      # half a rounding step, relative


class Batch:
    """Random tensors of one call.  ``q_lens`` and ``own`` are per sequence; ``pad`` rows belong to nobody."""

    def __init__(self, q_lens, own, *, q_heads=4, kv_heads=2, dim=64, page_size=16, prefix=0, dtype=torch.float16, seed=0,
                 head_major=False, pad=0, first=0, device="cuda", poison=False, spread=1.0, row_pad=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.q_lens, self.own, self.prefix, self.page_size = list(q_lens), list(own), prefix, page_size
        self.q_heads, self.kv_heads, self.dim, self.dtype, self.device = q_heads, kv_heads, dim, dtype, device
        self.first, self.batch = first, len(self.own)
        cu = [first]
        for n in self.q_lens:
            cu.append(cu[-1] + n)
        self.tokens = cu[-1] + pad

        def normal(*shape):
            shape = shape[:-1] + (shape[-1] + row_pad,)
            return (torch.randn(*shape, generator=g, device=device) * spread).to(dtype)[..., :shape[-1] - row_pad]

        need = [-(-n // page_size) for n in self.own]
        np_ = -(-prefix // page_size)
        self.pages = sum(need) + np_ + 2
        shape = (self.pages, kv_heads, page_size, dim) if head_major else (self.pages, page_size, kv_heads, dim)
        self.k_cache, self.v_cache = normal(*shape), normal(*shape)
        if head_major:
            self.k_cache, self.v_cache = self.k_cache.transpose(1, 2), self.v_cache.transpose(1, 2)
        order = torch.randperm(self.pages, generator=g, device=device).to(torch.int32)
        self.table = torch.full((self.batch, max(need + [0])), -1, dtype=torch.int32, device=device)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.prefix_table = order[at:at + np_].clone()
        if poison:          # everything behind the last token of its sequence, and pages of nobody
            keep = torch.zeros(self.pages, page_size, dtype=torch.bool, device=device)
            for b, n in enumerate(self.own):
                j = torch.arange(n, device=device)
                keep[self.table[b].long()[j // page_size], j % page_size] = True
            j = torch.arange(prefix, device=device)
            keep[self.prefix_table.long()[j // page_size], j % page_size] = True
            bits = torch.where(torch.rand(self.pages, page_size, generator=g, device=device) < 0.5, float("nan"), float("inf"))
            for cache in (self.k_cache, self.v_cache):
                cache[~keep] = bits[~keep][:, None, None].to(dtype).expand(-1, kv_heads, dim)
        self.q = normal(self.tokens, q_heads, dim)
        self.k, self.v = normal(self.tokens, kv_heads, dim), normal(self.tokens, kv_heads, dim)
        self.lens = torch.tensor(self.own, dtype=torch.int32, device=device)
        self.cu_q = torch.tensor(cu, dtype=torch.int32, device=device)

    def rows(self):
        at = self.first
        for b, n in enumerate(self.q_lens):
            yield b, at, n, self.own[b]
            at += n

    def attend(self, causal=True, scale=None, k_cache=None, v_cache=None, prefix_k=None, prefix_v=None, q=None):
        """Per row in 64 bits: result, log-sum, and the bound on what a kernel with 32-bit sums, 16-bit
        weights and one rounding at the end may be off by (None rows: nobody's)."""
        kc, vc = self.k_cache if k_cache is None else k_cache, self.v_cache if v_cache is None else v_cache
        pk, pv = (kc, vc) if prefix_k is None else (prefix_k, prefix_v)
        q = self.q if q is None else q
        scale = self.dim ** -0.5 if scale is None else scale
        group, u = self.q_heads // self.kv_heads, UNIT[self.dtype]
        out = torch.zeros(self.tokens, self.q_heads, self.dim, dtype=torch.float64, device=self.device)
        tol = torch.zeros_like(out)
        lse = torch.zeros(self.tokens, self.q_heads, dtype=torch.float64, device=self.device)
        lse_tol = torch.zeros_like(lse)
        own_rows = torch.zeros(self.tokens, dtype=torch.bool, device=self.device)
        jp = torch.arange(self.prefix, device=self.device)
        pre = self.prefix_table.long()[jp // self.page_size] if self.prefix else jp
        for b, at, n, length in self.rows():
            j = torch.arange(length, device=self.device)
            page = self.table[b].long()[j // self.page_size] if length else j
            keys = torch.cat((pk[pre, jp % self.page_size], kc[page, j % self.page_size])).double()
            vals = torch.cat((pv[pre, jp % self.page_size], vc[page, j % self.page_size])).double()
            for i in range(n):
                own_rows[at + i] = True
                seen = self.prefix + (max(0, length - n + i + 1) if causal else length)
                if seen == 0:
                    lse[at + i] = -math.inf
                    continue
                k = keys[:seen].repeat_interleave(group, 1)
                v = vals[:seen].repeat_interleave(group, 1)
                prod = q[at + i].double()[None] * k
                s = prod.sum(-1) * scale                                              # [seen, heads]
                l = s.logsumexp(0)
                p = (s - l).exp()
                out[at + i] = torch.einsum("kh,khd->hd", p, v)
                lse[at + i] = l
                # scores: dim products summed in 32 bits, and their scaling; exponentials to 2^-21
                ds = (self.dim + 8) * 2.0 ** -24 * (prod.abs().sum(-1) * abs(scale)).amax(0) + 2.0 ** -21
                mass = torch.einsum("kh,khd->hd", p, v.abs())
                # weights rounded to 16 bits (and, in fp16, to its smallest step), sums over the keys in
                # 32 bits, the result rounded once
                tol[at + i] = u * out[at + i].abs() + mass * (1.01 * u + 2 * ds[:, None] + 2 * seen * 2.0 ** -24)
                if self.dtype is torch.float16:
                    tol[at + i] += seen * 2.0 ** -25 * v.abs().amax(0) + 2.0 ** -25
                lse_tol[at + i] = 2 * ds + 2 * seen * 2.0 ** -24 + 2.0 ** -22 * (1 + l.abs())
        return out, lse, tol, lse_tol, own_rows

    def check(self, got, got_lse=None, **kw):
        out, lse, tol, lse_tol, own_rows = self.attend(**kw)
        diff = (got.double() - out).abs()
        assert torch.isfinite(got[own_rows]).all()
        worst = (diff[own_rows] - tol[own_rows]).max().item() if own_rows.any() else 0.0
        assert worst <= 0, f"off by {diff[own_rows].max().item():.3g}, {worst:.3g} above the bound"
        if got_lse is not None:
            empty = lse == -math.inf
            assert torch.equal(got_lse[own_rows] == -math.inf, empty[own_rows])
            ok = own_rows[:, None] & ~empty
            assert ((got_lse.double() - lse).abs()[ok] <= lse_tol[ok]).all()


def rotated(x, position, inv_freq, interleaved):
    """One token's heads in 64 bits: (values, bound of a kernel that forms angles in 64 bits, sine, cosine
    and products in 32, and rounds once)."""
    u, r = UNIT[x.dtype], 2 * inv_freq.shape[0]
    x = x.double()
    out, tol = x.clone(), torch.zeros_like(x)
    a = position * inv_freq
    c, s = a.cos(), a.sin()
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    out[..., lo] = x[..., lo] * c - x[..., hi] * s
    out[..., hi] = x[..., lo] * s + x[..., hi] * c
    # angle formed by three 64-bit roundings here and there, rounded to 32 bits in half turns (2^-24 pi); sine and
    # cosine to two units, three operations
    slack = (x[..., lo].abs() + x[..., hi].abs()) * (2.0 ** -20 + 6 * 2.0 ** -53 * a.abs())
    tol[..., lo] = u * out[..., lo].abs() + slack * 1.01
    tol[..., hi] = u * out[..., hi].abs() + slack * 1.01
    if u == UNIT[torch.float16]:
        tol[..., :r] += 2.0 ** -25                     # the smallest step of fp16
    return out, tol
