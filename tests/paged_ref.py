"""The paged cache's operators from their definitions, in 64 bits.

Written apart from the package: sequences one by one, pages by plain indexing.
Used by the paged GPU tests, which build batches with :class:`Batch`.
"""
import math
import random

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a step, relative
F32 = 2.0 ** -24
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(x):
    """``(codes, scales)`` of float64 ``[..., D]``: per 32 values the least 2^e
    (-23 <= e <= 13) with 6 * 2^e at least all of them, nearest E2M1 numbers, ties
    to the even code; a group with a non-finite value: byte 255, codes 0."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    odd = ~torch.isfinite(g).all(-1, keepdim=True)
    e = torch.full_like(top, -23)
    for i in range(-23, 13):
        e = torch.where(top > 6 * 2.0 ** i, torch.full_like(e, i + 1), e)
    a = (g.abs() / torch.exp2(e)).clamp(max=6.0)
    a = torch.where(odd, torch.zeros_like(a), a)
    lo = torch.searchsorted(E2M1.to(x.device), a.contiguous(), right=True).clamp(max=7) - 1
    lo = lo.clamp(0, 6)
    level = E2M1.to(x.device)
    below, above = a - level[lo], level[lo + 1] - a
    code = torch.where((above < below) | ((above == below) & (lo % 2 == 1)), lo + 1, lo)
    code = torch.where(odd, torch.zeros_like(code), code + 8 * torch.signbit(g).long()).flatten(-2)
    scale = torch.where(odd, torch.full_like(e, 255), e + 127)[..., 0]
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8), scale.to(torch.uint8)


def dequantize(codes, scales):
    c = codes.long()
    v = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    x = E2M1.to(codes.device)[v & 7] * torch.where(v >= 8, -1.0, 1.0)
    s = torch.where(scales == 255, float("nan"), torch.exp2(scales.double() - 127))
    return x * s.repeat_interleave(32, -1)


def rotate(x, cos, sin, interleaved):
    """float64 ``x [n, heads, D]`` with angle rows ``[n, rot / 2]``."""
    half = cos.shape[1]
    i = torch.arange(half, device=x.device)
    i, j = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s, y = cos.double()[:, None], sin.double()[:, None], x.double().clone()
    a, b = x[..., i].double(), x[..., j].double()
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    return y


class Batch:
    """Sequences ``[(new, cached with them), ...]`` over a shuffled pool of pages.

    Slots that no sequence covers, and the spare pages, hold NaN: nothing may read
    them into a result.  ``tail`` rows behind the last sequence."""

    def __init__(self, dev, seqs, D, H, Hkv, page, dtype, bits=16, layout="heads", tail=0, spare=2, seed=0, gain=1.0,
                 extra_columns=0):
        import longvideosparseattention_amd as lv

        self.seqs, self.D, self.H, self.Hkv, self.ps, self.dtype, self.bits = seqs, D, H, Hkv, page, dtype, bits
        self.dev, r = dev, random.Random(seed)
        self.gen = torch.Generator().manual_seed(seed)
        counts = [-(-L // page) for _, L in seqs]
        P = sum(counts) + spare
        order = list(range(P))
        r.shuffle(order)
        self.table = torch.full((len(seqs), max(counts + [0]) + extra_columns), -7, dtype=torch.int32)
        self.pages, at = [], 0
        for b, c in enumerate(counts):
            self.pages.append(order[at:at + c])
            self.table[b, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
            at += c
        ends = [0]
        for n, _ in seqs:
            ends.append(ends[-1] + n)
        self.n_rows, self.N = ends[-1], ends[-1] + tail
        self.ends = ends
        self.cu = torch.tensor(ends, dtype=torch.int32, device=dev)
        self.lens = torch.tensor([L for _, L in seqs], dtype=torch.int32, device=dev)
        self.table_dev = self.table.to(dev)
        self.K = [gain * torch.randn(L, Hkv, D, generator=self.gen) for _, L in seqs]   # values of each sequence
        self.V = [torch.randn(L, Hkv, D, generator=self.gen) for _, L in seqs]
        shape = (P, Hkv, page) if layout == "heads" else (P, page, Hkv)

        def rows(width, dt, fill):
            t = torch.full((*shape, width), fill, dtype=dt)
            return (t.transpose(1, 2) if layout == "heads" else t)

        if bits == 16:
            parts = [rows(D, dtype, float("nan")), rows(D, dtype, float("nan"))]
        else:
            parts = [rows(D // 2, torch.uint8, 0x77), rows(D // 2, torch.uint8, 0x77),
                     rows(D // 32, torch.uint8, 255), rows(D // 32, torch.uint8, 255)]
        for b, (_, L) in enumerate(seqs):
            for t, src in ((0, self.K), (1, self.V)):
                if bits == 16:
                    src[b] = src[b].to(dtype).double()
                    self._put(parts[t], b, src[b].to(dtype))
                else:
                    c, s = quantize(src[b].to(dtype).double())
                    src[b] = dequantize(c, s)
                    self._put(parts[t], b, c)
                    self._put(parts[t + 2], b, s)
        to = [torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev).copy_(t) for t in parts]
        self.cache = lv.PagedKVCache(*to)

    def _put(self, where, b, rows):
        for i, page in enumerate(self.pages[b]):
            part = rows[i * self.ps:(i + 1) * self.ps]
            where[page, :part.shape[0]] = part

    def randn(self, *shape, gain=1.0):
        return (gain * torch.randn(*shape, generator=self.gen)).to(self.dtype).to(self.dev)

    def call(self):
        return self.cu, self.lens, self.table_dev


def attention(b: Batch, q, causal=True, scale=None):
    """``(o, lse, tolerance of o, tolerance of lse)`` in float64, rows of no sequence 0 / -inf.

    Tolerances, from the arithmetic: scores are fp32 sums of D exact products
    (relative error D * 2^-24 of the sum of magnitudes) and the exponent's argument
    rounds twice more, so a weight is off by a factor 1 + d with d = (D + 4) * 2^-24 *
    scale * max sum |q||k| plus 4 * 2^-24 * |score| for the scaled maximum; weights
    enter the second product with half a step of the type (u); sums over L keys
    round in fp32 (L + 64 roundings at most); the result rounds once (u).  lse:
    the weights' d, the sum's roundings and the logarithm's."""
    u = U[b.dtype]
    scale = 1.0 / math.sqrt(b.D) if scale is None else scale
    g = b.H // b.Hkv
    o = torch.zeros(b.N, b.H, b.D, dtype=torch.float64)
    tol = torch.zeros_like(o)
    lse = torch.full((b.N, b.H), float("-inf"), dtype=torch.float64)
    lse_tol = torch.zeros_like(lse)
    q = q.double().cpu()
    for s, (n, L) in enumerate(b.seqs):
        if not n or not L:
            continue
        K = b.K[s].repeat_interleave(g, 1).transpose(0, 1)            # [H, L, D]
        V = b.V[s].repeat_interleave(g, 1).transpose(0, 1)
        Q = q[b.ends[s]:b.ends[s + 1]].transpose(0, 1)
        z = Q @ K.transpose(1, 2) * scale
        size = (Q.abs() @ torch.nan_to_num(K.abs(), nan=0.0, posinf=0.0).transpose(1, 2)) * scale
        pos = torch.arange(L - n, L)
        seen = torch.arange(L)[None] <= pos[:, None] if causal else torch.ones(n, L, dtype=torch.bool)
        z = torch.where(seen, z, torch.full_like(z, float("-inf")))
        size = torch.where(seen, size, torch.zeros_like(size))
        top = z.amax(-1, keepdim=True)
        some = top > float("-inf")
        w = torch.exp(z - torch.where(some, top, torch.zeros_like(top)))
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total > 0, total, torch.ones_like(total))
        row = torch.zeros(b.H, n, b.D, dtype=torch.float64)
        for h in range(b.H):                                          # unattended values out of the product
            for i in range(n) if not torch.isfinite(V[h]).all() else ():
                row[h, i] = w[h, i, seen[i]] @ V[h, seen[i]]
            if torch.isfinite(V[h]).all():
                row[h] = w[h] @ V[h]
        A = w @ torch.nan_to_num(V.abs(), nan=0.0, posinf=0.0)
        d = (b.D + 4) * F32 * size.amax(-1, keepdim=True) + 4 * F32 * torch.where(some, top, 0.0).abs()
        r = slice(b.ends[s], b.ends[s + 1])
        o[r] = row.transpose(0, 1)
        tol[r] = (u * row.abs() + A * (u + 2 * d + 2 * (L + 64) * F32)).transpose(0, 1)
        lse[r] = (top + total.log())[..., 0].T
        lse_tol[r] = (d + (L + 64) * F32 + 8 * F32 * (top.abs() + total.log().abs()))[..., 0].T
    return o, lse, tol, lse_tol


def check_close(got, want, tol, what):
    got, want = got.double().cpu(), want
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and torch.equal(torch.isinf(got), inf), f"{what}: infinities differ"
    fine = torch.isfinite(want)
    err, lim = (got - want).abs()[fine], tol.expand_as(want)[fine]
    if err.numel():
        worst = (err - lim).max().item()
        assert worst <= 0, f"{what}: off by {err.max().item():.3g}, {worst:.3g} more than allowed"
