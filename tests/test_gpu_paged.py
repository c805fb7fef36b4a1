"""The paged key/value cache against its definitions in 64 bits (tests/paged_ref.py)."""
import math

import pytest
import torch

import longvideosparseattention_amd as lv
from longvideosparseattention_amd import _capi

import paged_ref as ref
from paged_ref import Batch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _attend(b, q, causal=True, what="attention", **kw):
    o, lse = lv.paged_attention(q, b.cache, *b.call(), causal=causal, return_lse=True, **kw)
    wo, wl, tol, ltol = ref.attention(b, q, causal, kw.get("scale"))
    ref.check_close(o, wo, tol, what)
    ref.check_close(lse, wl, ltol, what + " lse")
    b.cache.check()
    return o, lse


# ── append ───────────────────────────────────────────────────────────────────

APPEND = [  # sequences, D, H, Hkv, page, rot, interleaved, layout, tail
    ([(1, 1)], 128, 4, 1, 16, 128, False, "heads", 0),
    ([(1, 40), (1, 1), (0, 9), (1, 17)], 64, 8, 2, 16, 64, True, "tokens", 0),
    ([(37, 37), (0, 0), (5, 70), (64, 64)], 128, 6, 3, 16, 64, False, "heads", 3),
    ([(23, 50), (9, 9)], 96, 5, 5, 7, 96, False, "heads", 0),
    ([(23, 50), (9, 9)], 96, 5, 5, 1, 48, True, "tokens", 2),
    ([(12, 33)], 192, 4, 2, 100, 192, True, "heads", 0),
    ([(12, 33), (3, 3)], 192, 3, 3, 5, 16, False, "tokens", 0),
    ([(20, 20), (1, 513)], 256, 8, 4, 64, 256, False, "heads", 1),
    ([(30, 31)], 64, 2, 2, 390, 0, False, "heads", 0),
]


def _angles(n, rot, dev, seed=3):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(n, rot // 2, generator=g, dtype=torch.float64) * 50
    return a.cos().float().to(dev), a.sin().float().to(dev)


def _append_case(gpu, case, dtype, bits, positions):
    seqs, D, H, Hkv, page, rot, inter, layout, tail = case
    b = Batch(gpu, seqs, D, H, Hkv, page, dtype, bits=bits, layout=layout, tail=tail, seed=5)
    k, v, q = b.randn(b.N, Hkv, D), b.randn(b.N, Hkv, D), b.randn(b.N, H, D)
    kw = {}
    longest = max(L for _, L in seqs)
    pos = torch.zeros(b.N, dtype=torch.long)
    for s, (n, L) in enumerate(seqs):
        pos[b.ends[s]:b.ends[s + 1]] = torch.arange(L - n, L)
    if rot:
        kw["cos"], kw["sin"] = _angles(2 * longest + 3, rot, gpu)
        if positions:
            pos = torch.randint(0, 2 * longest + 3, (b.N,), generator=b.gen)
            kw["positions"] = pos.to(torch.int32).to(gpu)
    return b, k, v, q, pos, kw, inter


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("i", range(len(APPEND)))
def test_append_16(gpu, i, dtype):
    b, k, v, q, pos, kw, inter = _append_case(gpu, APPEND[i], dtype, 16, positions=i % 2 == 1)
    before = [b.cache.k.cpu().clone(), b.cache.v.cpu().clone()]
    mark = torch.full_like(q, 7.0)
    got = lv.paged_kv_append(b.cache, k, v, *b.call(), q=q, interleaved=inter, q_out=mark, **kw)
    assert got is mark
    b.cache.check()
    want_k, want_q, tol_k, tol_q = [], [], [], []
    for x, w, t in ((k, want_k, tol_k), (q, want_q, tol_q)):
        x = x.double().cpu()
        y, size = x, torch.zeros_like(x)
        if kw:
            c, s = kw["cos"].cpu()[pos], kw["sin"].cpu()[pos]
            y = ref.rotate(x, c, s, inter)
            size = ref.rotate(x.abs(), c.abs(), -s.abs(), inter).abs() + ref.rotate(x.abs(), c.abs(), s.abs(), inter).abs()
        # two products and a sum in fp32 (3 roundings of at most the sum of magnitudes), one rounding to the type
        w.append(y)
        t.append(ref.U[dtype] * y.abs() + 4 * ref.F32 * size + 1e-30 + (2.0 ** -25 if dtype == HF else 0))
    n = b.n_rows
    ref.check_close(got[:n], want_q[0][:n], tol_q[0][:n], "q")
    assert (got[n:] == 7.0).all()
    kc, vc = b.cache.k.cpu(), b.cache.v.cpu()
    for s, (m, L) in enumerate(b.seqs):
        for j in range(m):
            p, t = L - m + j, b.ends[s] + j
            page, slot = b.pages[s][p // b.ps], p % b.ps
            ref.check_close(kc[page, slot], want_k[0][t], tol_k[0][t], f"key {p} of sequence {s}")
            assert torch.equal(vc[page, slot], v[t].cpu())
            before[0][page, slot], before[1][page, slot] = kc[page, slot], vc[page, slot]
    assert torch.equal(kc.nan_to_num(3.0), before[0].nan_to_num(3.0)), "a slot of no new key changed"
    assert torch.equal(vc.nan_to_num(3.0), before[1].nan_to_num(3.0)), "a slot of no new value changed"


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("i", range(len(APPEND)))
def test_append_4_bits_gives_the_exact_values_codes(gpu, i, dtype):
    b, k, v, q, pos, kw, inter = _append_case(gpu, APPEND[i], dtype, 4, positions=i % 2 == 0)
    if b.n_rows > 3:                                     # wide ranges, zeros, clamped and non-finite groups
        k[0] = 0
        k[1] *= 2.0 ** -30 if dtype == BF else 2.0 ** -12
        v[1, :, ::3] = 5.0 * 2.0 ** -4                    # ties of the code
        v[2, 0, 3], v[2, 0, 40] = float("nan"), float("-inf")
        k[3] *= 2.0 ** 20 if dtype == BF else 2.0 ** 13
    c = b.cache
    before = [t.cpu().clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    lv.paged_kv_append(c, k, v, *b.call(), q=q, interleaved=inter, **kw)
    c.check()
    x = k.double().cpu()
    if kw:
        x = ref.rotate(x, kw["cos"].cpu()[pos], kw["sin"].cpu()[pos], inter)
    wk, wv = ref.quantize(x), ref.quantize(v.double().cpu())
    for s, (m, L) in enumerate(b.seqs):
        for j in range(m):
            p, t = L - m + j, b.ends[s] + j
            page, slot = b.pages[s][p // b.ps], p % b.ps
            for i, w in ((0, wk[0]), (1, wv[0]), (2, wk[1]), (3, wv[1])):
                before[i][page, slot] = w[t]
    for name, w, g in zip(("key codes", "value codes", "key scales", "value scales"), before, (c.k, c.v, c.k_scale, c.v_scale)):
        g = g.cpu()
        assert torch.equal(g, w), f"{name}: {(g != w).sum().item()} of {g.numel()} bytes differ"


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("D,H,Hkv,rot,inter", [(64, 3, 1, 64, False), (96, 2, 2, 96, True), (128, 5, 1, 128, False),
                                               (192, 2, 1, 64, False), (256, 2, 1, 256, True)])
def test_many_tokens_equal_few_at_a_time(gpu, D, H, Hkv, rot, inter, bits):
    """Thousands of tokens in one call (a wave each) leave the bits that calls of a few hundred (four waves each) leave."""
    N, ps = 5000, 64
    g = torch.Generator().manual_seed(8)
    k, v, q = (torch.randn(N, h, D, generator=g).to(BF).to(gpu) for h in (Hkv, Hkv, H))
    cos, sin = _angles(N, rot, gpu)
    table = torch.randperm(80, generator=g)[None, :79].to(torch.int32).to(gpu)
    caches = [lv.PagedKVCache.allocate(80, ps, Hkv, D, bits=bits, device=gpu) for _ in range(2)]
    of = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    whole = lv.paged_kv_append(caches[0], k, v, of(0, N), of(N), table, q=q, cos=cos, sin=sin, interleaved=inter)
    for a in range(0, N, 700):
        e = min(a + 700, N)
        part = lv.paged_kv_append(caches[1], k[a:e], v[a:e], of(0, e - a), of(e), table, q=q[a:e], cos=cos, sin=sin,
                                  interleaved=inter)
        assert torch.equal(part, whole[a:e])
    for x in ("k", "v", "k_scale", "v_scale"):
        if getattr(caches[0], x) is not None:
            assert torch.equal(getattr(caches[0], x), getattr(caches[1], x))
    for c in caches:
        c.check()


def test_codes_of_ties_and_borders(gpu):
    """Every tie and its neighbours, at the smallest and the largest scale, both signs."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    x = torch.cat([mids, mids * (1 + 2.0 ** -7), mids * (1 - 2.0 ** -7), torch.tensor([6.0, 0.0, 4.5, 5.5])])   # 25 values
    group = torch.zeros(32)
    group[:25] = x
    tok = torch.stack([torch.cat([s * group * 2.0 ** e for s in (1, -1)]) for e in (-23, -22, 0, 12, 13)])      # [5, 64]
    cache = lv.PagedKVCache.allocate(1, 8, 1, 64, bits=4, device=gpu)
    kv = tok[:, None].to(BF).to(gpu)
    one = torch.tensor
    lv.paged_kv_append(cache, kv, kv, one([0, 5], dtype=torch.int32, device=gpu), one([5], dtype=torch.int32, device=gpu),
                       one([[0]], dtype=torch.int32, device=gpu))
    cache.check()
    codes, scales = ref.quantize(kv.double().cpu())
    for g, w in ((cache.k, codes), (cache.v, codes), (cache.k_scale, scales), (cache.v_scale, scales)):
        assert torch.equal(g[0, :5].cpu(), w)


def test_append_reads_strided_and_repacked_inputs(gpu):
    """Views of one packed projection, expanded heads, and rows that are not 16-byte aligned."""
    b = Batch(gpu, [(9, 20)], 128, 4, 2, 8, BF)
    qkv = b.randn(9, 8, 128)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    lv.paged_kv_append(b.cache, k, v, *b.call())
    first = [b.cache.k.clone(), b.cache.v.clone()]
    odd = torch.empty(9 * 2 * 128 + 1, dtype=BF, device=gpu)[1:].view(9, 2, 128)
    odd.copy_(k)
    out = lv.paged_kv_append(b.cache, odd, v.contiguous(), *b.call(), q=q)
    assert torch.equal(out, q)
    for a, w in zip((b.cache.k, b.cache.v), first):
        assert torch.equal(a.nan_to_num(3.0), w.nan_to_num(3.0))
    wide = k[:, :1].expand(9, 2, 128)
    lv.paged_kv_append(b.cache, wide, v, *b.call())
    got, _ = lv.paged_kv_gather(b.cache, b.lens, b.table_dev, 20)
    assert torch.equal(got[0, 11:], wide)


# ── gather ───────────────────────────────────────────────────────────────────


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,Hkv,page,layout", [(64, 3, 16, "heads"), (96, 1, 7, "tokens"), (128, 8, 64, "heads"),
                                               (192, 2, 1, "heads"), (256, 4, 390, "tokens")])
def test_gather(gpu, D, Hkv, page, layout, dtype, bits):
    b = Batch(gpu, [(0, 65), (0, 0), (0, 1), (0, 130)], D, Hkv, Hkv, page, dtype, bits=bits, layout=layout)
    for most in (130, 140, 33):
        got = lv.paged_kv_gather(b.cache, b.lens, b.table_dev, most, dtype=dtype)
        for g, src in zip(got, (b.K, b.V)):
            assert g.shape == (4, most, Hkv, D) and g.dtype == dtype
            for s, (_, L) in enumerate(b.seqs):
                m = min(L, most)
                assert torch.equal(g[s, :m].double().cpu(), src[s][:m])
                assert (g[s, m:] == 0).all()
    b.cache.check()
    k, v = lv.paged_kv_gather(b.cache, b.lens, b.table_dev, 0, dtype=dtype)
    assert k.shape == v.shape == (4, 0, Hkv, D)


@pytest.mark.parametrize("bits", [16, 4])
def test_gather_of_more_sequences_than_a_grid_has_rows(gpu, bits):
    B = 70000
    cache = lv.PagedKVCache.allocate(3, 4, 1, 64, bits=bits, device=gpu)
    one = torch.randn(3, 1, 64, generator=torch.Generator().manual_seed(1)).to(BF).to(gpu)
    table = torch.arange(3, dtype=torch.int32, device=gpu)[:, None]
    first = torch.arange(4, dtype=torch.int32, device=gpu)
    lv.paged_kv_append(cache, one, one, first, torch.ones(3, dtype=torch.int32, device=gpu), table)
    of = torch.arange(B, device=gpu) % 3
    k, v = lv.paged_kv_gather(cache, (of != 1).int(), of.int()[:, None].contiguous(), 2)
    few, _ = lv.paged_kv_gather(cache, torch.ones(3, dtype=torch.int32, device=gpu), table, 1)
    want = torch.where((of != 1)[:, None, None], few[of, 0], 0)
    assert torch.equal(k[:, 0], want) and torch.equal(v[:, 0], want) and (k[:, 1] == 0).all() and (v[:, 1] == 0).all()
    cache.check()


# ── attention: single tokens and few rows ────────────────────────────────────

DECODE = [  # sequences, D, H, Hkv, page, layout
    ([(1, 1)], 128, 4, 4, 16, "heads"),
    ([(1, 1001)], 128, 16, 4, 16, "heads"),
    ([(1, 31), (1, 32), (1, 33), (1, 127), (1, 128), (1, 129)], 128, 8, 2, 16, "heads"),
    ([(1, 300), (0, 0), (1, 1), (0, 50), (1, 700)], 128, 5, 1, 7, "tokens"),
    ([(1, 63), (1, 64), (1, 65), (1, 257)], 64, 12, 12, 1, "heads"),
    ([(3, 200), (1, 3), (2, 2), (4, 130)], 64, 9, 3, 32, "tokens"),
    ([(1, 640), (1, 5)], 96, 7, 1, 100, "heads"),
    ([(5, 333), (1, 12)], 96, 6, 2, 16, "tokens"),
    ([(1, 15), (1, 16), (1, 17), (1, 500)], 192, 8, 8, 16, "heads"),
    ([(2, 150), (8, 64)], 192, 8, 2, 64, "tokens"),
    ([(1, 700), (1, 9)], 256, 16, 1, 390, "heads"),
    ([(4, 90), (3, 91)], 256, 6, 1, 5, "heads"),
    ([(32, 32), (9, 400)], 128, 1, 1, 64, "heads"),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("i", range(len(DECODE)))
def test_attention_of_few_rows(gpu, i, dtype, bits, causal):
    seqs, D, H, Hkv, page, layout = DECODE[i]
    b = Batch(gpu, seqs, D, H, Hkv, page, dtype, bits=bits, layout=layout, seed=i)
    q = b.randn(b.N, H, D, gain=2.0)
    _attend(b, q, causal, max_q_len=max(n for n, _ in seqs))


@pytest.mark.parametrize("bits", [16, 4])
def test_a_long_sequence_is_shared_by_the_whole_launch(gpu, bits):
    """One row over 20,000 keys (partials from many work-groups), and beside many short ones."""
    for seqs in ([(1, 20000)], [(1, 9000)] + [(1, 3 + 7 * i) for i in range(70)]):
        b = Batch(gpu, seqs, 128, 4, 2, 64, BF, bits=bits, seed=2)
        _attend(b, b.randn(b.N, 4, 128, gain=1.5), max_q_len=1)


# ── attention: chunks ────────────────────────────────────────────────────────

CHUNKS = [  # sequences, D, H, Hkv, page, layout
    ([(200, 200)], 128, 2, 2, 16, "heads"),
    ([(130, 700), (1, 5), (0, 0), (77, 77), (64, 64)], 128, 6, 2, 16, "tokens"),
    ([(129, 400), (40, 41)], 64, 3, 1, 7, "heads"),
    ([(257, 257)], 64, 4, 4, 390, "heads"),
    ([(150, 333)], 96, 5, 1, 1, "tokens"),
    ([(65, 65), (100, 250)], 96, 2, 2, 32, "heads"),
    ([(140, 200), (3, 600)], 192, 3, 3, 64, "heads"),
    ([(90, 91)], 192, 4, 2, 5, "tokens"),
    ([(128, 128), (50, 320)], 256, 2, 1, 16, "heads"),
    ([(70, 500)], 256, 4, 4, 100, "tokens"),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("i", range(len(CHUNKS)))
def test_attention_of_chunks(gpu, i, dtype, bits, causal):
    seqs, D, H, Hkv, page, layout = CHUNKS[i]
    b = Batch(gpu, seqs, D, H, Hkv, page, dtype, bits=bits, layout=layout, seed=i)
    q = b.randn(b.N, H, D, gain=2.0)
    _attend(b, q, causal)


@pytest.mark.parametrize("n,L", [(40, 9000), (300, 5000)])
@pytest.mark.parametrize("bits,D", [(16, 128), (4, 64), (16, 256)])
def test_few_tiles_over_long_caches_run_in_parts(gpu, bits, D, n, L):
    b = Batch(gpu, [(n, L), (5, 5)], D, 2, 1, 64, BF, bits=bits, seed=4)
    for causal in (True, False):
        _attend(b, b.randn(b.N, 2, D, gain=1.5), causal)


@pytest.mark.parametrize("bits", [16, 4])
def test_hints_change_no_result_beyond_rounding(gpu, bits):
    """Wrong, missing and tight hints: every row is computed, within the same tolerance."""
    b = Batch(gpu, [(70, 300), (1, 900), (20, 20)], 128, 4, 2, 16, BF, bits=bits)
    q = b.randn(b.N, 4, 128)
    for kw in ({}, {"max_q_len": 1}, {"max_q_len": 8}, {"max_q_len": 70, "max_kv_len": 900}, {"max_q_len": 1, "max_kv_len": 1},
               {"max_kv_len": 1}, {"max_q_len": 10 ** 10, "max_kv_len": 10 ** 10}):
        _attend(b, q, True, what=str(kw), **kw)
        _attend(b, q, False, what=str(kw), **kw)


def test_single_tokens_need_no_hint(gpu):
    """As many rows as sequences: taken for single tokens, whoever's they are."""
    b = Batch(gpu, [(1, 900), (1, 5), (0, 30), (1, 300)], 128, 8, 2, 16, BF, tail=1)
    q = b.randn(b.N, 8, 128)
    o, lse = _attend(b, q)
    hint = lv.paged_attention(q, b.cache, *b.call(), max_q_len=1, return_lse=True)
    assert torch.equal(o, hint[0]) and torch.equal(lse, hint[1])
    b = Batch(gpu, [(0, 7), (4, 700), (0, 0), (0, 30)], 128, 8, 2, 16, BF)      # all of one sequence
    _attend(b, b.randn(b.N, 8, 128))


@pytest.mark.parametrize("B", [65, 128, 1100, 4300])
def test_many_sequences(gpu, B):
    """More sequences than a wave holds, than the plan takes at a time, and more row tiles than it keeps in LDS."""
    seqs = [(0 if s % 7 == 3 else 1 + (s % 11 == 0), s % 5 + (s * s) % 13) for s in range(B)]
    seqs = [(min(n, L), L) for n, L in seqs]
    b = Batch(gpu, seqs, 64, 2, 1, 8, BF, seed=6, tail=2)
    q, k, v = b.randn(b.N, 2, 64), b.randn(b.N, 1, 64), b.randn(b.N, 1, 64)
    lv.paged_kv_append(b.cache, k, v, *b.call())
    for s, (n, L) in enumerate(seqs):
        b.K[s][L - n:], b.V[s][L - n:] = k[b.ends[s]:b.ends[s + 1]].double().cpu(), v[b.ends[s]:b.ends[s + 1]].double().cpu()
    for hint in (2, 0):
        o, lse = _attend(b, q, max_q_len=hint)
        assert (o[b.n_rows:] == 0).all() and (lse[b.n_rows:] == float("-inf")).all()
    got, _ = lv.paged_kv_gather(b.cache, b.lens, b.table_dev, 17)
    assert all(torch.equal(got[s, :L].double().cpu(), b.K[s]) for s, (_, L) in enumerate(seqs))


@pytest.mark.parametrize("scale", [1e-6, 0.3, 40.0])
@pytest.mark.parametrize("n", [1, 150])
def test_scales(gpu, scale, n):
    b = Batch(gpu, [(n, 300)], 64, 2, 1, 16, HF)
    _attend(b, b.randn(n, 2, 64), scale=scale, max_q_len=n)


@pytest.mark.parametrize("n", [1, 4, 150])
def test_scores_far_from_zero(gpu, n):
    """Scores around -2000 and +2000 and rising along the keys: the running maximum moves block after block."""
    b = Batch(gpu, [(n, 500)], 64, 1, 1, 16, BF)
    for sign in (1.0, -1.0):
        b2 = Batch(gpu, [(n, 500)], 64, 1, 1, 16, BF)
        ramp = torch.linspace(1, 16, 500)[:, None, None].expand(500, 1, 64)
        b2.K[0] = ramp.to(BF).double()
        full = b2.cache.k
        host = torch.full(full.shape, float("nan"), dtype=BF)
        b2._put(host, 0, ramp.to(BF))
        full.copy_(host)
        q = torch.full((n, 1, 64), sign * 16.0, dtype=BF, device=gpu)
        _attend(b2, q, scale=0.125, max_q_len=n)


# ── empty rows, masked places, rows of no sequence ───────────────────────────


@pytest.mark.parametrize("hint", [1, 0])
def test_rows_without_keys(gpu, hint):
    """Rows before the first cached position, sequences without keys: 0 and -inf (causal), all keys otherwise."""
    b = Batch(gpu, [(6, 2), (3, 0), (40, 33), (1, 0)], 64, 4, 2, 16, BF, tail=3)
    q = b.randn(b.N, 4, 64)
    kw = {"max_q_len": hint} if hint else {}
    o, lse = _attend(b, q, True, **kw)
    assert (o[:4] == 0).all() and (lse[:4] == float("-inf")).all() and (o[6:9] == 0).all()
    assert (o[b.n_rows:] == 0).all() and (lse[b.n_rows:] == float("-inf")).all()
    out = torch.full_like(q, 9.0)
    got = lv.paged_attention(q, b.cache, *b.call(), out=out, **kw)
    assert got is out and (out[b.n_rows:] == 9.0).all() and torch.equal(out[:b.n_rows], o[:b.n_rows])


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("n,D", [(4, 128), (20, 64), (20, 256), (150, 128), (150, 64), (150, 192)])
def test_nothing_of_an_unattended_key_reaches_a_row(gpu, n, D, bits):
    """Infinities and NaN in keys and values of later tokens: earlier rows as without them, later ones as defined."""
    L = n + 60
    b = Batch(gpu, [(n, L)], D, 2, 1, 16, BF, bits=bits)
    q = b.randn(n, 2, D)
    clean, _ = _attend(b, q, max_q_len=n)
    where = L - n + n // 2                              # attended from row n / 2 on
    page, slot = b.pages[0][where // 16], where % 16
    if bits == 16:
        b.cache.v[page, slot, 0, 3] = float("inf")
        b.cache.v[page, slot, 0, 9] = float("nan")
        b.V[0][where, 0, 3], b.V[0][where, 0, 9] = float("inf"), float("nan")
        last = b.pages[0][(L - 1) // 16], (L - 1) % 16
        b.cache.v[last[0], last[1], 0, 3] = float("-inf")
        b.V[0][L - 1, 0, 3] = float("-inf")
    else:
        b.cache.v_scale[page, slot, 0, 1] = 255
        b.V[0][where, 0, 32:64] = float("nan")
    o, _ = _attend(b, q, max_q_len=n)
    assert torch.equal(o[:n // 2], clean[:n // 2])
    assert torch.isnan(o[n // 2:]).any()
    if bits == 16:                                       # a key of NaN spoils its rows whole, and only them
        b.cache.k[page, slot, 0, 0] = float("nan")
        o = lv.paged_attention(q, b.cache, *b.call(), max_q_len=n)
        assert torch.equal(o[:n // 2], clean[:n // 2]) and torch.isnan(o[n // 2:]).all()


@pytest.mark.parametrize("n", [1, 150])
def test_an_infinite_score(gpu, n):
    b = Batch(gpu, [(n, 200)], 64, 1, 1, 16, BF)
    q = b.randn(n, 1, 64).abs() + 0.25
    b.cache.k[b.pages[0][0], 5, 0, 0] = float("-inf")    # score -inf: weight 0
    b.K[0][5, 0, 0] = float("-inf")
    _attend(b, q, max_q_len=n)
    b.cache.k[b.pages[0][0], 6, 0, 0] = float("inf")     # score +inf: the softmax is undefined
    assert torch.isnan(lv.paged_attention(q, b.cache, *b.call(), max_q_len=n)).all()


def test_no_rows_no_sequences(gpu):
    b = Batch(gpu, [(0, 40), (0, 0)], 128, 4, 2, 16, BF)
    q = b.randn(0, 4, 128)
    assert lv.paged_attention(q, b.cache, *b.call()).shape == (0, 4, 128)
    assert lv.paged_kv_append(b.cache, b.randn(0, 2, 128), b.randn(0, 2, 128), *b.call(), q=q).shape == (0, 4, 128)
    none = torch.zeros(1, dtype=torch.int32, device=gpu)
    q = b.randn(3, 4, 128)
    for hint in (1, 100):
        o, lse = lv.paged_attention(q, b.cache, none, b.lens[:0], b.table_dev[:0], return_lse=True, max_q_len=hint)
        assert (o == 0).all() and (lse == float("-inf")).all()
    k, v = lv.paged_kv_gather(b.cache, b.lens[:0], b.table_dev[:0], 5)
    assert k.shape == (0, 5, 2, 128)
    b.cache.check()


# ── what the device finds wrong ──────────────────────────────────────────────


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("n", [1, 120])
@pytest.mark.parametrize("page", [-1, "past", 2 ** 31 - 1])
def test_bad_pages_spoil_their_sequence_only(gpu, page, n, bits):
    b = Batch(gpu, [(n, 150), (n, 140), (n, 333)], 128, 4, 2, 16, BF, bits=bits, spare=0)
    q = b.randn(b.N, 4, 128)
    good, _ = _attend(b, q, max_q_len=n)
    bad = b.cache.num_pages if page == "past" else page
    b.table_dev[1, 2] = bad
    o, lse = lv.paged_attention(q, b.cache, *b.call(), return_lse=True, max_q_len=n)
    assert torch.isnan(o[n:2 * n]).all() and torch.isnan(lse[n:2 * n]).all()
    assert torch.equal(o[:n], good[:n]) and torch.equal(o[2 * n:], good[2 * n:])
    with pytest.raises(ValueError, match="page number outside the cache"):
        b.cache.check()
    b.cache.check()                                       # told once
    k, _ = lv.paged_kv_gather(b.cache, b.lens, b.table_dev, 333)
    assert torch.isnan(k[1, 32:48]).all() and not torch.isnan(k[0]).any() and not torch.isnan(k[1, :32]).any()
    with pytest.raises(ValueError, match="page number"):
        b.cache.check()


@pytest.mark.parametrize("bits", [16, 4])
def test_bad_appends_leave_the_cache_alone(gpu, bits):
    b = Batch(gpu, [(4, 20), (2, 30), (5, 5)], 64, 2, 2, 16, BF, bits=bits)
    k, v, q = b.randn(b.N, 2, 64), b.randn(b.N, 2, 64), b.randn(b.N, 2, 64)
    cos, sin = _angles(25, 64, gpu)
    state = lambda: [t.clone() for t in (b.cache.k, b.cache.v, b.cache.k_scale, b.cache.v_scale) if t is not None]  # noqa: E731
    before = state()
    same = lambda: all(torch.equal(x.nan_to_num(3.0) if x.is_floating_point() else x,                               # noqa: E731
                                   y.nan_to_num(3.0) if y.is_floating_point() else y) for x, y in zip(state(), before))
    table = b.table_dev.clone()
    table[:] = b.cache.num_pages
    qo = lv.paged_kv_append(b.cache, k, v, b.cu, b.lens, table, q=q)
    assert same() and torch.isnan(qo).all()
    with pytest.raises(ValueError, match="page number"):
        b.cache.check()
    for lens, text in ((torch.tensor([3, -5, 1000]), "kv_lens"), (torch.tensor([3, 1, 4]), "more new tokens")):
        qo = lv.paged_kv_append(b.cache, k, v, b.cu, lens.to(torch.int32).to(gpu), table, q=q)
        assert same() and torch.isnan(qo).all()
        with pytest.raises(ValueError, match=text):
            b.cache.check()
    far = torch.tensor([25, -1, 2 ** 31 - 1, 99] * 3, dtype=torch.int32, device=gpu)[:b.N]
    qo = lv.paged_kv_append(b.cache, k, v, *b.call(), q=q, cos=cos, sin=sin, positions=far)
    assert same() and torch.isnan(qo).all()
    with pytest.raises(ValueError, match="cos and sin"):
        b.cache.check()
    # positions of the cache: rows 28 and 29 of sequence 1 have no angles, the others have
    qo = lv.paged_kv_append(b.cache, k, v, *b.call(), q=q, cos=cos, sin=sin)
    assert torch.isnan(qo[4:6]).all() and not torch.isnan(qo[:4]).any() and not torch.isnan(qo[6:]).any()
    with pytest.raises(ValueError, match="cos and sin"):
        b.cache.check()


@pytest.mark.parametrize("n", [2, 100])
def test_bad_lengths_and_row_ranges(gpu, n):
    """A bad length spoils its sequence; the others stay within the definition's tolerance (which work-groups share a
    sequence, and so its sums' order, depends on the whole batch's lengths)."""
    b = Batch(gpu, [(n, 150), (n, 140), (n, 133)], 128, 4, 2, 16, BF)
    q = b.randn(b.N, 4, 128)
    _attend(b, q, max_q_len=n)
    want, _, tol, _ = ref.attention(b, q)
    for bad in (-1, -2 ** 31, 2 ** 31 - 1, 161):
        lens = b.lens.clone()
        lens[1] = bad
        o = lv.paged_attention(q, b.cache, b.cu, lens, b.table_dev, max_q_len=n)
        assert torch.isnan(o[n:2 * n]).all()
        for r in (slice(0, n), slice(2 * n, 3 * n)):
            ref.check_close(o[r], want[r], tol[r], f"beside length {bad}")
        with pytest.raises(ValueError, match="kv_lens"):
            b.cache.check()
    for cu in ([0, n, 2 * n, 3 * n + 50], [0, 2 * n, n, 3 * n], [-5, n, 2 * n, 3 * n], [0, n, 2 ** 31 - 1, 3 * n]):
        cu = torch.tensor(cu, dtype=torch.int32, device=gpu)
        lv.paged_attention(q, b.cache, cu, b.lens, b.table_dev, max_q_len=n)
        with pytest.raises(ValueError, match="cu_seqlens"):
            b.cache.check()


# ── as a program uses them ───────────────────────────────────────────────────


@pytest.mark.parametrize("bits", [16, 4])
def test_a_serving_run(gpu, bits):
    """Prompts of different lengths, then single tokens, through append and attention; every step against the
    definition over the whole history."""
    D, H, Hkv, ps = 128, 8, 2, 16
    g = torch.Generator().manual_seed(0)
    prompts, steps = [35, 1, 64], 5
    B = len(prompts)
    cache = lv.PagedKVCache.allocate(40, ps, Hkv, D, bits=bits, device=gpu)
    table = torch.randperm(40, generator=g)[:B * 10].view(B, 10).to(torch.int32).to(gpu)
    cos, sin = _angles(200, D, gpu)
    hist = [(torch.zeros(0, Hkv, D, dtype=torch.float64), torch.zeros(0, Hkv, D, dtype=torch.float64)) for _ in range(B)]
    lens = [0] * B
    for step in range(steps):
        new = prompts if step == 0 else [1] * B
        lens = [a + n for a, n in zip(lens, new)]
        ends = [0]
        for n in new:
            ends.append(ends[-1] + n)
        N = ends[-1]
        k, v, q = ((torch.randn(N, h, D, generator=g)).to(BF).to(gpu) for h in (Hkv, Hkv, H))
        cu = torch.tensor(ends, dtype=torch.int32, device=gpu)
        kv = torch.tensor(lens, dtype=torch.int32, device=gpu)
        qr = lv.paged_kv_append(cache, k, v, cu, kv, table, q=q, cos=cos, sin=sin)
        o = lv.paged_attention(qr, cache, cu, kv, table, max_q_len=max(new))
        cache.check()
        b = object.__new__(Batch)
        b.D, b.H, b.Hkv, b.dtype, b.N, b.ends = D, H, Hkv, BF, N, ends
        b.seqs = list(zip(new, lens))
        b.K, b.V = [], []
        held = lv.paged_kv_gather(cache, kv, table, max(lens))
        for s in range(B):
            at = torch.arange(lens[s] - new[s], lens[s])
            x, c, d = k[ends[s]:ends[s + 1]].double().cpu(), cos.cpu()[at], sin.cpu()[at]
            kk, vv = ref.rotate(x, c, d, False), v[ends[s]:ends[s + 1]].double().cpu()
            got = held[0][s, :lens[s]].double().cpu()
            if bits == 16:               # as in test_append_16; the attention is then held to the keys that are kept
                size = ref.rotate(x.abs(), c.abs(), -d.abs(), False).abs() + ref.rotate(x.abs(), c.abs(), d.abs(), False).abs()
                ref.check_close(got[lens[s] - new[s]:], kk, ref.U[BF] * kk.abs() + 4 * ref.F32 * size + 1e-30, "key")
                kk = got[lens[s] - new[s]:]
            else:
                kk, vv = ref.dequantize(*ref.quantize(kk)), ref.dequantize(*ref.quantize(vv))
            hist[s] = torch.cat((hist[s][0], kk)), torch.cat((hist[s][1], vv))
            assert torch.equal(got, hist[s][0]) and torch.equal(held[1][s, :lens[s]].double().cpu(), hist[s][1])
            b.K.append(hist[s][0])
            b.V.append(hist[s][1])
        want, _, tol, _ = ref.attention(b, qr, True)
        ref.check_close(o, want, tol, f"step {step}")


def test_frames_chunk_by_chunk_against_the_dense_call(gpu):
    """A video stream: each new frame over all cached frames and itself, against the dense attention of the read-back
    cache; then the sparse call on it."""
    P, D, H = 130, 64, 3
    cache = lv.PagedKVCache.allocate(6, P, H, D, device=gpu)
    table = torch.tensor([[3, 0, 5, 1, 4]], dtype=torch.int32, device=gpu)
    g = torch.Generator().manual_seed(1)
    cu = torch.tensor([0, P], dtype=torch.int32, device=gpu)
    for f in range(5):
        q, k, v = (torch.randn(P, H, D, generator=g).to(BF).to(gpu) for _ in range(3))
        lens = torch.tensor([P * (f + 1)], dtype=torch.int32, device=gpu)
        lv.paged_kv_append(cache, k, v, cu, lens, table)
        o = lv.paged_attention(q, cache, cu, lens, table, causal=False)
        kk, vv = lv.paged_kv_gather(cache, lens, table, P * (f + 1))
        dense = lv.single_prefill_with_kv_cache(q, kk[0], vv[0])
        A = vv[0].abs().amax().item()
        assert (o - dense).abs().max().item() <= 4 * ref.U[BF] * A
    cache.check()
    m = lv.LVSAMetadata.build(total_latent_frames=5, num_patches=P, window_size=4, n_first_frames=1,
                              key_frame_interval=None, rank=0, world=1)
    qq = torch.randn(1, 5 * P, H, D, generator=g).to(BF).to(gpu)
    sparse = lv.lvsa_attention(qq, kk, vv, m)             # a window over every frame: the dense result
    whole = lv.paged_attention(qq[0], cache, torch.tensor([0, 5 * P], dtype=torch.int32, device=gpu), lens, table, causal=False)
    assert (sparse[0] - whole).abs().max().item() <= 4 * ref.U[BF] * vv.abs().amax().item()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("n", [1, 60])
def test_a_captured_step_serves_later_steps(gpu, n, bits):
    """Append and attention captured once, replayed with new tokens, lengths and tables, eager work in between."""
    _captured_step(gpu, n, bits, 20)


def _captured_step(gpu, n, bits, columns):
    D, H, Hkv, ps, B = 128, 4, 2, 16, 3
    g = torch.Generator().manual_seed(5)
    make = lambda: lv.PagedKVCache.allocate(64, ps, Hkv, D, bits=bits, device=gpu)  # noqa: E731
    cache, other = make(), make()
    table = torch.full((B, columns), -1, dtype=torch.int32, device=gpu)
    table[:, :20] = torch.randperm(64, generator=g)[:B * 20].view(B, 20).to(gpu)
    cos, sin = _angles(400, D, gpu)
    cu = (torch.arange(B + 1, dtype=torch.int32) * n).to(gpu)
    lens = torch.zeros(B, dtype=torch.int32, device=gpu)
    bufs = [torch.zeros(B * n, h, D, dtype=BF, device=gpu) for h in (Hkv, Hkv, H)]

    def step(c, k, v, q, kv):
        qr = lv.paged_kv_append(c, k, v, cu, kv, table, q=q, cos=cos, sin=sin)
        return lv.paged_attention(qr, c, cu, kv, table, max_q_len=n, return_lse=True)

    lens += n
    step(other, *bufs, lens)                              # warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache, *bufs, lens)
    eager = make()
    for i in range(4):                                    # 60 * 5 tokens: the table holds 20 * 16
        new = [torch.randn(B * n, h, D, generator=g).to(BF) for h in (Hkv, Hkv, H)]
        for t, x in zip(bufs, new):
            t.copy_(x)
        lens.copy_(torch.tensor([n * (i + 1), n, n * (i + 2)]))
        graph.replay()
        want = step(eager, *[x.to(gpu) for x in new], lens.clone())
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
        assert torch.equal(cache.k, eager.k) and torch.equal(cache.v, eager.v)
    cache.check()


def test_two_streams_at_once(gpu):
    """Calls on two streams over one cache (workspaces of their own), and a run repeated bit for bit."""
    b = Batch(gpu, [(1, 4000), (1, 50), (1, 2500)], 128, 8, 2, 16, BF)
    q = b.randn(b.N, 8, 128)
    first = lv.paged_attention(q, b.cache, *b.call(), max_q_len=1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(lv.paged_attention(q, b.cache, *b.call(), max_q_len=1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, first) for x in got)


def test_a_shared_prefix_and_a_row_strided_table(gpu):
    """Two sequences name the same pages; the table is a view of a wider one with other columns in between."""
    b = Batch(gpu, [(1, 100), (1, 100)], 128, 4, 4, 16, BF)
    wide = torch.full((2, 40), -1, dtype=torch.int32, device=gpu)
    wide[:, :7] = b.table_dev[:1]
    q = b.randn(2, 4, 128)
    q[1] = q[0]
    o = lv.paged_attention(q, b.cache, b.cu, b.lens, wide[:, :20], max_q_len=1)
    assert torch.equal(o[0], o[1])
    assert torch.equal(o[0], lv.paged_attention(q, b.cache, *b.call(), max_q_len=1)[0])
    b.cache.check()


@pytest.mark.parametrize("bits", [16, 4])
def test_offsets_beyond_32_bits(gpu, bits):
    """Pages whose bytes lie beyond 2^32 of the cache's start, written, read back and attended."""
    ps, Hkv, D = 1024, 8, 128
    row = Hkv * (D * 2 if bits == 16 else D // 2)
    pages = (1 << 32) // (ps * row) + 3
    shape = (pages, Hkv, ps)
    new = lambda w, dt: torch.empty(*shape, w, dtype=dt, device=gpu).transpose(1, 2)  # noqa: E731
    if bits == 16:
        cache = lv.PagedKVCache(new(D, BF), new(D, BF))
    else:
        cache = lv.PagedKVCache(new(D // 2, torch.uint8), new(D // 2, torch.uint8), new(D // 32, torch.uint8),
                                new(D // 32, torch.uint8))
    small = lv.PagedKVCache.allocate(4, ps, Hkv, D, bits=bits, device=gpu)
    g = torch.Generator().manual_seed(2)
    n = 1500
    k, v, q = (torch.randn(n, h, D, generator=g).to(BF).to(gpu) for h in (Hkv, Hkv, 16))
    cu = torch.tensor([0, n], dtype=torch.int32, device=gpu)
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    far = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=gpu)
    near = torch.tensor([[0, 2]], dtype=torch.int32, device=gpu)
    for c, t in ((cache, far), (small, near)):
        lv.paged_kv_append(c, k, v, cu, lens, t)
    for c, t in ((cache, far),):
        a, w = lv.paged_kv_gather(c, lens, t, n), lv.paged_kv_gather(small, lens, near, n)
        assert torch.equal(a[0], w[0]) and torch.equal(a[1], w[1])
        assert torch.equal(lv.paged_attention(q, c, cu, lens, t), lv.paged_attention(q, small, cu, lens, near))
        one = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
        assert torch.equal(lv.paged_attention(q[:1], c, one, lens, t, max_q_len=1),
                           lv.paged_attention(q[:1], small, one, lens, near, max_q_len=1))
    cache.check()


# ── chunks with room for long caches ─────────────────────────────────────────

# Where the page table leaves room for them, chunks run on the kernels of long caches whatever the lengths are: the
# chunks' tests again with such tables.
ROOM = 700000
ROOMY = ([(test_attention_of_chunks, dict(i=i, dtype=dtype, bits=bits, causal=causal)) for i in range(len(CHUNKS))
          for dtype in (BF, HF) for bits in (16, 4) for causal in (True, False)] +
         [(test_few_tiles_over_long_caches_run_in_parts, dict(bits=bits, D=D, n=n, L=L)) for bits, D in ((16, 128), (4, 64), (16, 256))
          for n, L in ((40, 9000), (300, 5000))] +
         [(test_hints_change_no_result_beyond_rounding, dict(bits=bits)) for bits in (16, 4)] +
         [(test_scales, dict(scale=scale, n=150)) for scale in (1e-6, 0.3, 40.0)] +
         [(test_scores_far_from_zero, dict(n=n)) for n in (40, 150)] +
         [(test_rows_without_keys, dict(hint=0))] +
         [(test_nothing_of_an_unattended_key_reaches_a_row, dict(n=n, D=D, bits=bits)) for bits in (16, 4)
          for n, D in ((20, 64), (20, 256), (40, 128), (60, 96), (150, 128), (150, 96), (150, 64), (150, 192))] +
         [(test_an_infinite_score, dict(n=n)) for n in (40, 150)] +
         [(test_bad_pages_spoil_their_sequence_only, dict(page=page, n=n, bits=bits)) for page in (-1, "past", 2 ** 31 - 1)
          for n in (30, 120) for bits in (16, 4)] +
         [(test_many_sequences, dict(B=B)) for B in (65, 1100)])


@pytest.mark.parametrize("i", range(len(ROOMY)), ids=lambda i: ROOMY[i][0].__name__[5:] + "-" + "-".join(
    str(v).replace("torch.", "") for v in ROOMY[i][1].values()))
def test_with_room(gpu, monkeypatch, i):
    class Roomy(Batch):
        def __init__(self, dev, seqs, D, H, Hkv, page, *a, **kw):
            super().__init__(dev, seqs, D, H, Hkv, page, *a, extra_columns=-(-(ROOM if len(seqs) < 10 else 20000) // page), **kw)

    monkeypatch.setitem(globals(), "Batch", Roomy)
    test, kw = ROOMY[i]
    test(gpu, **kw)


@pytest.mark.parametrize("n", [40, 100])
def test_bad_lengths_and_row_ranges_with_room(gpu, n):
    b = Batch(gpu, [(n, 150), (n, 140), (n, 133)], 128, 4, 2, 16, BF, extra_columns=ROOM // 16)
    q = b.randn(b.N, 4, 128)
    want, _, tol, _ = ref.attention(b, q)
    for bad in (-1, -2 ** 31, 2 ** 31 - 1, ROOM + 161):
        lens = b.lens.clone()
        lens[1] = bad
        o = lv.paged_attention(q, b.cache, b.cu, lens, b.table_dev, max_kv_len=ROOM) if bad < 0 else None
        if bad > 0:                                       # cut to the table's room, whose further pages are no pages
            lens[0] = lens[2] = 0
            q1 = q[:2 * n]
            o = lv.paged_attention(q1, b.cache, torch.tensor([0, n, n + 1, n + 1], dtype=torch.int32, device=gpu), lens, b.table_dev)
            assert torch.isnan(o[n]).all()
        else:
            assert torch.isnan(o[n:2 * n]).all()
            for r in (slice(0, n), slice(2 * n, 3 * n)):
                ref.check_close(o[r], want[r], tol[r], f"beside length {bad}")
        with pytest.raises(ValueError, match="kv_lens"):
            b.cache.check()
    for cu in ([0, n, 2 * n, 3 * n + 50], [0, 2 * n, n, 3 * n], [-5, n, 2 * n, 3 * n], [0, n, 2 ** 31 - 1, 3 * n]):
        cu = torch.tensor(cu, dtype=torch.int32, device=gpu)
        lv.paged_attention(q, b.cache, cu, b.lens, b.table_dev)
        with pytest.raises(ValueError, match="cu_seqlens"):
            b.cache.check()


@pytest.mark.parametrize("bits", [16, 4])
def test_a_captured_chunk_with_room(gpu, bits):
    _captured_step(gpu, 60, bits, ROOM // 16)


def test_chunks_on_two_streams(gpu):
    b = Batch(gpu, [(70, 900), (1, 50), (200, 200)], 128, 8, 2, 16, BF, extra_columns=ROOM // 16)
    q = b.randn(b.N, 8, 128)
    first, _ = _attend(b, q)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(lv.paged_attention(q, b.cache, *b.call()))
    torch.cuda.synchronize()
    assert all(torch.equal(x, first) for x in got)


# ── refusals ─────────────────────────────────────────────────────────────────


def test_refusals(gpu):
    b = Batch(gpu, [(2, 20)], 128, 4, 2, 16, BF)
    q, k = b.randn(2, 4, 128), b.randn(2, 2, 128)
    cu, lens, table = b.call()
    att = lambda *a, **kw: lv.paged_attention(*a, **kw)  # noqa: E731
    with pytest.raises(RuntimeError, match="GPU"):
        att(q.cpu(), b.cache, cu, lens, table)
    with pytest.raises(RuntimeError, match="GPU"):
        att(q, b.cache, cu.cpu(), lens, table)
    with pytest.raises(TypeError, match="int32"):
        att(q, b.cache, cu.long(), lens, table)
    with pytest.raises(TypeError, match="dtype"):
        att(q.half(), b.cache, cu, lens, table)
    with pytest.raises(TypeError, match="dtype"):
        att(q.float(), b.cache, cu, lens, table)
    with pytest.raises(ValueError, match="multiple of kv heads"):
        att(q[:, :3], b.cache, cu, lens, table)
    with pytest.raises(ValueError, match="cu_seqlens"):
        att(q, b.cache, cu[:1], lens, table)
    with pytest.raises(ValueError, match="kv_lens"):
        att(q, b.cache, cu, lens.repeat(2), table)
    for scale in (0.0, -1.0, 3e38, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            att(q, b.cache, cu, lens, table, scale=scale)
    with pytest.raises(ValueError, match="share memory"):
        att(q, b.cache, cu, lens, table, out=q)
    with pytest.raises(ValueError, match="out must be"):
        att(q, b.cache, cu, lens, table, out=torch.empty_like(q[:1]))
    with pytest.raises(ValueError, match="overlapping"):
        att(q, b.cache, cu, lens, table, out=torch.empty_like(q[:1]).expand(2, 4, 128))
    with pytest.raises(RuntimeError, match="gradient"):
        att(q.clone().requires_grad_(), b.cache, cu, lens, table)
    app = lambda **kw: lv.paged_kv_append(b.cache, k, k, cu, lens, table, **kw)  # noqa: E731
    cos, sin = _angles(30, 128, gpu)
    with pytest.raises(ValueError, match="go together"):
        app(cos=cos)
    with pytest.raises(ValueError, match="multiple of 16"):
        app(cos=cos[:, :20].contiguous(), sin=sin[:, :20].contiguous())
    with pytest.raises(TypeError, match="fp32"):
        app(cos=cos.double(), sin=sin.double())
    with pytest.raises(ValueError, match="positions without"):
        app(positions=torch.zeros(2, dtype=torch.int32, device=gpu))
    with pytest.raises(ValueError, match="share memory"):
        app(q=q, q_out=q)
    with pytest.raises(ValueError, match="share memory"):         # the keys' memory
        both = b.randn(2, 8, 128)
        lv.paged_kv_append(b.cache, both[:, 3:5], k, cu, lens, table, q=q, q_out=both[:, :4])
    with pytest.raises(ValueError, match="tokens"):
        lv.paged_kv_append(b.cache, k, k[:1], cu, lens, table)
    with pytest.raises(ValueError, match="max_len"):
        lv.paged_kv_gather(b.cache, lens, table, -1)
    with pytest.raises(ValueError, match="head_dim"):
        lv.PagedKVCache.allocate(2, 16, 2, 80, device=gpu)
    with pytest.raises(ValueError, match="bits"):
        lv.PagedKVCache.allocate(2, 16, 2, 128, bits=8, device=gpu)
    with pytest.raises(TypeError, match="dtype"):
        lv.PagedKVCache.allocate(2, 16, 2, 128, dtype=torch.float32, device=gpu)
    with pytest.raises(ValueError, match="overlapping"):
        t = torch.zeros(1, 16, 2, 128, dtype=BF, device=gpu).expand(4, 16, 2, 128)
        lv.PagedKVCache(t, t)
    with pytest.raises(ValueError, match="16 bytes"):
        t = torch.zeros(2 * 16 * 2 * 128 + 4, dtype=BF, device=gpu)[4:].view(2, 16, 2, 128)
        lv.PagedKVCache(t, t)
    with pytest.raises(ValueError, match="differ"):
        lv.PagedKVCache(b.cache.k, b.cache.v[:1])
    with pytest.raises(ValueError, match="share memory"):
        lv.PagedKVCache(b.cache.k, b.cache.k)
    b.cache.check()
