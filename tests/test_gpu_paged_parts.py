"""Block means, selection, attention over blocks, accumulated weights and eviction against their definitions in 64 bits
(tests/paged_parts_ref.py)."""
import math

import pytest
import torch

import longvideosparseattention_amd as lv

import paged_parts_ref as ref
import paged_ref
from paged_ref import F32, Batch, check_close

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


# ── means ────────────────────────────────────────────────────────────────────

MEANS = [  # sequences, D, H, Hkv, page, block, layout
    ([(1, 1)], 128, 2, 1, 16, 16, "heads"),
    ([(1, 40), (1, 33), (0, 9), (5, 17)], 64, 4, 2, 16, 8, "tokens"),
    ([(37, 37), (0, 0), (5, 70), (64, 64)], 128, 6, 3, 32, 32, "heads"),
    ([(23, 50), (9, 9)], 96, 5, 5, 7, 7, "heads"),
    ([(23, 50), (9, 9)], 96, 5, 5, 6, 1, "tokens"),
    ([(12, 233), (230, 230)], 192, 4, 2, 100, 20, "heads"),
    ([(20, 20), (1, 513), (400, 800)], 256, 8, 4, 390, 195, "heads"),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("i", range(len(MEANS)))
def test_means(gpu, i, dtype, bits):
    seqs, D, H, Hkv, page, block, layout = MEANS[i]
    b = Batch(gpu, seqs, D, H, Hkv, page, dtype, bits=bits, layout=layout, seed=3)
    want = ref.means(b, block)
    for cu in (b.cu, None):
        m = b.cache.allocate_means(block)
        m.fill_(7.0)
        assert lv.paged_kv_block_means(b.cache, m, b.lens, b.table_dev, cu_seqlens=cu) is m
        b.cache.check()
        expect = torch.full(m.shape, 7.0, dtype=torch.float64)
        tol = torch.zeros_like(expect)
        for s, (n, L) in enumerate(seqs):
            for j in range((L - n) // block if cu is not None else 0, -(-L // block) if n or cu is None else 0):
                at = b.pages[s][j * block // page], j * block % page // block
                K = b.K[s][j * block:(j + 1) * block].double()
                expect[at] = want[s][j]
                # fp32 sums of up to block / 8 keys, 64 bits across them, one rounding
                tol[at] = F32 * (want[s][j].abs() + (block / 8 + 1) * K.abs().mean(0))
        check_close(m, expect, tol, f"means, {'new blocks' if cu is not None else 'all blocks'}")


def test_means_in_another_layout_and_of_many_sequences(gpu):
    seqs = [(1, 1 + 7 * i % 90) for i in range(150)]
    b = Batch(gpu, seqs, 64, 2, 2, 8, BF, seed=4)
    m = torch.full((b.cache.num_pages, 2, 2, 64), 5.0, device=gpu)           # 4 slots a block, a page's heads side by side
    lv.paged_kv_block_means(b.cache, m, b.lens, b.table_dev, cu_seqlens=b.cu)
    want = ref.means(b, 4)
    got = m.cpu()
    for s, (_, L) in enumerate(seqs):
        j = (L - 1) // 4
        at = b.pages[s][j * 4 // 8], j * 4 % 8 // 4
        assert torch.allclose(got[at].double(), want[s][j], rtol=2e-6, atol=1e-6), s
        got[at] = 5.0
    assert (got == 5.0).all()


# ── selection ────────────────────────────────────────────────────────────────

SELECT = [  # sequences, D, H, Hkv, page, block, top, tile, first, last, causal
    ([(1, 1)], 128, 2, 1, 16, 16, 1, 1, 0, 1, True),
    ([(1, 400), (1, 33), (0, 9), (1, 170)], 64, 8, 2, 16, 8, 6, 1, 1, 1, True),
    ([(37, 300), (0, 0), (5, 70), (64, 64)], 128, 6, 3, 32, 32, 3, 1, 1, 1, True),
    ([(37, 300), (0, 0), (5, 70), (64, 64)], 128, 6, 3, 32, 4, 17, 16, 1, 3, True),
    ([(23, 150), (9, 9)], 96, 5, 5, 7, 7, 8, 8, 2, 2, False),
    ([(23, 50), (9, 9), (3, 2)], 96, 5, 5, 6, 1, 20, 8, 0, 1, True),
    ([(120, 2330), (230, 230)], 192, 4, 2, 100, 20, 14, 100, 1, 1, False),
    ([(20, 20), (1, 1513), (40, 800)], 256, 8, 4, 390, 15, 9, 7, 1, 0, True),
    ([(2, 9000)], 64, 1, 1, 8, 1, 1024, 1, 0, 0, False),        # more blocks than are ranked at a time
    ([(1, 30000), (3, 11000)], 64, 4, 2, 64, 2, 100, 2, 1, 2, True),
    ([(300, 700), (100, 900), (0, 50), (17, 17), (65, 64)], 64, 4, 2, 8, 8, 12, 1, 2, 2, True),
    ([(300, 700), (100, 900), (0, 50), (17, 17), (65, 64)], 64, 16, 8, 8, 8, 12, 1, 2, 2, True),   # sixteen lists at a time
    ([(300, 2000), (210, 250)], 128, 16, 16, 20, 2, 33, 5, 0, 3, False),
    ([(200, 300), (180, 200)], 96, 32, 16, 3, 1, 7, 3, 1, 0, True),
    ([(90, 130), (70, 75)], 192, 20, 20, 16, 4, 5, 2, 1, 1, True),
    ([(64, 700)], 256, 72, 24, 32, 8, 40, 1, 1, 1, False),
]


def _means_of(b, block, gen, dev):
    """Random means (their own values, as fp32), NaN in what no block of a sequence owns."""
    rows = [torch.randn(-(-L // block), b.Hkv, b.D, generator=gen) for _, L in b.seqs]
    like = b.cache.allocate_means(block)
    return rows, like.copy_(ref.paged(b, rows, block, float("nan"), like))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("i", range(len(SELECT)))
def test_select(gpu, i, dtype):
    seqs, D, H, Hkv, page, block, top, tile, first, last, causal = SELECT[i]
    b = Batch(gpu, seqs, D, H, Hkv, page, dtype, seed=6, tail=3)
    rows, m = _means_of(b, block, b.gen, gpu)
    q = b.randn(b.N, H, D)
    got = lv.paged_kv_select(q, b.cache, m, *b.call(), top, tile=tile, first=first, last=last, causal=causal)
    b.cache.check() if all(n <= L for n, L in seqs) else None
    want = ref.select(b, q, rows, block, top, tile, first, last, causal)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("n,Hkv", [(1, 1), (40, 20)])
def test_select_takes_the_lower_of_equal_blocks_and_nan_last(gpu, n, Hkv):
    seqs = [(n, 700), (n, 640)]
    b = Batch(gpu, seqs, 64, 2 * Hkv, Hkv, 10, BF, seed=7)
    q = torch.randint(-2, 3, (b.N, 2 * Hkv, 64), generator=b.gen).to(BF).to(gpu)  # whole numbers: sums are exact
    rows = [torch.randint(-1, 2, (-(-L // 10), Hkv, 64), generator=b.gen).float() for _, L in seqs]
    rows[0][5:60] = rows[0][5]                                                  # many alike
    rows[1][3:40] = float("nan")
    rows[1][45], rows[1][46] = float("inf"), 0.0
    rows[0][61] = rows[0][62] = 0.5
    rows[0][61, 0, 0] += 2.0 ** -24                                             # scores nearer than fp32 tells apart
    rows[0][8:11] = 0.0                                                         # and scores of 0
    like = b.cache.allocate_means(10)
    like.copy_(ref.paged(b, rows, 10, float("nan"), like))
    for top in (3, 20, 40, 61, 64, 70, 71):
        got = lv.paged_kv_select(q, b.cache, like, *b.call(), top, first=1, last=1)
        assert torch.equal(got.cpu(), ref.select(b, q, rows, 10, top, 1, 1, 1, True)), top


# ── attention over blocks ────────────────────────────────────────────────────

ATTEND = [  # sequences, D, H, Hkv, page, block, top, tile, causal, layout, tail
    ([(1, 1)], 128, 4, 1, 16, 16, 1, 1, True, "heads", 0),
    ([(1, 400), (1, 33), (0, 9), (1, 170)], 64, 8, 2, 16, 8, 6, 1, True, "tokens", 2),
    ([(37, 300), (0, 0), (5, 70), (64, 64)], 128, 6, 3, 32, 32, 4, 1, True, "heads", 1),
    ([(37, 300), (0, 0), (5, 70), (64, 64)], 128, 6, 3, 32, 4, 17, 16, True, "heads", 0),
    ([(23, 150), (9, 9)], 96, 5, 5, 7, 7, 8, 8, False, "heads", 0),
    ([(23, 50), (9, 9)], 96, 10, 5, 6, 1, 20, 8, True, "tokens", 0),
    ([(120, 930), (130, 230)], 192, 4, 2, 100, 20, 14, 100, True, "heads", 0),
    ([(20, 20), (1, 1513), (40, 800)], 256, 8, 4, 390, 15, 9, 7, True, "heads", 3),
    ([(20, 20), (1, 513), (40, 300)], 256, 24, 1, 64, 16, 9, 64, False, "heads", 0),
    ([(1, 900), (3, 1100)], 64, 17, 1, 64, 2, 100, 1, True, "heads", 0),
    ([(300, 700)], 128, 2, 2, 104, 104, 5, 128, True, "heads", 0),
    ([(300, 700)], 64, 2, 1, 40, 8, 30, 200, False, "tokens", 0),
]


def _lists(b, block, top, tile, causal, gen):
    """Random ascending lists: own blocks mostly among them, some empty, some short."""
    todo, T = ref.tiles(b, tile)
    out = torch.full((T, b.Hkv, top), -1, dtype=torch.int32)
    for at, s, r0, r1, p0 in todo:
        blocks = -(-b.seqs[s][1] // block)
        for h in range(b.Hkv):
            r = torch.rand((), generator=gen).item()
            k = 0 if r < 0.05 else min(top, blocks) if r < 0.7 else int(torch.randint(1, min(top, blocks) + 1, (), generator=gen))
            ids = torch.randperm(blocks, generator=gen)[:k]
            if k and r < 0.9:
                own = (p0 + r1 - r0 - 1) // block
                ids[0] = own if own not in ids.tolist() else ids[0]
            ids = ids.sort()[0]
            out[at, h, :k] = ids.int()
    return out


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("i", range(len(ATTEND)))
def test_block_attention(gpu, i, dtype, bits):
    seqs, D, H, Hkv, page, block, top, tile, causal, layout, tail = ATTEND[i]
    b = Batch(gpu, seqs, D, H, Hkv, page, dtype, bits=bits, layout=layout, tail=tail, seed=8)
    q = b.randn(b.N, H, D, gain=1.5)
    lists = _lists(b, block, top, tile, causal, b.gen)
    o, lse = lv.paged_block_attention(q, b.cache, lists.to(gpu), block, *b.call(), tile=tile, causal=causal, return_lse=True)
    b.cache.check()
    wo, wl, tol, ltol = ref.attention(b, q, lists, block, tile, causal)
    check_close(o, wo, tol, "o")
    check_close(lse, wl, ltol, "lse")
    mark = torch.full_like(q, 3.0)
    again = lv.paged_block_attention(q, b.cache, lists.to(gpu), block, *b.call(), tile=tile, causal=causal, out=mark)
    assert again is mark and torch.equal(mark[:b.n_rows], o[:b.n_rows]) and (mark[b.n_rows:] == 3.0).all()


def test_lists_of_all_blocks_are_dense_attention(gpu):
    seqs = [(70, 300), (1, 129), (40, 40)]
    b = Batch(gpu, seqs, 128, 4, 2, 32, BF, seed=9)
    q = b.randn(b.N, 4, 128)
    for tile in (1, 8, 64):
        T = ref.tiles(b, tile)[1]
        lists = torch.full((T, 2, 20), -1, dtype=torch.int32)
        for at, s, *_ in ref.tiles(b, tile)[0]:
            k = -(-seqs[s][1] // 16)
            lists[at, :, :k] = torch.arange(k, dtype=torch.int32)
        o = lv.paged_block_attention(q, b.cache, lists.to(gpu), 16, *b.call(), tile=tile)
        wo, _, tol, _ = paged_ref.attention(b, q, True)
        check_close(o, wo, tol, f"tiles of {tile}")


@pytest.mark.parametrize("tile", [1, 16, 128])
def test_keys_that_are_not_attended_have_no_effect(gpu, tile):
    """Infinities and NaN in blocks of no list, and in future positions of listed ones."""
    seqs = [(130, 400)]
    b = Batch(gpu, seqs, 64, 2, 1, 16, BF, seed=10)
    q = b.randn(b.N, 2, 64)
    lists = torch.full((ref.tiles(b, tile)[1], 1, 12), -1, dtype=torch.int32)
    for at, s, r0, r1, p0 in ref.tiles(b, tile)[0]:
        own = (p0 + r1 - r0 - 1) // 16
        ids = sorted({0, 3, 7, own, max(0, own - 1)} | set(range(max(p0, 0) // 16, own + 1)))[:12]
        lists[at, 0, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
    call = lambda: lv.paged_block_attention(q, b.cache, lists.to(gpu), 16, *b.call(), tile=tile)  # noqa: E731
    clean = call()
    for block in (1, 2, 4):
        b.cache.k[b.pages[0][block]] = float("nan")
        b.cache.v[b.pages[0][block]] = float("inf")
    assert torch.equal(call(), clean)
    # the last token's key and value: its own row alone attends them
    p = 399
    b.cache.k[b.pages[0][p // 16], p % 16] = float("nan")
    b.cache.v[b.pages[0][p // 16], p % 16] = float("-inf")
    got = call()
    assert torch.equal(got[:-1], clean[:-1]) and torch.isnan(got[-1]).all()


# ── weights ──────────────────────────────────────────────────────────────────

WEIGHTS = [  # sequences, D, H, Hkv, page, causal, layout, tail
    ([(1, 1)], 128, 4, 1, 16, True, "heads", 0),
    ([(1, 400), (1, 33), (0, 9), (1, 170)], 64, 8, 2, 16, True, "tokens", 2),
    ([(37, 300), (0, 0), (5, 70), (64, 64)], 128, 6, 3, 32, True, "heads", 1),
    ([(37, 300), (0, 0), (5, 70), (64, 64)], 128, 6, 3, 32, False, "heads", 0),
    ([(23, 150), (9, 9)], 96, 5, 5, 7, True, "heads", 0),
    ([(120, 930), (130, 230)], 192, 4, 2, 100, True, "heads", 0),
    ([(20, 20), (1, 1513), (40, 800)], 256, 8, 4, 390, False, "heads", 3),
    ([(300, 700), (260, 260)], 64, 6, 2, 40, True, "heads", 0),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("i", range(len(WEIGHTS)))
def test_weights(gpu, i, dtype, bits):
    seqs, D, H, Hkv, page, causal, layout, tail = WEIGHTS[i]
    b = Batch(gpu, seqs, D, H, Hkv, page, dtype, bits=bits, layout=layout, tail=tail, seed=11)
    q = b.randn(b.N, H, D, gain=1.5)
    _, lse = lv.paged_attention(q, b.cache, *b.call(), causal=causal, return_lse=True)
    if b.n_rows > 4:
        lse[1], lse[2, 0] = float("nan"), float("-inf")
    sums = ref.weights(b, q, lse, causal)
    for accumulate in (True, False):
        w = b.cache.allocate_weights()
        old = torch.rand(w.shape, generator=b.gen)
        w.copy_(old)
        got = lv.paged_kv_weights(q, lse, b.cache, w, *b.call(), causal=causal, accumulate=accumulate)
        assert got is w
        b.cache.check()
        want, tol = old.double(), torch.zeros(w.shape, dtype=torch.float64)
        for s, (n, L) in enumerate(seqs):
            for p in range(L if n else 0):
                at = b.pages[s][p // page], p % page
                base = want[at] if accumulate and p < L - n else torch.zeros(Hkv, dtype=torch.float64)
                want[at] = base + sums[s][0][p]
                tol[at] = sums[s][1][p] + F32 * want[at]
        check_close(w, want, tol, f"weights, accumulate {accumulate}")


# ── eviction ─────────────────────────────────────────────────────────────────

EVICT = [  # sequences' lengths, D, Hkv, page, keep, first, last, layout
    ([1, 5], 128, 1, 16, 4, 0, 0, "heads"),
    ([400, 33, 0, 170, 64], 64, 2, 16, 64, 4, 16, "tokens"),
    ([300, 70, 64], 128, 3, 32, 50, 0, 50, "heads"),
    ([150, 9], 96, 5, 7, 20, 20, 0, "heads"),
    ([930, 230], 192, 2, 100, 201, 1, 32, "heads"),
    ([20, 1513, 800], 256, 4, 390, 391, 3, 7, "tokens"),
    ([5000, 4000, 1], 64, 1, 64, 2500, 4, 64, "heads"),
    ([900], 128, 2, 16, 1, 0, 0, "heads"),
    ([900], 128, 2, 16, 1, 0, 1, "heads"),
]


def _rows(b, s, name, table):
    """What a cache tensor holds of a sequence along a table's row, on the CPU."""
    t = getattr(b.cache, name).cpu()
    return torch.cat([t[p] for p in table]) if len(table) else t[0][:0]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("i", range(len(EVICT)))
def test_evict(gpu, i, bits, in_place):
    lens, D, Hkv, page, keep, first, last, layout = EVICT[i]
    seqs = [(0, L) for L in lens]
    news = [-(-min(L, keep) // page) for L in lens]
    b = Batch(gpu, seqs, D, Hkv, Hkv, page, BF if i % 2 else HF, bits=bits, layout=layout, seed=12, spare=sum(news) + 2)
    free = sorted(set(range(b.cache.num_pages)) - {p for x in b.pages for p in x})
    new_pages = []
    for n in news:
        new_pages.append(free[:n])
        free = free[n:]
    width = -(-keep // page) + 1
    new_table = torch.full((len(lens), width), -5, dtype=torch.int32)
    for s, x in enumerate(new_pages):
        new_table[s, :len(x)] = torch.tensor(x, dtype=torch.int32)
    w = b.cache.allocate_weights()
    old = torch.randint(0, 40, w.shape, generator=b.gen).float() * torch.rand(w.shape, generator=b.gen).round()    # many alike
    old[torch.rand(w.shape, generator=b.gen) < 0.05] = float("nan")
    old[torch.rand(w.shape, generator=b.gen) < 0.02] = float("-inf")
    old[torch.rand(w.shape, generator=b.gen) < 0.02] = -0.0
    w.copy_(old)
    names = ["k", "v"] + (["k_scale", "v_scale"] if bits == 4 else [])
    before = {n: getattr(b.cache, n).cpu().clone() for n in names}
    got, kept = lv.paged_kv_evict(b.cache, w, b.lens, b.table_dev, keep, first=first, last=last,
                                  new_table=None if in_place else new_table.to(gpu), return_kept=True)
    b.cache.check()
    assert got.tolist() == [min(L, keep) for L in lens]
    want = {n: x.clone() for n, x in before.items()}
    want_w, kept = old.clone(), kept.cpu()
    for s, L in enumerate(lens):
        to = b.pages[s] if in_place else new_pages[s]
        for h in range(Hkv):
            mine = torch.cat([old[p, :, h] for p in b.pages[s]])[:L] if L else old[0, :0, h]
            stay = ref.kept(mine, L, keep, first, last)
            assert kept[s, h].tolist() == stay + [-1] * (keep - len(stay)), (s, h)
            for i, p in enumerate(stay):
                a, z = (b.pages[s][p // page], p % page, h), (to[i // page], i % page, h)
                want_w[z] = old[a]
                for n in names:
                    want[n][z] = before[n][a]
    assert torch.equal(w.cpu().view(torch.int32), want_w.view(torch.int32))
    for n in names:
        a, z = getattr(b.cache, n).cpu(), want[n]
        bad = (a.view(torch.int16) != z.view(torch.int16)) if bits == 16 else a != z
        assert not bad.any(), (n, bad.sum().item())


# ── a run of them together ───────────────────────────────────────────────────


@pytest.mark.parametrize("bits", [16, 4])
def test_a_stream_that_selects_and_evicts(gpu, bits):
    """Steps of append, means, selection, attention, weights and eviction, against the same from the definitions: what
    each call is given is taken from the device, so that every step is held to its own arithmetic."""
    D, H, Hkv, page, block, keep = 64, 4, 2, 16, 8, 96
    g = torch.Generator().manual_seed(2)
    cache = lv.PagedKVCache.allocate(12, page, Hkv, D, bits=bits, device=gpu)
    means, weights = cache.allocate_means(block), cache.allocate_weights()
    table = torch.randperm(12, generator=g).to(torch.int32)[None, :10].to(gpu)
    L, seen = 0, 0
    of = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    for n in (40, 60, 1, 1, 30, 1, 7):
        k, v, q = (torch.randn(n, h, D, generator=g).to(BF).to(gpu) for h in (Hkv, Hkv, H))
        L += n
        call = (of(0, n), of(L), table)
        lv.paged_kv_append(cache, k, v, *call)
        lv.paged_kv_block_means(cache, means, call[1], table, cu_seqlens=call[0])
        b = Batch.__new__(Batch)
        gk, gv = lv.paged_kv_gather(cache, call[1], table, L, dtype=BF)
        b.K, b.V, b.seqs, b.ends, b.N, b.n_rows = [gk[0].double().cpu()], [gv[0].double().cpu()], [(n, L)], [0, n], n, n
        b.D, b.H, b.Hkv, b.ps, b.dtype, b.pages = D, H, Hkv, page, BF, [table[0].tolist()]
        rows = torch.stack([means[b.pages[0][j * block // page], j * block % page // block].cpu() for j in range(-(-L // block))])
        assert torch.allclose(rows.double(), ref.means(b, block)[0], rtol=1e-6, atol=1e-6)
        lists = lv.paged_kv_select(q, cache, means, *call, 5)
        assert torch.equal(lists.cpu(), ref.select(b, q, [rows], block, 5, 1, 1, 1, True))
        o = lv.paged_block_attention(q, cache, lists, block, *call)
        wo, _, tol, _ = ref.attention(b, q, lists, block, 1, True)
        check_close(o, wo, tol, "o")
        _, lse = lv.paged_attention(q, cache, *call, return_lse=True)
        before = torch.stack([weights[b.pages[0][p // page], p % page].cpu() for p in range(L)]).double()
        lv.paged_kv_weights(q, lse, cache, weights, *call)
        after = torch.stack([weights[b.pages[0][p // page], p % page].cpu() for p in range(L)]).double()
        w, wtol = ref.weights(b, q, lse, True)[0]
        before[L - n:] = 0
        check_close(after, before + w, wtol + F32 * (before + w), "weights")
        if L > keep:
            lens, kept = lv.paged_kv_evict(cache, weights, call[1], table, keep, first=2, last=16, return_kept=True)
            for h in range(Hkv):
                assert kept[0, h].tolist() == ref.kept(after[:, h], L, keep, 2, 16)
            L = keep
            assert lens.tolist() == [L]
            gk2, gv2 = lv.paged_kv_gather(cache, lens, table, L, dtype=BF)
            for h in range(Hkv):
                assert torch.equal(gk2[0, :, h], gk[0, kept[0, h].long(), h]) and torch.equal(gv2[0, :, h], gv[0, kept[0, h].long(), h])
            lv.paged_kv_block_means(cache, means, lens, table)
    cache.check()
