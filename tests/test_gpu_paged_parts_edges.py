"""The paged cache's parts where calls go wrong or are made in unusual ways: bad batches, refusals, streams, graphs, layouts,
long caches (see test_gpu_paged_parts.py)."""
import math

import pytest
import torch

import longvideosparseattention_amd as lv

import paged_parts_ref as ref
import paged_ref
from paged_ref import F32, Batch, check_close

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _lists(b, block, top, tile=1):
    """The first block, the rows' own and those before them."""
    todo, T = ref.tiles(b, tile)
    out = torch.full((T, b.Hkv, top), -1, dtype=torch.int32)
    for at, s, r0, r1, p0 in todo:
        own = (p0 + r1 - r0 - 1) // block
        ids = sorted({0, 1, 3, own, max(0, own - 2)} | set(range(max(p0, 0) // block, own + 1)))[-top:]
        ids = [i for i in ids if i * block < b.seqs[s][1]]
        out[at, :, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
    return out


def _step(b, q, means, weights, block=8, top=6, lists=None):
    """Everything that reads, on one batch."""
    out = {"blocks": lv.paged_kv_select(q, b.cache, means, *b.call(), top)}
    out["o"], out["lse"] = lv.paged_block_attention(q, b.cache, out["blocks"] if lists is None else lists, block, *b.call(),
                                                    return_lse=True)
    _, lse = lv.paged_attention(q, b.cache, *b.call(), return_lse=True)
    out["weights"] = lv.paged_kv_weights(q, lse, b.cache, weights, *b.call())
    return out


# ── what the device finds ────────────────────────────────────────────────────

SEQS = [(20, 90), (1, 40), (0, 30), (33, 33)]


def _batch(gpu, tile=1, **kw):
    b = Batch(gpu, SEQS, 64, 4, 2, 16, BF, seed=21, tail=2, **kw)
    return b, b.randn(b.N, 4, 64)


@pytest.mark.parametrize("tile", [1, 8, 64])
def test_a_bad_list_spoils_its_rows_alone(gpu, tile):
    b, q = _batch(gpu)
    lists = _lists(b, 8, 12, tile)
    clean, clean_lse = lv.paged_block_attention(q, b.cache, lists.to(gpu), 8, *b.call(), tile=tile, return_lse=True)
    todo = ref.tiles(b, tile)[0]
    g = b.H // b.Hkv
    for bad in ([0, 12, 13], [3, 3], [4, 2], [0, 1 << 28], [0x7fffffff]):    # behind the end, twice, descending
        spoiled = lists.clone()
        at, s, r0, r1, _ = todo[0]
        spoiled[at, 1, :] = -1
        spoiled[at, 1, :len(bad)] = torch.tensor(bad, dtype=torch.int32)
        o, lse = lv.paged_block_attention(q, b.cache, spoiled.to(gpu), 8, *b.call(), tile=tile, return_lse=True)
        with pytest.raises(ValueError, match="list of blocks"):
            b.cache.check()
        assert torch.isnan(o[r0:r1, g:]).all() and torch.isnan(lse[r0:r1, g:]).all()
        o[r0:r1, g:], lse[r0:r1, g:] = clean[r0:r1, g:], clean_lse[r0:r1, g:]
        assert torch.equal(o, clean) and torch.equal(lse, clean_lse)
        b.cache.check()


def test_numbers_behind_a_lists_end_are_not_read(gpu):
    b, q = _batch(gpu)
    lists = _lists(b, 8, 12)
    clean = lv.paged_block_attention(q, b.cache, lists.to(gpu), 8, *b.call())
    for at in range(lists.shape[0]):
        for h in range(2):
            n = (lists[at, h] >= 0).sum().item()
            lists[at, h, n + 1:] = 0x7ffffff0
    assert torch.equal(lv.paged_block_attention(q, b.cache, lists.to(gpu), 8, *b.call()), clean)
    b.cache.check()


@pytest.mark.parametrize("bits", [16, 4])
def test_bad_pages(gpu, bits):
    b, q = _batch(gpu, bits=bits)
    rows = ref.means(b, 8)
    means = b.cache.allocate_means(8)
    weights = b.cache.allocate_weights().fill_(2.0)
    lists = _lists(b, 8, 12).to(gpu)
    clean = lv.paged_block_attention(q, b.cache, lists, 8, *b.call())
    _, lse = lv.paged_attention(q, b.cache, *b.call(), return_lse=True)
    lv.paged_kv_weights(q, lse, b.cache, weights, *b.call())
    table = b.table_dev.clone()
    for bad in (-1, b.cache.num_pages, 0x7fffffff):
        table[0, 1] = bad                                  # positions 16 .. 31: blocks 2 and 3 of the first sequence
        call = (b.cu, b.lens, table)
        m = torch.full_like(means, 9.0)
        lv.paged_kv_block_means(b.cache, m, b.lens, table)
        with pytest.raises(ValueError, match="page number"):
            b.cache.check()
        for s, pages in enumerate(b.pages):
            for j in range(-(-SEQS[s][1] // 8)):
                if (s, j * 8 // 16) != (0, 1):
                    assert torch.allclose(m[pages[j * 8 // 16], j % 2].cpu().double(), rows[s][j], rtol=1e-5, atol=1e-5)
        assert (m[b.pages[0][1]] == 9.0).all()
        got = lv.paged_kv_select(q, b.cache, m, *call, 6)
        with pytest.raises(ValueError, match="page number"):
            b.cache.check()
        nan = [r.float() for r in rows]
        nan[0] = nan[0].clone()
        nan[0][2:4] = float("nan")
        have = [torch.stack([m[b.pages[s][j * 8 // 16], j % 2].cpu() for j in range(len(r))]) if len(r) else r for s, r in enumerate(nan)]
        have[0][2:4] = float("nan")
        assert torch.equal(got.cpu(), ref.select(b, q, have, 8, 6, 1, 1, 1, True))
        o = lv.paged_block_attention(q, b.cache, lists, 8, *call)
        with pytest.raises(ValueError, match="page number"):
            b.cache.check()
        hit = ((lists == 2) | (lists == 3)).any(-1)        # [rows, Hkv]
        hit[20:] = False
        assert hit.any()
        spoiled = hit.repeat_interleave(2, 1)
        assert torch.isnan(o[spoiled]).all() and torch.equal(o[~spoiled], clean[~spoiled])
        w = torch.full_like(weights, 2.0)
        lv.paged_kv_weights(q, lse, b.cache, w, *call)
        with pytest.raises(ValueError, match="page number"):
            b.cache.check()
        assert (w[b.pages[0][1]] == 2.0).all()
        w[b.pages[0][1]] = weights[b.pages[0][1]]
        assert torch.equal(w, weights)
        # eviction leaves the sequence alone and cuts the others
        held = [x for x in (b.cache.k, b.cache.v, b.cache.k_scale, b.cache.v_scale) if x is not None]
        before = [x.clone() for x in held]
        w = torch.rand(weights.shape, generator=b.gen).to(gpu)
        lens, kept = lv.paged_kv_evict(b.cache, w.clone(), b.lens, table, 25, return_kept=True)
        with pytest.raises(ValueError, match="page number"):
            b.cache.check()
        assert lens.tolist() == [90, 25, 25, 25] and (kept[0] == -1).all() and (kept[1:] >= 0).all()
        for p in b.pages[0]:
            assert all(torch.equal(x[p].view(torch.uint8), y[p].view(torch.uint8)) for x, y in zip(held, before))
        for x, y in zip(held, before):
            x.copy_(y)


@pytest.mark.parametrize("tile", [1, 8])
def test_bad_lengths_and_row_ranges(gpu, tile):
    b, q = _batch(gpu)
    means, weights = b.cache.allocate_means(8), b.cache.allocate_weights().fill_(2.0)
    lists = _lists(b, 8, 12, tile).to(gpu)
    lse = torch.zeros(b.N, 4, device=gpu)
    for length in (-1, 6 * 16 + 1, 0x7fffffff):
        lens = b.lens.clone()
        lens[0] = length
        call = (b.cu, lens, b.table_dev)
        m = torch.full_like(means, 9.0)
        w = weights.clone()
        lv.paged_kv_block_means(b.cache, m, lens, b.table_dev, cu_seqlens=b.cu)
        got = lv.paged_kv_select(q, b.cache, means, *call, 12, tile=tile)
        o = lv.paged_block_attention(q, b.cache, lists, 8, *call, tile=tile)
        lv.paged_kv_weights(q, lse, b.cache, w, *call)
        new, kept = lv.paged_kv_evict(b.cache, w.clone(), lens, b.table_dev, 1000, return_kept=True)
        with pytest.raises(ValueError, match="kv_lens"):
            b.cache.check()
        assert (m[b.pages[0]] == 9.0).all() and (w[b.pages[0]] == 2.0).all()
        T0 = 20 if tile == 1 else 3
        assert (got[:T0] == -1).all() and (got[20 if tile == 1 else 3] >= -1).all()
        assert torch.isnan(o[:20]).all() and not torch.isnan(o[20:54]).any()
        assert new.tolist() == [length, 40, 30, 33] and (kept[0] == -1).all()
        new = lv.paged_kv_evict(b.cache, w.clone(), lens, b.table_dev, 1, new_table=torch.full_like(b.table_dev[:, :1], 1000))
        assert new.tolist() == [0, 0, 0, 0]
        with pytest.raises(ValueError, match="page number.*kv_lens|kv_lens.*page number"):
            b.cache.check()
    for cu in ([0, 20, 19, 19, 54], [0, 20, 21, 21, 57], [-3, 20, 21, 21, 54]):
        call = (torch.tensor(cu, dtype=torch.int32, device=gpu), b.lens, b.table_dev)
        got = lv.paged_kv_select(q, b.cache, means, *call, 12, tile=tile)
        o, l = lv.paged_block_attention(q, b.cache, lists, 8, *call, tile=tile, return_lse=True)
        lv.paged_kv_weights(q, lse, b.cache, weights.clone(), *call)
        with pytest.raises(ValueError, match="cu_seqlens"):
            b.cache.check()
        assert (got == -1).all() and torch.isnan(o).all() and torch.isnan(l).all()


def test_more_rows_than_keys(gpu):
    """Rows before a sequence's first position attend nothing and change nothing."""
    b = Batch(gpu, [(9, 5), (40, 12)], 64, 4, 2, 16, BF, seed=22)
    q = b.randn(b.N, 4, 64)
    for tile in (1, 4, 64):
        lists = torch.full((ref.tiles(b, tile)[1], 2, 4), -1, dtype=torch.int32)
        for at, s, *_ in ref.tiles(b, tile)[0]:
            n = -(-b.seqs[s][1] // 4)
            lists[at, :, :n] = torch.arange(n, dtype=torch.int32)
        o, lse = lv.paged_block_attention(q, b.cache, lists.to(gpu), 4, *b.call(), tile=tile, return_lse=True)
        wo, wl, tol, ltol = ref.attention(b, q, lists, 4, tile, True)
        check_close(o, wo, tol, "o")
        check_close(lse, wl, ltol, "lse")
    _, lse = lv.paged_attention(q, b.cache, *b.call(), return_lse=True)
    w = b.cache.allocate_weights()
    lv.paged_kv_weights(q, lse, b.cache, w, *b.call())
    for s, (sums, tol) in enumerate(ref.weights(b, q, lse, True)):
        got = torch.stack([w[b.pages[s][p // 16], p % 16].cpu() for p in range(b.seqs[s][1])])
        check_close(got, sums, tol, "weights")


def test_new_pages_that_are_the_sequences_own(gpu):
    b = Batch(gpu, [(0, 90), (0, 60)], 64, 2, 2, 16, BF, seed=23, spare=12)
    w = b.cache.allocate_weights().copy_(torch.rand(b.cache.num_pages, 16, 2, generator=b.gen))
    free = sorted(set(range(b.cache.num_pages)) - {p for x in b.pages for p in x})
    table = torch.tensor([[free[0], b.pages[0][4]], [free[2], free[3]]], dtype=torch.int32, device=gpu)
    before = b.cache.k.clone()
    lens, kept = lv.paged_kv_evict(b.cache, w, b.lens, b.table_dev, 20, new_table=table, return_kept=True)
    with pytest.raises(ValueError, match="page number"):
        b.cache.check()
    assert lens.tolist() == [0, 20] and (kept[0] == -1).all()
    for p in [free[0], *b.pages[0]]:
        assert torch.equal(b.cache.k[p].view(torch.int16), before[p].view(torch.int16))


# ── refusals ─────────────────────────────────────────────────────────────────


def test_refusals(gpu):
    b, q = _batch(gpu)
    c, call = b.cache, b.call()
    means, weights, lists = c.allocate_means(8), c.allocate_weights(), _lists(b, 8, 12).to(gpu)
    lse = torch.zeros(b.N, 4, device=gpu)
    bad = [
        (lambda: c.allocate_means(5), ValueError, "do not divide"),
        (lambda: c.allocate_means(0), ValueError, "do not divide"),
        (lambda: lv.paged_kv_block_means(c, means[:, :, :, :32], b.lens, b.table_dev), ValueError, "means must be"),
        (lambda: lv.paged_kv_block_means(c, means.half(), b.lens, b.table_dev), ValueError, "means must be"),
        (lambda: lv.paged_kv_block_means(c, torch.zeros(c.num_pages, 3, 2, 64, device=gpu), b.lens, b.table_dev), ValueError, "dividing"),
        (lambda: lv.paged_kv_block_means(c, means[:1].expand(c.num_pages, 2, 2, 64), b.lens, b.table_dev), ValueError, "overlapping"),
        (lambda: lv.paged_kv_block_means(c, torch.zeros(c.num_pages, 2, 2, 65, device=gpu)[..., :64], b.lens, b.table_dev), ValueError, "16 bytes"),
        (lambda: lv.paged_kv_block_means(c, means.clone().requires_grad_(), b.lens, b.table_dev), RuntimeError, "gradient"),
        (lambda: lv.paged_kv_block_means(c, means, b.lens[:2], b.table_dev), ValueError, "sequences"),
        (lambda: lv.paged_kv_select(q.float(), c, means, *call, 6), TypeError, "dtype"),
        (lambda: lv.paged_kv_select(q[:, :3], c, means, *call, 6), ValueError, "multiple"),
        (lambda: lv.paged_kv_select(q, c, means, *call, 0), ValueError, "lists of 0"),
        (lambda: lv.paged_kv_select(q, c, means, *call, 1025), ValueError, "1 to 1024"),
        (lambda: lv.paged_kv_select(q, c, means, *call, 6, tile=0), ValueError, "tiles of 0"),
        (lambda: lv.paged_kv_select(q, c, means, *call, 6, first=6), ValueError, "do not fit"),
        (lambda: lv.paged_kv_select(q, c, means, *call, 6, last=-1), ValueError, "do not fit"),
        (lambda: lv.paged_kv_select(q, c, means, *call, 6, tile=64), ValueError, "do not fit"),
        (lambda: lv.paged_block_attention(q, c, lists, 5, *call), ValueError, "do not divide"),
        (lambda: lv.paged_block_attention(q, c, lists.long(), 8, *call), TypeError, "int32"),
        (lambda: lv.paged_block_attention(q, c, lists[1:], 8, *call), ValueError, "blocks must be"),
        (lambda: lv.paged_block_attention(q, c, lists, 8, *call, tile=2), ValueError, "blocks must be"),
        (lambda: lv.paged_block_attention(q, c, lists, 8, *call, scale=0.0), ValueError, "scale"),
        (lambda: lv.paged_block_attention(q, c, lists, 8, *call, out=q), ValueError, "share memory"),
        (lambda: lv.paged_block_attention(q, c, lists.cpu(), 8, *call), RuntimeError, "no CPU path"),
        (lambda: lv.paged_block_attention(q.clone().requires_grad_(), c, lists, 8, *call), RuntimeError, "gradient"),
        (lambda: lv.paged_kv_weights(q, lse[1:], c, weights, *call), ValueError, "lse must be"),
        (lambda: lv.paged_kv_weights(q, lse.double(), c, weights, *call), ValueError, "lse must be"),
        (lambda: lv.paged_kv_weights(q, lse, c, weights[:, :8], *call), ValueError, "weights must be"),
        (lambda: lv.paged_kv_weights(q, lse, c, weights[:1].expand(weights.shape), *call), ValueError, "overlapping"),
        (lambda: lv.paged_kv_weights(q, lse, c, weights, *call, scale=float("nan")), ValueError, "scale"),
        (lambda: lv.paged_kv_weights(q, lse, c, weights, *call, max_q_len=-1), ValueError, "max_q_len"),
        (lambda: lv.paged_kv_evict(c, weights, b.lens, b.table_dev, 0), ValueError, "tokens to keep"),
        (lambda: lv.paged_kv_evict(c, weights, b.lens, b.table_dev, 5, first=3, last=3), ValueError, "tokens to keep"),
        (lambda: lv.paged_kv_evict(c, weights, b.lens, b.table_dev, 20, new_table=b.table_dev), ValueError, "leave it out"),
        (lambda: lv.paged_kv_evict(c, weights, b.lens, b.table_dev, 20, new_table=b.table_dev[:, :1].clone()), ValueError, "do not hold"),
        (lambda: lv.paged_kv_evict(c, weights, b.lens, b.table_dev, 20, new_table=b.table_dev[:2].clone()), ValueError, "sequences"),
        (lambda: lv.paged_kv_evict(c, c.k[..., 0].float(), b.lens, b.table_dev[:, :, None], 20), TypeError, "2-D"),
    ]
    for i, (call_, kind, text) in enumerate(bad):
        with pytest.raises(kind, match=text):
            call_()
    # memory of the cache under another name
    flat = torch.zeros(c.num_pages * 2 * 16 * 64 * 3, dtype=BF, device=gpu)
    n = c.num_pages * 2 * 16 * 64
    own = lv.PagedKVCache(flat[:n].view(c.num_pages, 16, 2, 64), flat[n:2 * n].view(c.num_pages, 16, 2, 64))
    inside = flat.view(torch.float32)[:c.num_pages * 32].view(c.num_pages, 16, 2)
    with pytest.raises(ValueError, match="share memory with the cache"):
        lv.paged_kv_weights(q, lse, own, inside, *call)
    c.check()


# ── streams, graphs, compile ─────────────────────────────────────────────────


def _parts(gpu, n=1, seed=24, **kw):
    b = Batch(gpu, [(n, 300), (n, 77), (0, 0), (n, 160)], 64, 8, 2, 16, BF, seed=seed, **kw)
    means, weights = b.cache.allocate_means(8), b.cache.allocate_weights()
    lv.paged_kv_block_means(b.cache, means, b.lens, b.table_dev)
    weights.copy_(torch.rand(weights.shape, generator=b.gen))
    return b, means, weights


@pytest.mark.parametrize("n", [1, 24])
def test_a_captured_step_follows_its_batch(gpu, n):
    """One graph of the whole step; lengths, queries and lists change between its replays, eager work beside it."""
    b, means, weights = _parts(gpu, n)
    q = b.randn(b.N, 8, 64)
    for _ in range(2):
        want = _step(b, q, means.clone(), weights.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    w = weights.clone()
    kept_w = weights.clone()
    with torch.cuda.graph(graph):
        lv.paged_kv_block_means(b.cache, means, b.lens, b.table_dev, cu_seqlens=b.cu)
        got = _step(b, q, means, w)
        lens, kept = lv.paged_kv_evict(b.cache, kept_w, b.lens, b.table_dev, 120, first=2, last=8, return_kept=True)
    state = b.cache.k.clone(), b.cache.v.clone()
    for i in range(4):
        b.lens.copy_(torch.tensor([300 - 40 * i, 77 - i, 0, 160 - 3 * i], dtype=torch.int32))
        q.copy_(b.randn(b.N, 8, 64))
        b.cache.k.copy_(state[0])
        b.cache.v.copy_(state[1])
        w.copy_(weights)
        kept_w.copy_(weights)
        means2, w2, kw2 = means.clone(), weights.clone(), weights.clone()
        lv.paged_kv_block_means(b.cache, means2, b.lens, b.table_dev, cu_seqlens=b.cu)
        want = _step(b, q, means2, w2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in want:
            assert torch.equal(got[name].nan_to_num(7.0), want[name].nan_to_num(7.0)), (i, name)
        assert torch.equal(means.nan_to_num(7.0), means2.nan_to_num(7.0))
        after = b.cache.k.clone()
        b.cache.k.copy_(state[0])
        b.cache.v.copy_(state[1])
        lens2, kept2 = lv.paged_kv_evict(b.cache, kw2, b.lens, b.table_dev, 120, first=2, last=8, return_kept=True)
        assert torch.equal(lens, lens2) and torch.equal(kept, kept2) and torch.equal(kept_w.nan_to_num(3.0), kw2.nan_to_num(3.0))
        assert torch.equal(after.view(torch.int16), b.cache.k.view(torch.int16))
    b.cache.check()


def test_two_graphs_of_one_pool(gpu):
    a, am, aw = _parts(gpu, 24, seed=25)
    b, bm, bw = _parts(gpu, 1, seed=26)
    qa, qb = a.randn(a.N, 8, 64), b.randn(b.N, 8, 64)
    want = [_step(a, qa, am, aw.clone()), _step(b, qb, bm, bw.clone())]
    torch.cuda.synchronize()
    graphs, got, ws = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], [], [aw.clone(), bw.clone()]
    for g, x, q, m, w in ((graphs[0], a, qa, am, ws[0]), (graphs[1], b, qb, bm, ws[1])):
        with torch.cuda.graph(g, pool=None if not got else graphs[0].pool()):
            got.append(_step(x, q, m, w))
    for i in (0, 1, 0, 1, 1, 0):
        ws[i].copy_((aw, bw)[i])
        graphs[i].replay()
        torch.cuda.synchronize()
        for name in want[i]:
            assert torch.equal(got[i][name].nan_to_num(7.0), want[i][name].nan_to_num(7.0)), (i, name)


def test_two_streams_at_once(gpu):
    b, means, weights = _parts(gpu, 24)
    qs = [b.randn(b.N, 8, 64) for _ in range(2)]
    want = [_step(b, q, means, weights.clone()) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(_step(b, q, means, weights.clone()))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(g[n].nan_to_num(7.0), w[n].nan_to_num(7.0)) for n in w)


def test_inside_compile(gpu):
    b, means, weights = _parts(gpu)
    q = b.randn(b.N, 8, 64)

    def step(q, w):
        lists = lv.paged_kv_select(q + 0, b.cache, means, *b.call(), 6)
        o, lse = lv.paged_block_attention(q, b.cache, lists, 8, *b.call(), return_lse=True)
        return o * 2, lv.paged_kv_weights(q, lse, b.cache, w, *b.call()) + 1

    want = step(q, weights.clone())
    got = torch.compile(step, backend="eager")(q, weights.clone())
    assert all(torch.equal(g.nan_to_num(7.0), w.nan_to_num(7.0)) for g, w in zip(got, want))


# ── layouts and sizes ────────────────────────────────────────────────────────


def test_strided_tensors(gpu):
    """Queries, results, lists, means, weights and tables that are parts of larger tensors."""
    b, means, weights = _parts(gpu, 24)
    q = b.randn(b.N, 8, 64)
    lists = _lists(b, 8, 12)
    want = _step(b, q, means, weights.clone(), lists=lists.to(gpu))
    wide = torch.zeros(b.N, 16, 128, dtype=BF, device=gpu)
    q2 = wide[:, ::2, 32:96]
    q2.copy_(q)
    odd = torch.zeros(b.N, 8, 65, dtype=BF, device=gpu)[..., 1:]
    odd.copy_(q)
    big = torch.zeros(b.cache.num_pages + 3, 5, 4, 72, device=gpu)[2:-1, 1:5:2, ::2, 4:68]
    big.copy_(means)
    w2 = torch.zeros(3, b.cache.num_pages, 40, device=gpu).permute(1, 2, 0)[:, 4:36:2, :2]
    w2.copy_(weights)
    l2 = torch.full((b.N, 4, 16), 5, dtype=torch.int32, device=gpu)[:, 1:3, 2:14]
    l2.copy_(lists)
    table = torch.zeros(4, 2 * b.table.shape[1], dtype=torch.int32, device=gpu)[:, :b.table.shape[1]]
    table.copy_(b.table_dev)
    out = torch.full((b.N, 10, 64), 3.0, dtype=BF, device=gpu)[:, 1:9]
    for x in (q2, odd):
        b.table_dev = table
        assert torch.equal(lv.paged_kv_select(x, b.cache, big, *b.call(), 6), want["blocks"])
        o, lse = lv.paged_block_attention(x, b.cache, l2, 8, *b.call(), return_lse=True, out=out)
        assert o is out and torch.equal(o, want["o"]) and torch.equal(lse, want["lse"])
        _, dense = lv.paged_attention(x, b.cache, *b.call(), return_lse=True)
        w2.copy_(weights)
        assert torch.equal(lv.paged_kv_weights(x, dense.T.contiguous().T, b.cache, w2, *b.call()), want["weights"])
    m2 = torch.zeros_like(big)
    big.zero_()
    lv.paged_kv_block_means(b.cache, big, b.lens, b.table_dev)
    lv.paged_kv_block_means(b.cache, m2, b.lens, b.table_dev)
    assert torch.equal(big.nan_to_num(3.0), m2.nan_to_num(3.0))
    a1, a2 = weights.clone(), w2.copy_(weights)
    k = b.cache.k.clone()
    one = lv.paged_kv_evict(b.cache, a1, b.lens, b.table_dev, 50, return_kept=True)
    k1 = b.cache.k.clone()
    b.cache.k.copy_(k)
    two = lv.paged_kv_evict(b.cache, a2, b.lens, b.table_dev, 50, return_kept=True)
    assert all(torch.equal(x, y) for x, y in zip(one, two)) and torch.equal(a1, a2)
    assert torch.equal(b.cache.k.view(torch.int16), k1.view(torch.int16))


@pytest.mark.parametrize("tile", [50, 1 << 20, (1 << 31) - 1])
def test_tiles_longer_than_a_sequence(gpu, tile):
    b = Batch(gpu, [(30, 200), (12, 12), (0, 0), (1, 90)], 64, 4, 2, 200, BF, seed=27)
    q = b.randn(b.N, 4, 64)
    means = b.cache.allocate_means(200)
    rows = [torch.randn(-(-L // 200), 2, 64, generator=b.gen) for _, L in b.seqs]
    means.copy_(ref.paged(b, rows, 200, 0.0, means))
    if tile == 50:
        assert torch.equal(lv.paged_kv_select(q, b.cache, means, *b.call(), 4, tile=tile).cpu(),
                           ref.select(b, q, rows, 200, 4, tile, 1, 1, True))
    lists = lv.paged_kv_select(q, b.cache, means, *b.call(), 1, tile=tile, first=0, last=0)
    assert torch.equal(lists.cpu(), ref.select(b, q, rows, 200, 1, tile, 0, 0, True))
    o = lv.paged_block_attention(q, b.cache, lists, 200, *b.call(), tile=tile)
    wo, _, tol, _ = ref.attention(b, q, lists, 200, tile, True)
    check_close(o, wo, tol, "o")


@pytest.mark.parametrize("blocks", [700, 1000, 1024, 1025])
def test_selection_among_about_a_thousand_blocks(gpu, blocks):
    """The table's width decides which kernel ranks: sixteen lists at once up to 1024 blocks, in 131 KB of LDS."""
    b = Batch(gpu, [(100, 4 * blocks - 1)], 64, 16, 16, 4, BF, seed=28)
    rows = [torch.randn(blocks, 16, 64, generator=b.gen)]
    means = b.cache.allocate_means(4)
    means.copy_(ref.paged(b, rows, 4, 0.0, means))
    q = b.randn(100, 16, 64)
    for top in (20, 1000):
        assert torch.equal(lv.paged_kv_select(q, b.cache, means, *b.call(), top).cpu(), ref.select(b, q, rows, 4, top, 1, 1, 1, True))


def test_rows_of_many_sequences(gpu):
    """More sequences than a wave has lanes, and more work-groups than units."""
    seqs = [(1 + i % 3, 3 + (7 * i) % 60) for i in range(150)]
    b = Batch(gpu, seqs, 64, 4, 2, 8, HF, seed=29)
    q = b.randn(b.N, 4, 64)
    rows = ref.means(b, 4)
    means = b.cache.allocate_means(4)
    lv.paged_kv_block_means(b.cache, means, b.lens, b.table_dev)
    have = [torch.stack([means[b.pages[s][j * 4 // 8], j % 2].cpu() for j in range(len(r))]) for s, r in enumerate(rows)]
    for tile in (1, 2):
        lists = lv.paged_kv_select(q, b.cache, means, *b.call(), 5, tile=tile)
        assert torch.equal(lists.cpu(), ref.select(b, q, have, 4, 5, tile, 1, 1, True))
        o = lv.paged_block_attention(q, b.cache, lists, 4, *b.call(), tile=tile)
        wo, _, tol, _ = ref.attention(b, q, lists, 4, tile, True)
        check_close(o, wo, tol, "o")
    _, lse = lv.paged_attention(q, b.cache, *b.call(), return_lse=True)
    w = b.cache.allocate_weights()
    lv.paged_kv_weights(q, lse, b.cache, w, *b.call())
    want, wtol = torch.zeros(w.shape, dtype=torch.float64), torch.zeros(w.shape, dtype=torch.float64)
    for s, (sums, tol) in enumerate(ref.weights(b, q, lse, True)):
        for p in range(seqs[s][1]):
            want[b.pages[s][p // 8], p % 8], wtol[b.pages[s][p // 8], p % 8] = sums[p], tol[p]
    check_close(w, want, wtol, "weights")
    many = b.cache.allocate_weights()
    lv.paged_kv_weights(q, lse, b.cache, many, *b.call(), max_q_len=1000)        # the kernel for many rows
    check_close(many, want, wtol, "weights by the rows' kernel")
    lens, kept = lv.paged_kv_evict(b.cache, w, b.lens, b.table_dev, 9, last=2, return_kept=True)
    assert lens.tolist() == [min(9, L) for _, L in seqs]
    for s, (_, L) in enumerate(seqs):
        got = want.new_tensor([[many[b.pages[s][p // 8], p % 8, h].item() for h in range(2)] for p in range(L)])
        first = torch.stack([w.cpu()[b.pages[s][i // 8], i % 8] for i in range(min(9, L))])
        for h in range(2):
            ids = kept[s, h][:min(9, L)].tolist()
            assert ids == sorted(set(ids)) and all(p in ids for p in range(max(0, L - 2), L))
            assert torch.allclose(first[:, h].double(), got[ids, h], rtol=1e-5, atol=1e-6)


def test_rows_that_share_their_work_groups_keys(gpu):
    """Prompts over few keys: several work-groups add to one key's weight; the same bits every time."""
    b = Batch(gpu, [(500, 600)], 128, 16, 1, 64, BF, seed=30)
    q = b.randn(b.N, 16, 128)
    _, lse = lv.paged_attention(q, b.cache, *b.call(), return_lse=True)
    got = [lv.paged_kv_weights(q, lse, b.cache, b.cache.allocate_weights(), *b.call()) for _ in range(3)]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    sums, tol = ref.weights(b, q, lse, True)[0]
    check_close(torch.stack([got[0][b.pages[0][p // 64], p % 64].cpu() for p in range(600)]), sums, tol, "weights")
    total = got[0].double().sum().item()
    assert abs(total - 500 * 16) < 500 * 16 * 2e-5        # every row gives 1 in all


@pytest.mark.parametrize("page", [64, 4096])
def test_a_cache_past_32_bits(gpu, page):
    """17 million keys of one head: offsets of keys, values, means and positions past 2^31 bytes."""
    D, L = 64, 17 * 1000 * 1000
    P = -(-L // page)
    k = torch.zeros(P, page, 1, D, dtype=BF, device=gpu)
    v = torch.zeros(P, page, 1, D, dtype=BF, device=gpu)
    cache = lv.PagedKVCache(k, v)
    g = torch.Generator().manual_seed(5)
    table = torch.randperm(P, generator=g).to(torch.int32)
    of = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    call = (of(0, 1), of(L), table.to(gpu)[None])
    block = 64
    hot = sorted({5, 99999, L // block // 2, L // block - 2, (L - 1) // block})
    at = lambda p: (int(table[p // page]), p % page)  # noqa: E731
    K, V = {}, {}
    for j in hot:
        n = min(block, L - j * block)
        K[j], V[j] = torch.randn(n, D, generator=g).to(BF), torch.randn(n, D, generator=g).to(BF)
        K[j][:, 0] = 3.0
        pg, sl = at(j * block)
        k[pg, sl:sl + n, 0], v[pg, sl:sl + n, 0] = K[j].to(gpu), V[j].to(gpu)
    means = cache.allocate_means(block)
    lv.paged_kv_block_means(cache, means, call[1], call[2])
    for j in hot:
        pg, sl = at(j * block)
        assert torch.allclose(means[pg, sl // block, 0].cpu().double(), K[j].double().mean(0), rtol=1e-5, atol=1e-6)
    q = torch.zeros(1, 2, D, dtype=BF, device=gpu)
    q[:, :, 0] = 1.0
    lists = lv.paged_kv_select(q, cache, means, *call, len(hot), first=0, last=1)
    assert lists.tolist() == [[hot]]
    q += torch.randn(q.shape, generator=g).to(BF).to(gpu) * 0.5
    o, lse = lv.paged_block_attention(q, cache, lists, block, *call, return_lse=True)
    Ks, Vs = torch.cat([K[j] for j in hot]).double(), torch.cat([V[j] for j in hot]).double()
    z = q[0].double().cpu() @ Ks.T / 8
    assert torch.allclose(lse[0].double().cpu(), torch.logsumexp(z, -1), atol=1e-4)
    assert torch.allclose(o[0].double().cpu(), torch.softmax(z, -1) @ Vs, atol=2e-2)
    w = cache.allocate_weights()
    _, dense = lv.paged_attention(q, cache, *call, return_lse=True)
    lv.paged_kv_weights(q, dense, cache, w, *call)
    pos = torch.tensor([j * block + i for j in hot for i in range(min(block, L - j * block))])
    got = torch.stack([w[at(int(p))] for p in pos])[:, 0].double().cpu()
    want = torch.exp(z - dense[0].double().cpu()[:, None]).sum(0)
    assert torch.allclose(got, want, rtol=1e-4, atol=0)
    keep = 2 * len(pos)
    w.zero_()
    for p in pos.tolist():
        w[at(p)] = 1.0
    lens, kept = lv.paged_kv_evict(cache, w, call[1], call[2], keep, first=1, last=1, return_kept=True)
    ids = kept[0, 0].cpu()
    rest = [p for p in range(keep) if p not in set(pos.tolist())][:keep - len(pos)]
    expect = sorted(set(pos.tolist()) | set(rest))
    assert lens.tolist() == [keep] and ids.tolist() == expect
    where = {p: i for i, p in enumerate(expect)}
    for j in hot:
        for i in (0, len(K[j]) - 1):
            assert torch.equal(k[at(where[j * block + i])][0].cpu(), K[j][i]) and torch.equal(v[at(where[j * block + i])][0].cpu(), V[j][i])
    cache.check()


def test_nothing_to_do(gpu):
    b = Batch(gpu, [(0, 0), (0, 20)], 64, 4, 2, 16, BF, seed=31)
    q = b.randn(0, 4, 64)
    means, weights = b.cache.allocate_means(8), b.cache.allocate_weights().fill_(2.0)
    lv.paged_kv_block_means(b.cache, means, b.lens, b.table_dev, cu_seqlens=b.cu)
    assert (means == 0).all()
    assert lv.paged_kv_select(q, b.cache, means, *b.call(), 4).shape == (0, 2, 4)
    lists = lv.paged_kv_select(q, b.cache, means, *b.call(), 4, tile=16, first=1, last=1)
    assert lists.shape == (2, 2, 4) and (lists == -1).all()
    assert lv.paged_block_attention(q, b.cache, lists, 8, *b.call(), tile=16).shape == (0, 4, 64)
    lv.paged_kv_weights(q, torch.zeros(0, 4, device=gpu), b.cache, weights, *b.call())
    assert (weights == 2.0).all()
    none = torch.zeros(0, 3, dtype=torch.int32, device=gpu)
    empty = (torch.zeros(1, dtype=torch.int32, device=gpu), none[:, 0], none)
    q = b.randn(3, 4, 64)
    lv.paged_kv_block_means(b.cache, means, empty[1], none)
    assert (lv.paged_kv_select(q, b.cache, means, *empty, 4) == -1).all()
    o, lse = lv.paged_block_attention(q, b.cache, torch.zeros(3, 2, 4, dtype=torch.int32, device=gpu), 8, *empty, return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()
    lv.paged_kv_weights(q, lse, b.cache, weights, *empty)
    lens, kept = lv.paged_kv_evict(b.cache, weights, empty[1], none, 4, return_kept=True)
    assert lens.shape == (0,) and kept.shape == (0, 2, 4)
    b.cache.check()
