"""Every instantiation of the paged cache's parts that sizes choose and test_gpu_paged_parts.py's tables do not reach: tiles
of 16, 32 and 128 rows, joined and not, few and many rows' weights at every head size, eviction by the ranks a thread
holds."""
import pytest
import torch

import longvideosparseattention_amd as lv

import paged_parts_ref as ref
from paged_ref import F32, Batch, check_close
from test_gpu_paged_parts import _lists

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16

# rows of a list (tile x heads of a key head): up to 16, 32, more
ATTEND = [  # sequences, D, H, Hkv, page, block, top, tile, causal, layout
    ([(9, 700), (1, 40), (33, 33)], 96, 3, 1, 24, 12, 40, 7, True, "heads"),
    ([(9, 700), (1, 40), (33, 33)], 96, 6, 1, 24, 12, 40, 5, True, "tokens"),
    ([(90, 700), (1, 40), (33, 33)], 96, 6, 2, 24, 12, 40, 30, True, "heads"),
    ([(200, 500)], 96, 2, 2, 50, 50, 6, 200, False, "heads"),
    ([(9, 900), (2, 300), (0, 5)], 192, 4, 2, 20, 20, 30, 4, True, "heads"),
    ([(9, 900), (2, 300), (0, 5)], 192, 8, 2, 20, 10, 60, 8, True, "tokens"),
    ([(9, 900), (2, 300), (0, 5)], 192, 8, 2, 20, 10, 60, 8, False, "heads"),
    ([(1, 900), (1, 300), (1, 1)], 192, 32, 1, 64, 16, 30, 1, True, "heads"),
    ([(9, 900), (2, 300), (40, 40)], 256, 6, 3, 32, 16, 50, 4, True, "heads"),
    ([(9, 900), (2, 300), (40, 40)], 256, 8, 1, 32, 16, 50, 4, True, "tokens"),
    ([(9, 900), (2, 300), (40, 40)], 256, 8, 1, 32, 16, 50, 4, False, "heads"),
    ([(1, 900), (1, 300), (1, 17)], 256, 20, 1, 64, 16, 30, 1, True, "heads"),
    ([(9, 700), (1, 40), (33, 33)], 64, 6, 1, 24, 12, 40, 5, False, "tokens"),
    ([(9, 700), (1, 40), (33, 33)], 128, 6, 1, 24, 12, 40, 5, False, "tokens"),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("i", range(len(ATTEND)))
def test_block_attention(gpu, i, dtype, bits):
    seqs, D, H, Hkv, page, block, top, tile, causal, layout = ATTEND[i]
    b = Batch(gpu, seqs, D, H, Hkv, page, dtype, bits=bits, layout=layout, tail=1, seed=50)
    q = b.randn(b.N, H, D, gain=1.5)
    lists = _lists(b, block, top, tile, causal, b.gen)
    o, lse = lv.paged_block_attention(q, b.cache, lists.to(gpu), block, *b.call(), tile=tile, causal=causal, return_lse=True)
    b.cache.check()
    wo, wl, tol, ltol = ref.attention(b, q, lists, block, tile, causal)
    check_close(o, wo, tol, "o")
    check_close(lse, wl, ltol, "lse")
    for _ in range(2):                       # the same bits every time
        o2, lse2 = lv.paged_block_attention(q, b.cache, lists.to(gpu), block, *b.call(), tile=tile, causal=causal, return_lse=True)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("tile,H", [(4, 4), (4, 8), (16, 4)])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_keys_that_are_not_attended_have_no_effect(gpu, D, tile, H):
    """Infinities and NaN in blocks of no list, and in future positions of listed ones, for tiles of 16, 32 and 64 rows."""
    L, block = 420, 12
    b = Batch(gpu, [(61, L)], D, H, 1, 24, BF, seed=51)
    q = b.randn(b.N, H, D)
    lists = torch.full((ref.tiles(b, tile)[1], 1, 9), -1, dtype=torch.int32)
    for at, s, r0, r1, p0 in ref.tiles(b, tile)[0]:
        own = (p0 + r1 - r0 - 1) // block
        ids = sorted({0, 5, 9, max(0, own - 2)} | set(range(p0 // block, own + 1)))
        lists[at, 0, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
    call = lambda: lv.paged_block_attention(q, b.cache, lists.to(gpu), block, *b.call(), tile=tile)  # noqa: E731
    clean = call()
    for j in (1, 4, 7, 10):
        at = b.pages[0][j * block // 24], slice(j * block % 24, j * block % 24 + block)
        b.cache.k[at], b.cache.v[at] = float("nan"), float("inf")
    assert torch.equal(call(), clean)
    for p, k, v in ((L - 1, "nan", "-inf"), (L - 7, "inf", "nan")):      # attended from its own row on
        b.cache.k[b.pages[0][p // 24], p % 24] = float(k)
        b.cache.v[b.pages[0][p // 24], p % 24] = float(v)
    got = call()
    assert torch.equal(got[:-7], clean[:-7]) and torch.isnan(got[-1]).all()


WEIGHTS = [  # sequences, D, H, Hkv, page, causal, layout, most rows of a sequence
    ([(1, 700), (1, 33), (0, 9), (1, 1)], 192, 8, 2, 16, True, "heads", 1),
    ([(1, 5000), (1, 33), (0, 9), (1, 1)], 192, 40, 2, 50, True, "tokens", 1),
    ([(7, 700), (3, 3), (2, 1)], 192, 6, 1, 16, False, "heads", 7),
    ([(1, 700), (1, 33), (0, 9), (1, 1)], 256, 8, 2, 16, True, "heads", 1),
    ([(1, 5000), (1, 33), (0, 9), (1, 1)], 256, 40, 2, 50, True, "tokens", 1),
    ([(7, 700), (3, 3), (2, 1)], 256, 6, 1, 16, False, "heads", 7),
    ([(120, 600), (70, 70), (0, 3)], 96, 3, 3, 20, True, "heads", 120),
    ([(120, 600), (70, 70), (0, 3)], 96, 10, 2, 7, True, "tokens", 120),      # rows shared by several work-groups
    ([(200, 260)], 96, 12, 1, 64, False, "heads", 200),
    ([(50, 90), (1, 40)], 192, 12, 2, 20, True, "tokens", 50),
    ([(50, 90), (1, 40)], 256, 12, 2, 20, True, "tokens", 50),
    ([(1, 3000), (1, 40)], 96, 24, 1, 24, True, "heads", 1),
    ([(1, 3000), (1, 40)], 128, 24, 1, 24, True, "heads", 1),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("i", range(len(WEIGHTS)))
def test_weights(gpu, i, dtype, bits):
    seqs, D, H, Hkv, page, causal, layout, most = WEIGHTS[i]
    b = Batch(gpu, seqs, D, H, Hkv, page, dtype, bits=bits, layout=layout, tail=2, seed=52)
    q = b.randn(b.N, H, D, gain=1.5)
    _, lse = lv.paged_attention(q, b.cache, *b.call(), causal=causal, return_lse=True)
    sums = ref.weights(b, q, lse, causal)
    old = torch.rand(b.cache.allocate_weights().shape, generator=b.gen)
    for accumulate in (True, False):
        got = []
        for hint in (most, most, None):
            w = b.cache.allocate_weights().copy_(old)
            got.append(lv.paged_kv_weights(q, lse, b.cache, w, *b.call(), causal=causal, accumulate=accumulate, max_q_len=hint))
        b.cache.check()
        assert torch.equal(got[0], got[1])
        want, tol = old.double(), torch.zeros(old.shape, dtype=torch.float64)
        for s, (n, L) in enumerate(seqs):
            for p in range(L if n else 0):
                at = b.pages[s][p // page], p % page
                base = want[at] if accumulate and p < L - n else torch.zeros(Hkv, dtype=torch.float64)
                want[at] = base + sums[s][0][p]
                tol[at] = sums[s][1][p] + F32 * want[at]
        for w in got[1:]:
            check_close(w, want, tol, f"weights, accumulate {accumulate}")


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("columns,L", [(64, 4096), (65, 4097), (256, 16384), (257, 16385), (300, 19000), (512, 32768), (513, 32769),
                                       (700, 2500)])
def test_evict_by_the_tables_room(gpu, columns, L, in_place):
    """Pages of 64: 4, 16 and 32 ranks a thread, and none, with sequences that fill the table and that do not."""
    keep, page, lens = L // 2 + 3, 64, [L, 700, 3]
    seqs = [(0, x) for x in lens]
    b = Batch(gpu, seqs, 64, 2, 2, page, BF, seed=53, spare=sum(-(-min(x, keep) // page) for x in lens), extra_columns=columns - -(-L // page))
    assert b.table.shape[1] == columns
    free = iter(sorted(set(range(b.cache.num_pages)) - {p for x in b.pages for p in x}))
    to = torch.full((3, -(-keep // page)), -1, dtype=torch.int32)
    for s, x in enumerate(lens):
        for i in range(-(-min(x, keep) // page)):
            to[s, i] = next(free)
    old = torch.randint(0, 3000, (b.cache.num_pages, page, 2), generator=b.gen).float()           # some alike
    w = b.cache.allocate_weights().copy_(old)
    k = b.cache.k.cpu()
    got, kept = lv.paged_kv_evict(b.cache, w, b.lens, b.table_dev, keep, first=4, last=9, new_table=None if in_place else to.to(gpu),
                                  return_kept=True)
    b.cache.check()
    assert got.tolist() == [min(x, keep) for x in lens]
    now, w, kept = b.cache.k.cpu(), w.cpu(), kept.cpu()
    for s, x in enumerate(lens):
        at = torch.tensor(b.pages[s] if in_place else to[s].tolist())
        for h in range(2):
            was = torch.tensor(b.pages[s])[torch.arange(x) // page], torch.arange(x) % page, h
            stay = ref.kept(old[was], x, keep, 4, 9)
            assert kept[s, h].tolist() == stay + [-1] * (keep - len(stay))
            i = torch.arange(len(stay))
            here = at[i // page], i % page, h
            assert torch.equal(w[here], old[was][stay])
            assert torch.equal(now[here].view(torch.int16), k[was][stay].view(torch.int16))


@pytest.mark.parametrize("tile", [1, 2, 8])
def test_a_bad_length_leaves_the_other_sequences_lists(gpu, tile):
    seqs = [(20, 90), (1, 40), (0, 30), (33, 33)]
    for H in (2, 64):                        # a work-group a list; sixteen lists together
        b = Batch(gpu, seqs, 64, H, H, 16, HF, seed=54, tail=2)
        q = b.randn(b.N, H, 64)
        means = b.cache.allocate_means(8)
        lv.paged_kv_block_means(b.cache, means, b.lens, b.table_dev)
        clean = lv.paged_kv_select(q, b.cache, means, *b.call(), 4, tile=tile)
        assert (clean[0] >= 0).all()
        for at, rows in ((0, (0, 20)), (1, (20, 21)), (3, (21, 54))):
            want = clean.clone()
            if tile == 1:
                want[rows[0]:rows[1]] = -1
            else:
                first = rows[0] // tile + at
                want[first:first - (-(rows[1] - rows[0]) // tile)] = -1
            for length in (-1, 6 * 16 + 1, 0x7fffffff):
                lens = b.lens.clone()
                lens[at] = length
                got = lv.paged_kv_select(q, b.cache, means, b.cu, lens, b.table_dev, 4, tile=tile)
                with pytest.raises(ValueError, match="kv_lens"):
                    b.cache.check()
                assert torch.equal(got, want), (H, at, length)
