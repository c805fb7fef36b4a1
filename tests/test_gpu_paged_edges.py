"""The paged cache where calls leave the usual path: padded batches with the caller's result, arguments that the
device finds wrong, values that a type cannot hold, far larger and smaller weights, many sequences, other streams."""
import ctypes

import pytest
import torch

import longvideosparseattention_amd as lv
from longvideosparseattention_amd import _capi, hip_ops, paged_kv

import paged_ref as ref
from paged_ref import Batch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
ROOM = 700000        # keys a page table may have room for: chunks then run on the kernels of long caches


# ── rows of no sequence ──────────────────────────────────────────────────────


@pytest.mark.parametrize("n,room", [(1, 0), (20, 0), (60, ROOM), (150, ROOM)])
def test_lse_of_rows_of_no_sequence_beside_out(gpu, n, room):
    """A padded batch with the caller's result: its rows of no sequence stay as they were, their lse is -inf."""
    b = Batch(gpu, [(n, 200), (n, 170)], 128, 4, 2, 16, BF, tail=5, extra_columns=room // 16)
    q = b.randn(b.N, 4, 128)
    want = lv.paged_attention(q, b.cache, *b.call(), max_q_len=n, return_lse=True)
    out = torch.full_like(q, 9.0)
    held = [torch.full((b.N, 4), 5.0, device=gpu) for _ in range(8)]      # what a new tensor finds in its memory
    del held
    o, lse = lv.paged_attention(q, b.cache, *b.call(), max_q_len=n, out=out, return_lse=True)
    assert o is out and (o[b.n_rows:] == 9.0).all() and (lse[b.n_rows:] == float("-inf")).all()
    assert torch.equal(o[:b.n_rows], want[0][:b.n_rows]) and torch.equal(lse, want[1])
    lv.paged_attention(q, b.cache, *b.call(), max_q_len=n, out=out.fill_(3.0))
    assert (out[b.n_rows:] == 3.0).all() and torch.equal(out[:b.n_rows], want[0][:b.n_rows])
    b.cache.check()


# ── row ranges that do not ascend within the rows ────────────────────────────


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("D,n,room", [(128, 1, 0), (128, 20, 0), (64, 60, ROOM), (128, 150, ROOM), (256, 60, ROOM)])
def test_bad_row_ranges_spoil_the_whole_result(gpu, D, n, room, bits):
    """Which rows are whose is unknown: every row is NaN, none is left unwritten, with the caller's result or a new one."""
    b = Batch(gpu, [(n, 150), (n, 160), (n, 153)], D, 4, 2, 16, BF, bits=bits, extra_columns=room // 16)
    q = b.randn(b.N, 4, D)
    good = lv.paged_attention(q, b.cache, *b.call(), max_q_len=n, return_lse=True)
    big = 2 ** 31 - 1
    for cu in ([0, n, 2 * n, 3 * n + 50], [0, 2 * n, n, 3 * n], [-5, n, 2 * n, 3 * n], [0, n, big, 3 * n], [0, 3 * n, 0, 3 * n],
               [3 * n, 0, 3 * n, 0], [2 * n, n, -1, 0], [-2 ** 31, big, -2 ** 31, big], [big, big, big, big], [0, 3 * n, n, n]):
        cu_dev = torch.tensor(cu, dtype=torch.int32, device=gpu)
        for out in (None, torch.zeros_like(q)):
            o, lse = lv.paged_attention(q, b.cache, cu_dev, b.lens, b.table_dev, max_q_len=n, out=out, return_lse=True)
            assert torch.isnan(o).all() and torch.isnan(lse).all(), cu
            with pytest.raises(ValueError, match="cu_seqlens"):
                b.cache.check()
    o, lse = lv.paged_attention(q, b.cache, *b.call(), max_q_len=n, return_lse=True)
    assert torch.equal(o, good[0]) and torch.equal(lse, good[1])
    b.cache.check()


@pytest.mark.parametrize("where", [3, 70, 199])
@pytest.mark.parametrize("room", [0, ROOM])
def test_a_bad_row_range_among_many_sequences(gpu, room, where):
    """Of 200 sequences one range descends, in whichever 64 of them: the same."""
    B = 200
    b = Batch(gpu, [(1, 5 + i % 9) for i in range(B)], 64, 2, 1, 8, BF, extra_columns=min(room, 20000) // 8)
    q = b.randn(b.N, 2, 64)
    kw = {"max_q_len": 100} if room else {"max_q_len": 1}
    cu = b.cu.clone()
    cu[where + 1] = cu[where] - 1 if where < B - 1 else b.N + 1
    o, lse = lv.paged_attention(q, b.cache, cu, b.lens, b.table_dev, return_lse=True, **kw)
    assert torch.isnan(o).all() and torch.isnan(lse).all()
    with pytest.raises(ValueError, match="cu_seqlens"):
        b.cache.check()


@pytest.mark.parametrize("B,where", [(3, 1), (150, 10), (150, 100), (150, 149)])
def test_an_append_reports_every_bad_row_range(gpu, B, where):
    """A descending range without rows of its own is reported too; rows are the first sequence's that holds them."""
    b = Batch(gpu, [(2, 8)] * B, 64, 1, 1, 8, BF)
    k, v, q = b.randn(b.N, 1, 64), b.randn(b.N, 1, 64), b.randn(b.N, 1, 64)
    cu = b.cu.clone()
    cu[where + 1] = cu[where] - 1 if where < B - 1 else 2 ** 31 - 1
    before = b.cache.k.clone()
    qo = lv.paged_kv_append(b.cache, k, v, cu, b.lens, b.table_dev, q=q)
    with pytest.raises(ValueError, match="cu_seqlens"):
        b.cache.check()
    host = cu.tolist()
    for t in range(b.N):
        s = next((s for s in range(B) if host[s] <= t < host[s + 1]), None)
        if s is None:
            continue
        if host[s + 1] > b.N:                             # its own range is bad: left out
            assert torch.isnan(qo[t]).all()
            page = b.pages[s][0]
            assert torch.equal(b.cache.k[page].nan_to_num(3.0), before[page].nan_to_num(3.0))
        else:
            slot = 8 - (host[s + 1] - host[s]) + t - host[s]
            assert torch.equal(b.cache.k[b.pages[s][0], slot], k[t]) and torch.equal(qo[t], q[t])


# ── 4-bit values beyond the range of 16 bits ─────────────────────────────────


@pytest.mark.parametrize("dtype,byte", [(HF, 141), (HF, 143), (HF, 254), (BF, 253), (BF, 254)])
@pytest.mark.parametrize("n,D,room", [(4, 128, 0), (20, 192, 0), (60, 64, ROOM), (60, 256, ROOM), (150, 96, ROOM), (150, 64, ROOM),
                                      (150, 128, ROOM), (150, 192, ROOM)])
def test_4_bit_values_beyond_the_types_range(gpu, n, D, room, dtype, byte):
    """Scales whose larger values the queries' type holds as infinities (as the gather returns them): without effect on
    rows that do not attend the key, in the result of those that do."""
    L = n + 60
    b = Batch(gpu, [(n, L)], D, 2, 1, 16, dtype, bits=4, extra_columns=room // 16)
    q = b.randn(n, 2, D)
    b.V[0] *= 0.25                                        # no sums of its own beyond the type's range
    b.cache.v_scale.copy_(torch.where(b.cache.v_scale == 255, 255, b.cache.v_scale - 2))
    clean, _ = lv.paged_attention(q, b.cache, *b.call(), max_q_len=n, return_lse=True)
    where = L - n + n // 2                                # attended from row n / 2 on
    page, slot = b.pages[0][where // 16], where % 16
    b.cache.v_scale[page, slot, 0, 1] = byte
    codes = b.cache.v[page, slot, 0, 16:32].cpu()
    codes[0], codes[1], codes[2] = 0x7F, 0x10, 0x02        # -6 and 6, 0 and 0.5, 1 and 0
    b.cache.v[page, slot, 0, 16:32] = codes.to(gpu)
    held = ref.dequantize(codes, torch.tensor([byte], dtype=torch.uint8)).to(dtype).double()
    assert held[:2].isinf().all() and held[2] == 0
    b.V[0][where, 0, 32:64] = held
    kept, _ = lv.paged_kv_gather(b.cache, b.lens, b.table_dev, L, dtype=dtype)[::-1]
    assert torch.equal(kept[0, where, 0, 32:64].double().cpu(), held)
    o = lv.paged_attention(q, b.cache, *b.call(), max_q_len=n)
    assert torch.equal(o[:n // 2], clean[:n // 2])
    want, _, tol, _ = ref.attention(b, q)
    inf = held.isinf()
    got = o[n // 2:].double().cpu()
    assert torch.equal(got[..., 32:64][..., inf], want[n // 2:, :, 32:64][..., inf])
    rest = torch.ones(D, dtype=torch.bool)
    rest[32:64] = held == 0                               # finite values of that scale: sums may leave the type's range
    ref.check_close(got[..., rest], want[n // 2:][..., rest], tol[n // 2:][..., rest], "beside the infinities")
    b.cache.check()


# ── weights far below their row's largest ────────────────────────────────────


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("gap", [8.0, 14.0, 16.0])
@pytest.mark.parametrize("seqs,D,H,room", [([(1, 600)] * 40, 128, 8, 0), ([(2, 600)] * 40, 256, 8, 0), ([(20, 600)] * 30, 64, 8, 0),
                                           ([(140, 900)] * 16, 64, 8, ROOM), ([(100, 900)] * 16, 128, 8, ROOM),
                                           ([(100, 900)] * 12, 256, 8, ROOM)])
def test_small_weights_beside_keys_far_above_them(gpu, seqs, D, H, room, gap, dtype):
    """The keys that take nearly all the weight have values of 0, so the rest is the whole result.  Weights down to 2^-23 =
    e^-15.94 of their row's largest keep half a step in both types; the smallest here, e^-16, are off by 1.06 of it, which
    the reference's 2 * 664 fp32 roundings of the sums (0.16 of it) leave room for."""
    L = seqs[0][1]
    b = Batch(gpu, seqs, D, H, H, 64, dtype, extra_columns=room // 64)
    g = torch.Generator().manual_seed(1)
    K, V = torch.zeros(L, H, D), torch.randn(L, H, D, generator=g) + 1
    K[:, :, 0] = 0.5 * torch.rand(L, H, generator=g)      # the others' weights: e^(0 .. 0.5 - gap)
    tops = [7, 39, 71, 103]                               # one for each wave of a step
    K[tops, :, 0], V[tops] = gap, 0.0
    for t, x, mine in ((b.cache.k, K, b.K), (b.cache.v, V, b.V)):
        host = torch.zeros(t.shape, dtype=dtype)
        for s in range(len(seqs)):
            b._put(host, s, x.to(dtype))
            mine[s] = x.to(dtype).double()
        t.copy_(host)
    q = torch.zeros(b.N, H, D, dtype=dtype, device=gpu)
    q[:, :, 0] = 1
    o, lse = lv.paged_attention(q, b.cache, *b.call(), scale=1.0, max_q_len=seqs[0][0], return_lse=True)
    wo, wl, tol, ltol = ref.attention(b, q, True, 1.0)
    # The results are down to 2e-5.  fp16 has normal numbers from 2^-14 = 6e-5 on; below, they are multiples of 2^-24, and
    # rounding to them is off by up to 2^-25, which the reference's relative half step (2^-11 of the value) is less than.
    ref.check_close(o, wo, tol + (2.0 ** -25 if dtype == HF else 0.0), "attention")
    ref.check_close(lse, wl, ltol, "lse")
    b.cache.check()


@pytest.mark.parametrize("dtype,size", [(HF, 2.0 ** 19), (HF, 2.0 ** 21), (HF, 2.0 ** 23), (HF, 2.0 ** 25), (BF, 2.0 ** 25), (BF, 2.0 ** 29)])
@pytest.mark.parametrize("n,D,room", [(1, 128, 0), (20, 64, 0), (150, 64, ROOM), (100, 128, ROOM), (60, 256, ROOM)])
def test_scores_of_millions(gpu, n, D, room, dtype, size):
    """Scores that rise, or fall, along the keys up to +-``size``, far more than a weight's range apart: a row's result is
    the value of its largest score's key, its lse that score."""
    L = 300
    b = Batch(gpu, [(n, L)], D, 2, 1, 16, dtype, extra_columns=room // 16)
    k = torch.zeros(L, 1, D)
    k[:, 0, 0] = (torch.arange(1, L + 1) / 512.0).to(dtype).float()       # rising; in bf16 neighbours may be equal
    host = torch.zeros(b.cache.k.shape, dtype=dtype)
    b._put(host, 0, k.to(dtype))
    b.cache.k.copy_(host)
    for sign in (1.0, -1.0):
        q = torch.zeros(n, 2, D, dtype=dtype, device=gpu)
        q[:, :, 0] = sign * 2.0 ** 10
        scale = size / 2.0 ** 9
        o, lse = lv.paged_attention(q, b.cache, *b.call(), scale=scale, max_q_len=n, return_lse=True)
        b.cache.check()
        z = sign * 2.0 ** 10 * scale * k[:, 0, 0].double()
        for i in range(n):
            mine = z[:L - n + i + 1]
            top = (mine == mine.max()).nonzero()[:, 0]    # several where bf16 rounds keys alike: their mean
            want = b.V[0][top, 0].mean(0)
            # equal weights of a few keys, a rounding of each and of the result
            assert (o[i].double().cpu() - want).abs().max() <= 3 * ref.U[dtype] * b.V[0][top, 0].abs().amax()
            # roundings of the score, the scale, its product with log2(e), the sum with the weights' logarithm and ln 2, and
            # the logarithm of at most four equal weights
            assert (lse[i].double().cpu() - mine.max() ).abs().max() <= 6 * ref.F32 * mine.abs().max() + 4


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("base,step", [(0, 4), (2 ** 13, 4), (2 ** 17, 4), (2 ** 23, 4), (2 ** 24, 6), (2 ** 25, 4)])
@pytest.mark.parametrize("n,D,room", [(1, 128, 0), (20, 64, 0), (150, 64, ROOM), (100, 128, ROOM), (60, 256, ROOM)])
def test_scores_a_few_units_apart_around_a_large_one(gpu, n, D, room, base, step, dtype):
    """``base`` plus a small number that rises by one or two steps from keys to keys, scale 1: exact in fp32, so the weights are those
    of the small numbers alone, each e^x with a relative error of 2^-24 |x| and its roundings."""
    L = 700
    b = Batch(gpu, [(n, L)], D, 2, 1, 16, dtype, extra_columns=room // 16)
    j = torch.arange(L)
    small = (step * (j // 50 + j // 130)).to(dtype)       # up to 18 steps
    k = torch.zeros(L, 1, D, dtype=dtype)
    k[:, 0, 0], k[:, 0, 1] = small, float(base) / 4096 if base > 4096 else float(base)
    host = torch.zeros(b.cache.k.shape, dtype=dtype)
    b._put(host, 0, k)
    b.cache.k.copy_(host)
    q = torch.zeros(n, 2, D, dtype=dtype, device=gpu)
    q[:, :, 0], q[:, :, 1] = 1.0, 4096.0 if base > 4096 else 1.0
    o, lse = lv.paged_attention(q, b.cache, *b.call(), scale=1.0, max_q_len=n, return_lse=True)
    b.cache.check()
    z = small.double()[None] + base
    seen = j[None] <= torch.arange(L - n, L)[:, None]
    w = torch.softmax(torch.where(seen, z, float("-inf")), -1)
    V = b.V[0][:, 0]
    want, A = w @ V, w @ V.abs()
    # a weight's exponent is off by 110 * 2^-23, the weight by half a step of its type and the sums by 764 roundings
    u, F = ref.U[dtype], ref.F32
    tol = u * want.abs() + A * (u + 2 * 220 * F + 2 * 764 * F) + (2.0 ** -25 if dtype == HF else 0.0)
    ref.check_close(o[:, 0], want, tol, "attention")
    ref.check_close(o[:, 1], want, tol, "attention")
    wl = torch.logsumexp(torch.where(seen, z, float("-inf")), -1)[:, None].expand(n, 2)
    ref.check_close(lse, wl, 6 * F * wl.abs() + 764 * F + 220 * F, "lse")


# ── pages of keys that some rows do not attend ───────────────────────────────


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("D,n,room", [(64, 700, ROOM), (128, 700, ROOM), (128, 100, ROOM), (192, 700, ROOM), (256, 400, ROOM),
                                      (64, 300, 0)])
@pytest.mark.parametrize("at", ["near", "far", "last"])
def test_a_bad_page_spoils_all_rows_of_its_sequence(gpu, at, D, n, room, bits):
    """Also those of a causal chunk that come before the page's keys, however far before."""
    ps = 16
    b = Batch(gpu, [(70, 90), (n, n + 5), (40, 333)], D, 2, 1, ps, BF, bits=bits, extra_columns=room // ps)
    q = b.randn(b.N, 2, D)
    good, glse = lv.paged_attention(q, b.cache, *b.call(), return_lse=True)
    assert not torch.isnan(good).any()
    key = {"near": 5 + (130 if n > 200 else 70), "far": n - 40, "last": n + 4}[at]
    b.table_dev[1, key // ps] = b.cache.num_pages
    o, lse = lv.paged_attention(q, b.cache, *b.call(), return_lse=True)
    assert torch.isnan(o[70:70 + n]).all() and torch.isnan(lse[70:70 + n]).all()
    assert torch.equal(o[:70], good[:70]) and torch.equal(o[70 + n:], good[70 + n:])
    assert torch.equal(lse[:70], glse[:70]) and torch.equal(lse[70 + n:], glse[70 + n:])
    with pytest.raises(ValueError, match="page number"):
        b.cache.check()


@pytest.mark.parametrize("room", [0, ROOM])
def test_a_bad_page_behind_rows_without_keys(gpu, room):
    """More rows than cached keys: rows before the first cached position are spoiled like the rest of their sequence."""
    b = Batch(gpu, [(300, 40), (90, 90)], 128, 1, 1, 8, BF, extra_columns=room // 8)
    q = b.randn(b.N, 1, 128)
    o = lv.paged_attention(q, b.cache, *b.call())
    assert (o[:260] == 0).all() and not torch.isnan(o).any()
    b.table_dev[0, 4] = -1
    o = lv.paged_attention(q, b.cache, *b.call())
    assert torch.isnan(o[:300]).all() and not torch.isnan(o[300:]).any()
    with pytest.raises(ValueError, match="page number"):
        b.cache.check()


# ── the cache's status ───────────────────────────────────────────────────────


def test_check_waits_for_every_stream(gpu):
    """A call that runs late on another stream is in the answer, and the answer is given once."""
    b = Batch(gpu, [(1, 100)], 128, 4, 2, 16, BF)
    q = b.randn(1, 4, 128)
    bad = torch.full_like(b.table_dev, -1)
    x = torch.randn(8192, 8192, device=gpu, dtype=BF)
    torch.mm(x, x)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(40):                               # some 40 ms
            torch.mm(x, x)
        lv.paged_attention(q, b.cache, b.cu, b.lens, bad, max_q_len=1)
    with pytest.raises(ValueError, match="page number"):
        b.cache.check()
    torch.cuda.synchronize()
    b.cache.check()


def test_check_takes_what_it_reports(gpu):
    """What is found between the read and the end of a check is the next one's."""
    b = Batch(gpu, [(1, 100)], 128, 4, 2, 16, BF)
    b.cache.status.fill_(_capi.PAGED_BAD_PAGE | _capi.PAGED_BAD_POSITION)
    found = torch.zeros(1, dtype=torch.int32, device=gpu)
    hip_ops._call(gpu, "lvsa_paged_take_status", b.cache.status.data_ptr(), found.data_ptr())
    b.cache.status.fill_(_capi.PAGED_BAD_LENGTH)
    assert found.item() == _capi.PAGED_BAD_PAGE | _capi.PAGED_BAD_POSITION
    with pytest.raises(ValueError) as e:
        b.cache.check()
    assert "kv_lens" in str(e.value) and "page number" not in str(e.value)
    b.cache.check()


# ── tensors that share memory ────────────────────────────────────────────────


@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("rot,inter", [(0, False), (128, False), (64, True)])
def test_new_tokens_that_are_the_caches_own(gpu, rot, inter, layout):
    """Keys and values taken from the pages that the call writes, each shifted by some slots: as from a copy of them."""
    ps, Hkv, D, n = 64, 2, 128, 40
    b = Batch(gpu, [(n, 70), (20, 30)], D, 4, Hkv, ps, BF, layout=layout)
    cos, sin = (torch.rand(70, rot // 2, device=gpu) for _ in range(2))
    kw = {"cos": cos, "sin": sin, "interleaved": inter} if rot else {}
    page = b.pages[0][0]
    b.cache.k.nan_to_num_(0.25)
    b.cache.v.nan_to_num_(0.5)
    k, v = b.cache.k[page, 2:62], b.cache.v[page, 1:61]                   # [60, Hkv, D] of the first page
    want = [lv.PagedKVCache(b.cache.k.clone(), b.cache.v.clone())]
    lv.paged_kv_append(want[0], k.clone(), v.clone(), *b.call(), **kw)
    lv.paged_kv_append(b.cache, k, v, *b.call(), **kw)
    assert torch.equal(b.cache.k, want[0].k) and torch.equal(b.cache.v, want[0].v)
    b.cache.check()


def test_results_in_the_caches_memory_are_refused(gpu):
    b = Batch(gpu, [(4, 20)], 128, 2, 2, 16, BF)
    q, k = b.randn(4, 2, 128), b.randn(4, 2, 128)
    for t in (b.cache.k, b.cache.v):
        inside = t[0, 3:7]
        with pytest.raises(ValueError, match="share memory with the cache"):
            lv.paged_attention(q, b.cache, *b.call(), out=inside)
        with pytest.raises(ValueError, match="share memory with the cache"):
            lv.paged_kv_append(b.cache, k, k, *b.call(), q=q, q_out=inside)
    b.cache.check()


def test_gradients_of_angles_and_pages_are_refused(gpu):
    b = Batch(gpu, [(4, 20)], 128, 2, 2, 16, BF)
    k = b.randn(4, 2, 128)
    cos, sin = (torch.rand(20, 64, device=gpu) for _ in range(2))
    for kw in ({"cos": cos.clone().requires_grad_(), "sin": sin}, {"cos": cos, "sin": sin.clone().requires_grad_()}):
        with pytest.raises(RuntimeError, match="gradient"):
            lv.paged_kv_append(b.cache, k, k, *b.call(), **kw)
        with torch.no_grad():
            lv.paged_kv_append(b.cache, k, k, *b.call(), **kw)
    with pytest.raises(RuntimeError, match="gradient"):
        lv.PagedKVCache(b.cache.k.clone().requires_grad_(), b.cache.v)
    with pytest.raises(RuntimeError, match="gradient"):
        lv.PagedKVCache(b.cache.k, b.cache.v.clone().requires_grad_())
    b.cache.check()


# ── inside torch.compile ─────────────────────────────────────────────────────


def test_calls_inside_a_compiled_function(gpu):
    """The calls break the graph and run as they are, with the same results, also for other lengths later."""
    b = Batch(gpu, [(3, 40), (3, 20)], 128, 4, 2, 16, BF)
    cos, sin = (torch.rand(64, 64, device=gpu) for _ in range(2))

    def f(q, k, v, lens):
        qr = lv.paged_kv_append(b.cache, k * 1.0, v * 1.0, b.cu, lens, b.table_dev, q=q * 1.0, cos=cos, sin=sin)
        o, lse = lv.paged_attention(qr, b.cache, b.cu, lens, b.table_dev, max_q_len=3, return_lse=True)
        kk, vv = lv.paged_kv_gather(b.cache, lens, b.table_dev, 40)
        b.cache.check()
        return o * 2.0, lse + 1.0, kk + 0, vv + 0

    g = torch.compile(f, backend="eager")
    for back in (0, 1, 2):
        x = b.randn(6, 4, 128), b.randn(6, 2, 128), b.randn(6, 2, 128), b.lens - back
        want, got = f(*x), g(*x)
        assert all(torch.equal(a.nan_to_num(3.0), c.nan_to_num(3.0)) for a, c in zip(want, got))
    b.cache.check()


# ── many sequences and tiles on the kernels of long caches ───────────────────


def _workspace(b, heads, hint, sequences):
    """Bytes that a call of the batch, cut to its first sequences, asks for."""
    a = _capi.PagedAttnArgs.from_buffer_copy(
        b.cache._pack(b.dtype) + paged_kv._batch(b.cache, b.cu[:sequences + 1], b.lens[:sequences], b.table_dev[:sequences], b.N) +
        bytes(paged_kv._ATTN.size))
    a.q = a.o = 1 << 20
    a.q_str = a.o_str = _capi._Str2(heads * b.D, b.D)
    a.scale, a.H, a.max_q_len = 1.0, heads, hint
    n = ctypes.c_int64()
    assert _capi.lib().lvsa_paged_attn_workspace_query(ctypes.byref(a), ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,hint", [(64, 40), (64, 200), (256, 40)])
@pytest.mark.parametrize("B", [65, 1100, 5200])
def test_many_sequences_of_the_plan(gpu, B, D, hint, causal):
    """More sequences than the plan takes at a time, more row tiles than it keeps whole (1024) or in LDS at all (4096),
    shares that span many tiles: on the 128-row and 256-row kernels.  Then a bad page in a late sequence."""
    seqs = [(0 if s % 7 == 3 else 1 + (s % 11 == 0), s % 5 + (s * s) % 13) for s in range(B)]
    seqs = [(min(n, L), L) for n, L in seqs]
    seqs[B // 2] = (300, 301)                             # several tiles of one sequence in between
    if B > 5000:
        seqs[-3] = (600, 600)
    b = Batch(gpu, seqs, D, 2, 1, 8, BF, seed=6, tail=2, extra_columns=(20000 if B < 1000 else 2400) // 8)
    # every tile takes 56 bytes of the plan; the decode kernel's workspace does not follow the sequences here
    assert _workspace(b, 2, hint, B) - _workspace(b, 2, hint, B // 2) >= 56 * (B - B // 2) - 16
    q = b.randn(b.N, 2, D)
    o, lse = lv.paged_attention(q, b.cache, *b.call(), causal=causal, return_lse=True, max_q_len=hint)
    wo, wl, tol, ltol = ref.attention(b, q, causal)
    ref.check_close(o, wo, tol, "attention")
    ref.check_close(lse, wl, ltol, "lse")
    b.cache.check()
    late = B - 3 if B > 5000 else B // 2
    b.table_dev[late, 37] = -1                            # keys 296 .. 303: behind the first tile's
    bad, _ = lv.paged_attention(q, b.cache, *b.call(), causal=causal, return_lse=True, max_q_len=hint)
    lo, hi = b.ends[late], b.ends[late + 1]
    assert torch.isnan(bad[lo:hi]).all() and torch.equal(bad[:lo], o[:lo]) and torch.equal(bad[hi:], o[hi:])
    with pytest.raises(ValueError, match="page number"):
        b.cache.check()


# ── layouts and sizes ────────────────────────────────────────────────────────


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("n,D,room", [(1, 128, 0), (20, 96, 0), (60, 64, ROOM), (150, 128, ROOM), (60, 256, ROOM)])
def test_strided_queries_results_and_pages(gpu, n, D, room, bits):
    """Queries and results that are views of packed tensors, keys with their heads' rows apart, values with their tokens'."""
    H, Hkv, ps = 4, 2, 16
    b = Batch(gpu, [(n, 200), (n, 170)], D, H, Hkv, ps, BF, bits=bits, extra_columns=room // ps)
    q = b.randn(b.N, H, D)
    want, wl = lv.paged_attention(q, b.cache, *b.call(), max_q_len=n, return_lse=True)
    c = b.cache

    def tokens(t):                                        # one half of [pages, 2, page_size, heads, X]
        wide = torch.full((t.shape[0], 2, *t.shape[1:]), 77, dtype=t.dtype, device=gpu)
        wide[:, 1] = t
        return wide[:, 1]

    def heads(t):                                         # [heads, pages, page_size, X]
        return torch.empty(t.shape[2], t.shape[0], t.shape[1], t.shape[3], dtype=t.dtype, device=gpu).permute(1, 2, 0, 3).copy_(t)

    both = (c.k, c.v) if bits == 16 else (c.k, c.v, c.k_scale, c.v_scale)
    other = lv.PagedKVCache(*[(heads if i % 2 == 0 else tokens)(t) for i, t in enumerate(both)])
    packed = torch.full((b.N, 3 * H, D), float("nan"), dtype=BF, device=gpu)
    packed[:, H:2 * H] = q
    out = torch.full((H + 1, b.N + 2, D), 9.0, dtype=BF, device=gpu)
    view = out[1:, 1:-1].transpose(0, 1)                  # [N, H, D], a head's rows next to each other
    got, gl = lv.paged_attention(packed[:, H:2 * H], other, *b.call(), max_q_len=n, out=view, return_lse=True)
    assert torch.equal(got, want) and torch.equal(gl, wl)
    assert (out[0] == 9.0).all() and (out[:, 0] == 9.0).all() and (out[:, -1] == 9.0).all()
    k, v = lv.paged_kv_gather(other, b.lens, b.table_dev, 200)
    wk, wv = lv.paged_kv_gather(c, b.lens, b.table_dev, 200)
    assert torch.equal(k, wk) and torch.equal(v, wv)
    new = b.randn(b.N, 3 * Hkv, D)
    for x in (c, other):
        lv.paged_kv_append(x, new[:, :Hkv], new[:, Hkv:2 * Hkv], *b.call())
    for t, u in zip(both, (other.k, other.v) if bits == 16 else (other.k, other.v, other.k_scale, other.v_scale)):
        assert torch.equal(t.nan_to_num(3.0) if bits == 16 else t, u.nan_to_num(3.0) if bits == 16 else u)
    c.check()
    other.check()


def test_more_tokens_and_rows_than_a_launch_has_work_groups(gpu):
    """1.2 million tokens appended, and 1.1 million output rows over a few keys on the decode kernel's merge."""
    N, ps, D = 1_200_000, 4096, 64
    cache = lv.PagedKVCache.allocate(300, ps, 1, D, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(1)
    k, v = (torch.randn(N, 1, D, generator=g, device=gpu).to(BF) for _ in range(2))
    of = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    table = torch.randperm(300, generator=g, device=gpu)[None, :293].to(torch.int32)
    lv.paged_kv_append(cache, k, v, of(0, N), of(N), table)
    got = lv.paged_kv_gather(cache, of(N), table, N)
    assert torch.equal(got[0][0], k) and torch.equal(got[1][0], v)
    n, H, L = 70_000, 16, 10
    q = torch.randn(n, H, D, generator=g, device=gpu).to(BF)
    o = lv.paged_attention(q, cache, of(0, n), of(L), table, causal=False, max_q_len=1)
    w = torch.softmax(q.float().flatten(0, 1) @ k[:L, 0].float().T / 8.0, -1)
    want, A = w @ v[:L, 0].float(), w @ v[:L, 0].float().abs()
    # weights and results rounded to bf16, scores of 64 products and the sums in fp32 on both sides
    err = (o.float().flatten(0, 1) - want).abs() - (ref.U[BF] * want.abs() + A * (ref.U[BF] + 2.0 ** -14))
    assert err.max().item() <= 0
    cache.check()


@pytest.mark.parametrize("bits", [16, 4])
def test_seventeen_million_keys(gpu, bits):
    """Positions past 2^24: keys of 0 weigh alike, so a result is the mean of the values, here 1 for the first half of the
    keys and 3 for the rest, and the lse the logarithm of their number."""
    L, ps, D, n = 17_000_000, 50_000, 64, 300
    pages = L // ps
    one, three = (0x22, 0x55) if bits == 4 else (1.0, 3.0)               # E2M1: 2 is 1.0, 5 is 3.0
    shape = (pages, ps, 1, D // 2 if bits == 4 else D)
    dt = torch.uint8 if bits == 4 else BF
    k, v = (torch.zeros(shape, dtype=dt, device=gpu) for _ in range(2))
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).to(torch.int32).to(gpu)[None]
    v[table[0, :pages // 2].long()], v[table[0, pages // 2:].long()] = one, three
    scales = [torch.full((pages, ps, 1, D // 32), 127, dtype=torch.uint8, device=gpu) for _ in range(2)] if bits == 4 else []
    cache = lv.PagedKVCache(k, v, *scales)
    cu, lens = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([0, n], [L]))
    q = torch.ones(n, 1, D, dtype=BF, device=gpu)
    o, lse = lv.paged_attention(q, cache, cu, lens, table, return_lse=True)
    o1, lse1 = lv.paged_attention(q[:1], cache, cu.clamp(max=1), lens, table, return_lse=True)
    seen = torch.arange(L - n + 1, L + 1, dtype=torch.float64)
    half = pages // 2 * ps
    want = (half + 3.0 * (seen - half)) / seen
    # counts of equal weights and of their values, each summed in fp32: under 2^17 terms to a partial sum of a lane
    tol = ref.U[BF] * want + want * (2.0 ** 17 * ref.F32)
    assert ((o[:, 0].double().cpu() - want[:, None]).abs() <= tol[:, None]).all()
    assert ((o1[:, 0].double().cpu() - want[-1]).abs() <= tol[-1]).all()
    for got, w in ((lse[:, 0], seen.log()), (lse1[:, 0], seen[-1:].log())):
        assert ((got.double().cpu() - w).abs() <= 2.0 ** 17 * ref.F32 + 8 * ref.F32 * w).all()
    cache.check()


@pytest.mark.parametrize("bits", [16, 4])
def test_two_captured_graphs_of_one_pool(gpu, bits):
    """A step of single tokens and a chunk, captured into one memory pool (their workspaces may be the same memory) and
    replayed in turn with eager calls in between: each as its eager result."""
    one = Batch(gpu, [(1, 4000), (1, 50), (1, 2500)], 128, 8, 2, 16, BF, bits=bits, tail=1)
    many = Batch(gpu, [(70, 900), (150, 150)], 128, 8, 2, 16, BF, bits=bits, extra_columns=ROOM // 16)
    runs = []
    for b, hint in ((one, 1), (many, 150)):
        q, out = b.randn(b.N, 8, 128), torch.zeros(b.N, 8, 128, dtype=BF, device=gpu)
        call = lambda b=b, q=q, hint=hint, out=out: lv.paged_attention(q, b.cache, *b.call(), max_q_len=hint, out=out,  # noqa: E731
                                                                       return_lse=True)
        want = [x.clone() for x in call()]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=runs[0][1].pool() if runs else None):
            got = call()
        runs.append((call, graph, got, want))
    for i in range(4):
        for call, graph, got, want in runs if i % 2 else runs[::-1]:
            for x in got:
                x.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x[:-1], w[:-1]) for x, w in zip(got, want)), i
            assert (got[0][-1] == 7.0).all() if call is runs[0][0] else torch.equal(got[0][-1], want[0][-1])
            assert torch.equal(got[1], want[1])
            assert all(torch.equal(x[:-1], w[:-1]) for x, w in zip(call(), want))
    one.cache.check()
    many.cache.check()
