"""Parts of the paged key/value cache instead of all of it, as measurable cases.

A long cache is neither read whole by every step nor kept whole for ever:

* block means: the mean key of every block of ``block`` consecutive tokens, kept
  beside the pages and renewed where new tokens were appended;
* select: for every tile of ``tile`` newest tokens and every key head, the ``top``
  blocks whose mean key scores highest with the tile's queries, its own blocks and
  the sequence's first ones always among them;
* block attention: the newest tokens' attention over the keys of their blocks;
* weights: the attention weight that the newest tokens give to every cached token,
  added to what it had from earlier ones;
* evict: of every sequence and key head the ``keep`` tokens that count, the first,
  the newest and the heaviest, moved together in their order.

Geometry of a case: ``B`` sequences of up to ``L`` cached tokens, the newest ``n`` of
them this call's, the last ``empty`` sequences without any; ``H`` query and ``Hkv``
key heads of size ``D``; pages of ``page`` slots, each of ``page / block`` blocks.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
SPARE_PAGES = 3


def _case(name, kind, B, n, L, H, Hkv, D, page, block=0, top=0, tile=1, bits=16, dtype="bf16", causal=True, ragged=False,
          empty=0, lse=False, accumulate=True, keep=0, first=1, last=1, in_place=False):
    return {"name": name, "kind": kind, "B": B, "n": n, "L": L, "H": H, "Hkv": Hkv, "D": D, "page": page, "block": block or page,
            "top": top, "tile": tile, "bits": bits, "dtype": dtype, "causal": causal, "ragged": ragged, "empty": empty,
            "lse": lse, "accumulate": accumulate, "keep": keep, "first": first, "last": last, "in_place": in_place}


def listed():
    return [
        # A serving batch's newest tokens: the one block that each changes, the small call of every decoding step.
        _case("means_step", "means", 32, 1, 2100, 32, 8, 128, 16, ragged=True),
        # Three new frames of a video stream, fifteen blocks a frame.
        _case("means_frames", "means", 1, 4680, 28080, 12, 12, 128, 1560, block=104),
        # A serving batch's next tokens over long ragged caches, grouped heads, three slots without a request.
        _case("select_step", "select", 48, 1, 16000, 32, 8, 128, 64, top=32, ragged=True, empty=3),
        # Ragged prompts' newest parts, every token its own blocks, fp16, small heads.
        _case("select_prompts", "select", 6, 1700, 5200, 16, 4, 64, 16, top=64, dtype="f16", ragged=True, last=4),
        # One stream's next token: the smallest attention, nothing but latency.
        _case("attend_one", "attend", 1, 1, 4100, 16, 4, 128, 16, top=32),
        # The serving batch's next tokens over the blocks selected for them.
        _case("attend_batch", "attend", 48, 1, 16000, 32, 8, 128, 64, top=32, ragged=True, empty=3, lse=True),
        # A larger batch over a cache that only fits in 4 bits.
        _case("attend_batch_4bit", "attend", 40, 1, 32000, 32, 8, 128, 64, top=64, bits=4, ragged=True),
        # Three new frames of a video stream over a sixth of fifteen cached ones and themselves, tiles of 128 tokens.
        _case("attend_frames", "attend", 1, 4680, 28080, 12, 12, 128, 1560, block=104, top=48, tile=128, causal=False),
        # What the serving batch's next tokens add to the weights of all that is cached.
        _case("weights_step", "weights", 48, 1, 16000, 32, 8, 128, 64, ragged=True, empty=3),
        # Ragged prompts, causal, the weights of every token from the start.
        _case("weights_prompts", "weights", 6, 1700, 5200, 16, 4, 64, 16, dtype="f16", ragged=True, accumulate=False),
        # Prompts cut to an eighth into pages of their own once they are through.
        _case("evict_prompts", "evict", 8, 0, 16000, 32, 8, 128, 64, ragged=True, keep=2048, first=4, last=64),
        # A serving batch back to its budget after some steps, where it lies.
        _case("evict_steps", "evict", 32, 0, 2112, 32, 8, 128, 16, keep=2048, first=4, last=256, in_place=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    """One more call of the listed ranges: every operator, head size, type, page and block size and group of heads."""
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["means", "select", "attend", "attend", "attend", "weights", "evict"])
        D, Hkv, group = rng.choice([64, 96, 128, 128, 192, 256]), rng.choice([1, 2, 4, 5, 8, 12]), rng.choice([1, 1, 2, 3, 4, 6, 8])
        page = rng.choice([7, 16, 16, 32, 64, 64, 100, 256, 390, 1560])
        block = page // rng.choice([x for x in (1, 1, 2, 4, 5, 10, 13, 15) if page % x == 0])
        bits, tile = rng.choice([16, 16, 4]), rng.choice([1, 1, 1, 8, 32, 64, 100, 128, 256])
        style = rng.choice(["step", "few", "chunk"])
        if style == "step":
            B, n, L = _log_int(rng, 1, 64), 1, _log_int(rng, 1, 32000)
        elif style == "few":
            B, n, L = _log_int(rng, 1, 24), rng.randint(2, 9), _log_int(rng, 9, 16000)
        else:
            B, L = _log_int(rng, 1, 8), _log_int(rng, 40, 28000)
            n = _log_int(rng, min(16, L), min(L, 4700))
        first, last = rng.choice([0, 1, 1, 2, 4]), rng.choice([1, 1, 2, 3])
        top = first + last + -(-tile // block) + _log_int(rng, 1, 100)
        keep = 0
        if kind == "evict":
            n, keep, first, last = 0, _log_int(rng, 1, max(1, L)), rng.choice([0, 1, 4, 16]), rng.choice([0, 1, 32, 100])
            keep = max(keep, first + last + 1)
        causal = rng.random() < 0.6 or kind == "select" and tile == 1
        if kind == "attend" and causal:
            tile = min(tile, 64)
        case = _case("", kind, B, n, L, Hkv * group, Hkv, D, page, block, top, tile, bits, rng.choice(["bf16", "bf16", "f16"]), causal,
                     B > 1 and rng.random() < 0.7, rng.choice([0, 0, 1]) if B > 1 else 0, kind == "attend" and rng.random() < 0.3,
                     rng.random() < 0.6, keep, first, last, rng.random() < 0.4)
        del case["name"]
        # what the plain forms hold at once: padded sequences, and every tile's keys
        scores = B * Hkv * group * max(n, 1) * L if kind == "weights" else 0
        tiles = B * -(-n // tile) * Hkv
        gathered = tiles * min(top * block, L + block) * (D + tile * group) if kind == "attend" else 0
        ranked = tiles * (L // block + 1) if kind == "select" else 0
        if (_cost(case) <= most and scores <= 1.6e9 and gathered <= 1.5e9 and ranked <= 1.5e8 and top <= 1024
                and B * L * Hkv * D <= 1.0e9):
            return case


# ── what a case's inputs are ─────────────────────────────────────────────────


def _lengths(case):
    """(new tokens, cached tokens with them) of every sequence: from the case alone."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    got = []
    for b in range(case["B"]):
        n, L = case["n"], case["L"]
        if case["ragged"] and b:
            L = max(1, int(L * r.uniform(0.2, 1.0)))
            n = min(L, max(min(n, 1), int(n * r.uniform(0.3, 1.0))))
        if b >= case["B"] - case["empty"]:
            n = L = 0
        got.append((min(n, L), L))
    return got


def _rows(shape, dtype, fill):
    """A ``[pages, slots, Hkv, X]`` tensor, a page's rows of one head next to each other."""
    P, ps, Hkv = shape[:3]
    t = torch.empty((P, Hkv, ps) + shape[3:], dtype=dtype, device="cuda").transpose(1, 2)
    return t.copy_(fill)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, kind = DTYPES[case["dtype"]], case["kind"]
    B, H, Hkv, D, ps, bs = case["B"], case["H"], case["Hkv"], case["D"], case["page"], case["block"]
    lens = _lengths(case)
    N = sum(n for n, _ in lens)
    counts = [-(-L // ps) for _, L in lens]
    kept = [-(-min(L, case["keep"]) // ps) for _, L in lens] if kind == "evict" and not case["in_place"] else [0] * B
    P = sum(counts) + sum(kept) + SPARE_PAGES
    order, at = torch.randperm(P, generator=g, device="cuda").to(torch.int32).cpu(), 0
    tables = []
    for of in (counts, kept):
        t = torch.zeros(B, max(max(of), 1), dtype=torch.int32)
        for b, c in enumerate(of):
            t[b, :c] = order[at:at + c]
            at += c
        tables.append(t.cuda())
    s = {"case": case, "N": N, "max_n": max(n for n, _ in lens), "max_L": max(L for _, L in lens), "table": tables[0],
         "new_table": tables[1], "scale": 1.0 / math.sqrt(D),
         "cu": torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32).cuda(),
         "lens": torch.tensor([L for _, L in lens], dtype=torch.int32).cuda()}

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    channel = 0.5 + 1.5 * torch.rand(Hkv, D, generator=g, device="cuda")      # keys: channels of different size
    centre = 0.5 * normal(P, ps // bs, 1, Hkv, D)                             # and what a block's keys have in common
    for name in ("k", "v"):
        x = normal(P, ps, Hkv, D)
        if name == "k":
            x.unflatten(1, (ps // bs, bs)).add_(centre)
            x *= channel
        if case["bits"] == 16:
            s[name] = _rows((P, ps, Hkv, D), dt, x)
        else:
            codes, scales = _quantize(x)
            s[name] = _rows((P, ps, Hkv, D // 2), torch.uint8, codes)
            s[name + "_scale"] = _rows((P, ps, Hkv, D // 32), torch.uint8, scales)
    if kind in ("select", "attend", "weights"):
        s["q"] = (1.5 * normal(N, H, D)).to(dt)
    if kind in ("means", "select"):                                           # of the tokens before
        s["means"] = _rows((P, ps // bs, Hkv, D), torch.float32, centre[:, :, 0] * channel + 0.125 * normal(P, ps // bs, Hkv, D))
    if kind in ("weights", "evict"):                                          # a few tokens have most of it, some none
        w = (1.5 * normal(P, ps, Hkv)).exp_() * (torch.rand(P, ps, Hkv, generator=g, device="cuda") > 0.02)
        s["weights"] = _rows((P, ps, Hkv), torch.float32, w)
    if kind == "attend":
        p0, _, lim, _, real = _tiles(s)
        nb = -(-lim // bs)
        rank = torch.rand(p0.numel(), Hkv, -(-s["max_L"] // bs), generator=g, device="cuda", dtype=torch.float64)
        s["blocks"] = _take(rank, s, nb, real)
    if kind == "weights":
        s["lse"] = _logsumexp(s)
    return s


# ── the plain forms ──────────────────────────────────────────────────────────


def _quantize(x):
    """(codes, scales) of values ``[..., D]``: for every 32 the smallest 2^e with 6 * 2^e >= all of them (e from -23 to
    13, kept as e + 127), and the nearest E2M1 number of each quotient, ties to even, two to a byte, the even one low."""
    D = x.shape[-1]
    x = x.unflatten(-1, (D // 32, 32))
    mant, e = torch.frexp(x.abs().amax(-1))                          # amax = mant * 2^e, mant in [0.5, 1)
    e = torch.where(mant > 0, e - 3 + (mant > 0.75), -23).clamp(-23, 13)
    a = x.abs() * _power(-e)[..., None]
    up = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (up + 8 * torch.signbit(x)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _power(e):
    """2^e as fp32, from the bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _values(s, name, *at):
    """Cached rows in 32 bits."""
    if s["case"]["bits"] == 16:
        return s[name][at].float()
    codes, scales = s[name][at], s[name + "_scale"][at]
    levels = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=codes.device)
    x = torch.stack((levels[(codes & 15).int()], levels[(codes >> 4).int()]), -1).flatten(-2)
    return x * _power(scales.to(torch.int32) - 127).repeat_interleave(32, -1)


def _places(s, pos, lens, table):
    """Page and slot of position ``pos[b, i]`` of sequence b; positions behind the end: its first page's."""
    ps = s["case"]["page"]
    pos = torch.where((pos >= 0) & (pos < lens[:, None]), pos, 0)
    return torch.gather(table.long(), 1, pos // ps), pos % ps


def _token_places(s):
    """Sequence and number in it of each new token."""
    t = torch.arange(s["N"], device="cuda")
    b = torch.searchsorted(s["cu"].long(), t, right=True) - 1
    return b, t - s["cu"].long()[b]


def _tile_of(s, b, i):
    """The tile of token i of sequence b: rows of a tile start at multiples of ``tile`` within their sequence."""
    tile = s["case"]["tile"]
    return s["cu"].long()[b] + i if tile == 1 else s["cu"].long()[b] // tile + b + i // tile


def _tiles(s):
    """Of every tile: the position of its first row and behind its last one, how far its rows see, its sequence; and
    whether there is such a tile."""
    case, (b, i) = s["case"], _token_places(s)
    T = s["N"] if case["tile"] == 1 else s["N"] // case["tile"] + case["B"]
    at = _tile_of(s, b, i)
    lens, n = s["lens"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    p0, p1 = torch.full((T,), 1 << 30, device="cuda"), torch.zeros(T, dtype=torch.long, device="cuda")
    p0.scatter_reduce_(0, at, lens[b] - n[b] + i, "amin")
    p1.scatter_reduce_(0, at, lens[b] - n[b] + i + 1, "amax")
    seq = torch.zeros(T, dtype=torch.long, device="cuda").index_copy_(0, at, b)
    real = p1 > 0
    lim = torch.where(real, p1 if case["causal"] else lens[seq], 0)
    return torch.where(real, p0, 0), p1, lim, seq, real


def _take(score, s, nb, real):
    """The ``top`` blocks of every row of ``score [T, Hkv, blocks]``, of its first ``nb[T]``, ascending, -1 behind."""
    case = s["case"]
    p0, p1, _, _, _ = _tiles(s)
    j = torch.arange(score.shape[2], device="cuda")
    near = (j >= (p0 // case["block"])[:, None] - (case["last"] - 1)) & (j <= ((p1 - 1) // case["block"])[:, None])
    always = (j < case["first"]) | (near if case["last"] else torch.zeros_like(near))
    there = (j < nb[:, None]) & real[:, None]
    score = torch.where(always[:, None], float("inf"), score)
    score = torch.where(there[:, None], score, float("-inf"))
    top = min(case["top"], score.shape[2])
    best = score.sort(dim=-1, descending=True, stable=True)[1][..., :top]
    best = torch.where(best < nb[:, None, None], best, 1 << 30)
    best = torch.where(real[:, None, None], best, 1 << 30).sort(-1)[0]
    best = torch.where(best < 1 << 30, best, -1)
    return torch.nn.functional.pad(best, (0, case["top"] - top), value=-1).to(torch.int32)


def _means(s):
    case, lens = s["case"], s["lens"].long()
    ps, bs = case["page"], case["block"]
    blocks = -(-s["max_L"] // bs)
    j = torch.arange(blocks, device="cuda").expand(case["B"], -1)
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    changed = (j >= ((lens - n) // bs)[:, None]) & (j * bs < lens[:, None]) & (n > 0)[:, None]
    b, j = changed.nonzero(as_tuple=True)
    pos = j[:, None] * bs + torch.arange(bs, device="cuda")                          # [blocks, bs]
    inside = pos < lens[b, None]
    page = s["table"].long()[b, j * bs // ps]
    x = _values(s, "k", page[:, None], pos % ps)                                     # [blocks, bs, Hkv, D]
    x = torch.where(inside[..., None, None], x, 0.0).sum(1, dtype=torch.float64)
    s["means"][page, j * bs % ps // bs] = (x / inside.sum(1)[:, None, None]).float()
    return s["means"]


def _select(s):
    case = s["case"]
    Hkv, D, bs, parts = case["Hkv"], case["D"], case["block"], case["page"] // case["block"]
    p0, _, lim, seq, real = _tiles(s)
    b, i = _token_places(s)
    q = s["q"].double().unflatten(1, (Hkv, -1)).sum(2)                               # [N, Hkv, D]
    q = torch.zeros(p0.numel(), Hkv, D, dtype=torch.float64, device="cuda").index_add_(0, _tile_of(s, b, i), q)
    nb = -(-lim // bs)
    # the tiles and the means of a sequence next to each other, padded
    j = torch.arange(-(-s["max_L"] // bs), device="cuda").expand(case["B"], -1)
    page, slot = _places(s, j * bs, s["lens"].long(), s["table"])
    m = s["means"][page, slot // bs].double().permute(0, 2, 3, 1).contiguous()       # [B, Hkv, D, blocks]
    place = torch.arange(p0.numel(), device="cuda")
    place = place - torch.full((case["B"],), 1 << 30, device="cuda").scatter_reduce(0, seq[real], place[real], "amin")[seq]
    place = torch.where(real, place, 0)
    padded = torch.zeros(case["B"], int(-(-s["max_n"] // case["tile"])) or 1, Hkv, D, dtype=torch.float64, device="cuda")
    padded[seq[real], place[real]] = q[real]
    score = torch.matmul(padded.transpose(1, 2).contiguous(), m)                     # [B, Hkv, tiles, blocks]
    return _take(score.transpose(1, 2)[seq, place], s, nb, real)


def _attend(s):
    case, blocks = s["case"], s["blocks"].long()
    H, Hkv, D, ps, bs, tile = case["H"], case["Hkv"], case["D"], case["page"], case["block"], case["tile"]
    p0, _, _, seq, real = _tiles(s)
    T, g, lens = p0.numel(), H // Hkv, s["lens"].long()
    b, i = _token_places(s)
    at, row = _tile_of(s, b, i), i % tile
    rows = torch.zeros(T, tile, dtype=torch.long, device="cuda")
    rows[at, row] = torch.arange(s["N"], device="cuda")
    pos = (blocks[..., None] * bs + torch.arange(bs, device="cuda")).flatten(2)      # [T, Hkv, W * bs]
    there = (pos >= 0) & (pos < lens[seq][:, None, None])
    where = torch.where(there, pos, 0)
    page = s["table"].long()[seq[:, None, None], where // ps]
    head = torch.arange(Hkv, device="cuda")[None, :, None]
    k, v = (_values(s, x, page, where % ps, head) for x in "kv")                     # [T, Hkv, W * bs, D]
    q = s["q"][rows].float().unflatten(2, (Hkv, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    p = torch.matmul(q, k.transpose(2, 3)) * s["scale"]                              # [T, Hkv, tile * g, W * bs]
    end = p0[:, None] + torch.arange(tile, device="cuda") if case["causal"] else lens[seq][:, None].expand(T, tile)
    seen = there[:, :, None] & (pos[:, :, None] <= end[:, None, :, None])
    p = p.unflatten(2, (tile, g)).masked_fill_(~seen[:, :, :, None], float("-inf")).flatten(2, 3)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    o = o.unflatten(2, (tile, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)               # [T, tile, H, D]
    out = {"o": o[at, row].to(s["q"].dtype)}
    if case["lse"]:
        lse = (top + total.log())[..., 0].unflatten(2, (tile, g)).permute(0, 2, 1, 3).flatten(2, 3)
        out["lse"] = lse[at, row]
    return out


def _scores(s):
    """Scaled scores ``[B, Hkv, g, n, max_L]`` of the newest rows in 32 bits, -inf for what a row does not attend, and the
    row of the packed tensors that each is."""
    case, q = s["case"], s["q"]
    B, H, Hkv, n = case["B"], case["H"], case["Hkv"], s["max_n"]
    lens, cu = s["lens"].long(), s["cu"].long()
    j = torch.arange(s["max_L"], device="cuda")
    page, slot = _places(s, j.expand(B, -1), lens, s["table"])
    k = _values(s, "k", page, slot).permute(0, 2, 3, 1).contiguous()                 # [B, Hkv, D, max_L]
    i = torch.arange(n, device="cuda")
    count = cu[1:] - cu[:-1]
    last = (lens - count)[:, None] + i if case["causal"] else (lens - 1)[:, None].expand(B, n)
    row = (cu[:-1, None] + i).clamp(max=s["N"] - 1)
    qb = q[row].float().unflatten(2, (Hkv, H // Hkv)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    z = (torch.matmul(qb, k) * s["scale"]).unflatten(2, (H // Hkv, n))
    seen = (j < lens[:, None, None]) & (j <= last[:, :, None]) & (i < count[:, None])[:, :, None]
    return z.masked_fill_(~seen[:, None, None], float("-inf")), row


def _logsumexp(s):
    """lse ``[N, H]`` of the newest rows over all that they attend."""
    z, _ = _scores(s)
    top = z.amax(-1, keepdim=True)
    total = z.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_().sum(-1, dtype=torch.float64)
    lse = (top[..., 0].double() + total.log()).float()                               # [B, Hkv, g, n]
    b, i = _token_places(s)
    return lse.flatten(1, 2)[b, :, i].contiguous()


def _weights(s):
    case, lens = s["case"], s["lens"].long()
    z, row = _scores(s)
    lse = s["lse"][row].unflatten(2, (case["Hkv"], -1)).permute(0, 2, 3, 1)          # [B, Hkv, g, n]
    w = z.sub_(lse[..., None]).exp_().sum((2, 3), dtype=torch.float64)               # [B, Hkv, max_L]
    n = (s["cu"][1:] - s["cu"][:-1]).long()
    j = torch.arange(s["max_L"], device="cuda").expand(case["B"], -1)
    b, at = ((j < lens[:, None]) & (n > 0)[:, None]).nonzero(as_tuple=True)
    page, slot = s["table"].long()[b, at // case["page"]], at % case["page"]
    old = (at < (lens - n)[b])[:, None] & case["accumulate"]
    s["weights"][page, slot] = (torch.where(old, s["weights"][page, slot].double(), 0.0) + w[b, :, at]).float()
    return s["weights"]


def _evict(s):
    case, lens = s["case"], s["lens"].long()
    B, Hkv, keep = case["B"], case["Hkv"], case["keep"]
    j = torch.arange(s["max_L"], device="cuda").expand(B, -1)
    page, slot = _places(s, j, lens, s["table"])
    w = s["weights"][page, slot].permute(0, 2, 1)                                    # [B, Hkv, max_L]
    always = (j < case["first"]) | (j >= (lens - case["last"])[:, None])
    w = torch.where(always[:, None], float("inf"), w)
    w = torch.where((j < lens[:, None])[:, None], w, float("-inf"))
    best = w.sort(dim=-1, descending=True, stable=True)[1][..., :keep]
    left = lens.clamp(max=keep)
    best = torch.where(best < lens[:, None, None], best, 1 << 30).sort(-1)[0]
    kept = torch.nn.functional.pad(torch.where(best < 1 << 30, best, -1), (0, keep - best.shape[2]), value=-1)
    b, h, i = (kept >= 0).nonzero(as_tuple=True)
    old, new = kept[b, h, i], s["table" if case["in_place"] else "new_table"].long()[b, i // case["page"]]
    at, to = (s["table"].long()[b, old // case["page"]], old % case["page"], h), (new, i % case["page"], h)
    for name in ("k", "v", "k_scale", "v_scale", "weights"):
        if name in s:
            s[name][to] = s[name][at]
    out = {"kept": kept.to(torch.int32), "lens": left.to(torch.int32), "weights": s["weights"]}
    if case["bits"] == 16:
        return out | {"k": s["k"], "v": s["v"]}
    i = torch.arange(keep, device="cuda").expand(B, -1)
    at = _places(s, i, left, s["table" if case["in_place"] else "new_table"])
    inside = (i < left[:, None])[..., None, None]
    return out | {x: torch.where(inside, _values(s, x, *at), 0.0).to(DTYPES[case["dtype"]]) for x in "kv"}


# ── the calls ────────────────────────────────────────────────────────────────


def _run_own(s):
    import longvideosparseattention_amd as lv

    case, kind = s["case"], s["case"]["kind"]
    if "cache" not in s:                       # the handle that a program keeps beside its pages
        s["cache"] = lv.PagedKVCache(s["k"], s["v"], s.get("k_scale"), s.get("v_scale"))
    cache, batch = s["cache"], (s["cu"], s["lens"], s["table"])
    if kind == "means":
        return lv.paged_kv_block_means(cache, s["means"], s["lens"], s["table"], cu_seqlens=s["cu"])
    if kind == "select":
        return lv.paged_kv_select(s["q"], cache, s["means"], *batch, case["top"], tile=case["tile"], first=case["first"],
                                  last=case["last"], causal=case["causal"])
    if kind == "attend":
        o = lv.paged_block_attention(s["q"], cache, s["blocks"], case["block"], *batch, tile=case["tile"], causal=case["causal"],
                                     scale=s["scale"], return_lse=case["lse"])
        return {"o": o[0], "lse": o[1]} if case["lse"] else {"o": o}
    if kind == "weights":
        return lv.paged_kv_weights(s["q"], s["lse"], cache, s["weights"], *batch, causal=case["causal"], scale=s["scale"],
                                   accumulate=case["accumulate"])
    to = None if case["in_place"] else s["new_table"]
    lens, kept = lv.paged_kv_evict(cache, s["weights"], s["lens"], s["table"], case["keep"], first=case["first"], last=case["last"],
                                   new_table=to, return_kept=True)
    out = {"kept": kept, "lens": lens, "weights": s["weights"]}
    if case["bits"] == 16:
        return out | {"k": s["k"], "v": s["v"]}
    k, v = lv.paged_kv_gather(cache, lens, s["table"] if to is None else to, case["keep"], dtype=DTYPES[case["dtype"]])
    return out | {"k": k, "v": v}


def run(state):
    if own:
        return _run_own(state)
    return {"means": _means, "select": _select, "attend": _attend, "weights": _weights, "evict": _evict}[state["case"]["kind"]](state)


def work(case):
    lens, kind = _lengths(case), case["kind"]
    N = sum(n for n, _ in lens)
    H, Hkv, D, bs, tile = case["H"], case["Hkv"], case["D"], case["block"], case["tile"]
    row = Hkv * (2 * D if case["bits"] == 16 else D // 2 + D // 32)             # one token's keys, or values
    total = {"bytes": 0, "flops": 0}

    def add(bytes_, flops=0):
        total["bytes"] += bytes_
        total["flops"] += flops

    for n, L in lens:
        if kind == "means" and n:
            changed = -(-L // bs) - (L - n) // bs
            add((L - (L - n) // bs * bs) * row + 4 * changed * Hkv * D, (L - (L - n) // bs * bs) * Hkv * D)
        if kind == "select" and n:
            tiles = -(-n // tile)
            mean = (L + L - n + 1) / 2 if case["causal"] else L                  # keys that a row sees, on average
            add(2 * n * H * D + 4 * -(-L // bs) * Hkv * D + 4 * tiles * Hkv * case["top"],
                n * H * D + 2 * tiles * Hkv * D * mean / bs)
        if kind == "attend" and n:
            tiles = -(-n // tile)
            mean = (L + L - n + 1) / 2 if case["causal"] else L
            keys = min(case["top"] * bs, mean)                                   # of a row
            add(2 * min(L, tiles * keys) * row + 4 * n * H * D + 4 * n * H * case["lse"] + 4 * tiles * Hkv * case["top"],
                4 * n * H * keys * D)
        if kind == "weights" and n:
            pairs = n * L - (n * (n - 1) // 2 if case["causal"] else 0)
            add(L * row + 2 * n * H * D + 4 * n * H + 4 * Hkv * (L + (L - n) * case["accumulate"]), 2 * D * H * pairs)
        if kind == "evict":
            left = min(L, case["keep"])
            add(4 * L * Hkv + 4 * Hkv * left + 4 * Hkv * case["keep"] + (4 * left * row if left < L or not case["in_place"] else 0))
            if case["bits"] == 4:
                add(2 * left * row + 4 * case["keep"] * Hkv * D)                 # read back
    return total


# ── the same from the definitions, in 64 bits ────────────────────────────────


def _wide(s, name, pages, count):
    """``[count, Hkv, D]`` in 64 bits: the first cached rows of a sequence on ``pages``."""
    x = s[name][pages].flatten(0, 1)[:count]
    if s["case"]["bits"] == 16:
        return x.double()
    c = x.long()
    c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    e, m = (c >> 1) & 3, (c & 1).double()                                        # sign, two exponent bits (bias 1), one of mantissa
    size = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * (1 << (e - 1).clamp(min=0)).double())
    size = torch.where(c >= 8, -size, size)
    step = (s[name + "_scale"][pages].flatten(0, 1)[:count].long() + 896 << 52).view(torch.float64)      # 2^(scale - 127)
    return (size.unflatten(-1, (-1, 32)) * step[..., None]).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    lens, ps, bs, kind, tile = _lengths(case), case["page"], case["block"], case["kind"], case["tile"]
    Hkv, group, H = case["Hkv"], case["H"] // case["Hkv"], case["H"]
    seqs, t0 = [], 0
    for b, (n, L) in enumerate(lens):
        seqs.append((b, n, L, slice(t0, t0 + n), s["table"][b, :-(-L // ps)].long()))
        t0 += n
    if kind == "means":
        out = s["means"].double()
        for b, n, L, _, pages in seqs:
            k = _wide(s, "k", pages, L)
            for j in range((L - n) // bs if n else 1 << 30, -(-L // bs)):
                out[pages[j * bs // ps], j * bs % ps // bs] = k[j * bs:(j + 1) * bs].mean(0)
        return out
    if kind == "select":
        T = s["N"] if tile == 1 else s["N"] // tile + case["B"]
        out = torch.full((T, Hkv, case["top"]), -1, dtype=torch.int32, device="cuda")
        for b, n, L, rows, pages in seqs:
            if not n:
                continue
            blocks, tiles = -(-L // bs), -(-n // tile)
            m = s["means"][pages].flatten(0, 1)[:blocks].double()
            q = torch.zeros(tiles * tile, H, case["D"], dtype=torch.float64, device="cuda")
            q[:n] = s["q"][rows].double()
            q = q.view(tiles, tile, Hkv, group, -1).sum((1, 3))
            i = torch.arange(tiles, device="cuda")
            first, behind = L - n + i * tile, torch.clamp(L - n + (i + 1) * tile, max=L)
            sees = behind if case["causal"] else torch.full_like(behind, L)
            j = torch.arange(blocks, device="cuda")[None]
            always = (j < case["first"]) | (case["last"] > 0) & (j > first[:, None] // bs - case["last"]) & (j <= (behind[:, None] - 1) // bs)
            outside = j * bs >= sees[:, None]
            at = rows.start if tile == 1 else rows.start // tile + b
            for h in range(Hkv):
                z = -(q[:, h] @ m[:, h].T)
                z[always] = -math.inf
                z[outside] = math.inf
                order = np.argsort(z.cpu().numpy(), axis=1, kind="stable")[:, :case["top"]]
                order = torch.from_numpy(order).cuda()
                order = torch.where(torch.gather(outside, 1, order), blocks, order).sort(1)[0]
                out[at:at + tiles, h, :order.shape[1]] = torch.where(order < blocks, order, -1).int()
        return out
    if kind == "evict":
        keep, out = case["keep"], {"weights": s["weights"].double()}
        out |= {"kept": torch.full((case["B"], Hkv, keep), -1, dtype=torch.int32, device="cuda"),
                "lens": torch.tensor([min(L, keep) for _, L in lens], dtype=torch.int32, device="cuda")}
        shape = s["k"].shape if case["bits"] == 16 else (case["B"], keep, Hkv, case["D"])
        out |= {x: s[x].double() if case["bits"] == 16 else torch.zeros(shape, dtype=torch.float64, device="cuda") for x in "kv"}
        for b, n, L, _, pages in seqs:
            if not L:
                continue
            w = s["weights"][pages].flatten(0, 1)[:L]
            rank = w.cpu().numpy().copy()
            rank[:case["first"]] = rank[max(0, L - case["last"]):] = np.inf
            kv = {x: _wide(s, x, pages, L) for x in "kv"}
            left = min(L, keep)
            i = torch.arange(left, device="cuda")
            to = s["table" if case["in_place"] else "new_table"][b].long()[i // ps]
            for h in range(Hkv):
                kept = np.sort(np.lexsort((np.arange(L), -rank[:, h]))[:left])
                kept = torch.from_numpy(kept).cuda()
                out["kept"][b, h, :left] = kept.int()
                out["weights"][to, i % ps, h] = w[kept, h].double()
                for x in "kv":
                    if case["bits"] == 16:
                        out[x][to, i % ps, h] = kv[x][kept, h]
                    else:
                        out[x][b, :left, h] = kv[x][kept, h]
        return out
    if kind == "weights":
        out = s["weights"].double()
    else:
        out = {"o": torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")}
        if case["lse"]:
            out["lse"] = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for b, n, L, rows, pages in seqs:
        if not n:
            continue
        K, j = _wide(s, "k", pages, L), torch.arange(L, device="cuda")
        V = _wide(s, "v", pages, L) if kind == "attend" else None
        page = pages[j // ps]
        for h in range(H):
            z = (s["q"][rows, h].double() @ K[:, h // group].T) * s["scale"]
            if case["causal"]:
                z += torch.full_like(z, -math.inf).triu(L - n + 1)
            if kind == "weights":
                w = torch.exp(z - s["lse"][rows, h].double()[:, None]).sum(0)
                if h % group == 0:
                    out[page[L - n if case["accumulate"] else 0:], (j % ps)[L - n if case["accumulate"] else 0:], h // group] = 0
                out[page, j % ps, h // group] += w
                continue
            at = rows.start if tile == 1 else rows.start // tile + b
            lists = s["blocks"][at:at + -(-n // tile), h // group].long()
            named = torch.zeros(lists.shape[0], -(-L // bs) + 1, dtype=torch.bool, device="cuda")
            named.scatter_(1, torch.where(lists < 0, named.shape[1] - 1, lists), True)
            z[~named[torch.arange(n, device="cuda") // tile][:, j // bs]] = -math.inf
            out["o"][rows, h] = torch.softmax(z, -1) @ V[:, h // group]
            if case["lse"]:
                out["lse"][rows, h] = torch.logsumexp(z, -1)
    return out
