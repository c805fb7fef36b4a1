"""The paged key/value cache of this package as measurable cases.

A sequence's keys and values stay in pages of ``page`` token slots; a table
names the pages of each sequence in order.  Four operators work on it:

* append: new tokens' keys and values written behind a sequence's cached ones,
  rotated by their positions on the way (and their queries with them), in 16
  bits or quantised to 4;
* gather: the cached keys and values of every sequence read back as padded
  ``[B, S, H, D]`` tensors;
* attention over the pages: queries of the newest tokens of every sequence
  over all its cached tokens, causal or not;
* the same over pages held in 4 bits (E2M1 codes, a power-of-two scale for
  every 32 values of a row).

Geometry of a case: ``B`` sequences of up to ``L`` cached tokens, the newest
``n`` of them this call's, the last ``empty`` sequences without any; ``H``
query and ``Hkv`` key heads of size ``D``; ``rot`` rotated dimensions.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
SPARE_PAGES = 3


def _case(name, kind, B, n, L, H, Hkv, D, page, bits=16, dtype="bf16", causal=True, ragged=False, empty=0,
          rot=0, interleaved=False, layout="heads", lse=False):
    return {"name": name, "kind": kind, "B": B, "n": n, "L": L, "H": H, "Hkv": Hkv, "D": D, "page": page, "bits": bits,
            "dtype": dtype, "causal": causal, "ragged": ragged, "empty": empty, "rot": rot,
            "interleaved": interleaved, "layout": layout, "lse": lse}


def listed():
    return [
        # One token for each of a batch of text streams: rotated and appended, the small call of every decoding step.
        _case("append_step", "append", 32, 1, 2100, 32, 8, 128, 16, ragged=True, rot=128),
        # Three new frames of a video stream, one frame a page, rotated in pairs as the video models do.
        _case("append_frames", "append", 1, 4680, 9360, 12, 12, 128, 1560, rot=128, interleaved=True),
        # Prompts of different lengths put into a 4-bit cache, and the values that it now stands for read back.
        _case("append_prompts_4bit", "append_gather", 8, 1900, 1900, 32, 8, 128, 64, bits=4, dtype="f16", ragged=True,
              rot=64),
        # The cached frames of a stream handed to the sparse attention as plain tensors.
        _case("gather_frames", "gather", 1, 0, 15600, 12, 12, 128, 1560),
        # Cached prompts of a small head size read back from 4 bits, padded to the longest.
        _case("gather_4bit", "gather", 12, 0, 2500, 16, 16, 64, 32, bits=4, ragged=True),
        # One stream's next token after a prompt: the smallest call, nothing but latency.
        _case("decode_one", "attend", 1, 1, 1001, 16, 4, 128, 16),
        # A serving batch's next tokens over long ragged caches, grouped heads, three slots without a request.
        _case("decode_batch", "attend", 48, 1, 16000, 32, 8, 128, 64, ragged=True, empty=3, lse=True),
        # Ragged prompts' newest parts over what was cached before them, fp16, causal.
        _case("prompts_causal", "attend", 6, 1700, 5200, 16, 4, 64, 16, dtype="f16", ragged=True),
        # Three new frames of a video stream over fifteen cached and themselves, no causal order inside the chunk.
        _case("frames_chunk", "attend", 1, 4680, 28080, 12, 12, 128, 1560, causal=False, layout="tokens"),
        # One stream's next token over a 4-bit cache.
        _case("decode_one_4bit", "attend", 1, 1, 1001, 16, 4, 128, 16, bits=4),
        # A serving batch over caches that only fit in 4 bits.
        _case("decode_batch_4bit", "attend", 40, 1, 32000, 32, 8, 128, 64, bits=4, ragged=True),
        # A low-resolution stream's new frames over a long 4-bit history, the widest heads.
        _case("frames_chunk_4bit", "attend", 1, 780, 31200, 12, 4, 256, 390, bits=4, causal=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    """One more call of the listed ranges: every operator, head size, type, page size and group of heads."""
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["append", "append_gather", "gather", "attend", "attend", "attend", "attend"])
        D, Hkv, group = rng.choice([64, 96, 128, 128, 192, 256]), rng.choice([1, 2, 4, 5, 8, 12]), rng.choice([1, 1, 2, 3, 4, 6, 8])
        page = rng.choice([1, 7, 16, 16, 32, 64, 64, 100, 256, 390, 1560])
        bits = 4 if kind == "append_gather" else rng.choice([16, 4])
        rot = rng.choice([0, 32, D // 2, D, D]) if kind.startswith("append") else 0
        style = rng.choice(["step", "few", "chunk"])
        if style == "step":
            B, n, L = _log_int(rng, 1, 64), 1, _log_int(rng, 1, 32000)
        elif style == "few":
            B, n, L = _log_int(rng, 1, 24), rng.randint(2, 9), _log_int(rng, 9, 16000)
        else:
            B, L = _log_int(rng, 1, 8), _log_int(rng, 40, 28000)
            n = _log_int(rng, min(16, L), min(L, 4700))
        if kind in ("append", "append_gather"):
            L = min(L, max(n, 9000))
        if kind == "gather":
            n, L = 0, min(L, 16000)
        empty = rng.choice([0, 0, 1]) if B > 1 else 0
        causal = kind != "attend" or rng.random() < 0.6
        case = _case("", kind if bits == 4 or kind != "append_gather" else "append", B, n, L, Hkv * group, Hkv, D, page, bits,
                     rng.choice(["bf16", "bf16", "f16"]), causal, B > 1 and rng.random() < 0.7, empty, rot, rng.random() < 0.4,
                     rng.choice(["heads", "tokens"]), kind == "attend" and rng.random() < 0.3)
        del case["name"]
        if kind == "append" and bits == 4:
            case["kind"] = "append_gather"
        scores = B * case["H"] * max(n, 1) * L                      # of the plain form, which pads every sequence
        if _cost(case) <= most and scores <= 3.2e9 and B * L * Hkv * D <= 2.2e9:
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


def _strided(shape, layout, dtype, fill=None):
    """A ``[pages, page, Hkv, X]`` tensor, a page's rows of one head next to each other or a token's heads."""
    P, ps, Hkv, X = shape
    t = torch.empty((P, Hkv, ps, X) if layout == "heads" else shape, dtype=dtype, device="cuda")
    t = t.transpose(1, 2) if layout == "heads" else t
    if fill is not None:
        t.copy_(fill)
    return t


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    B, H, Hkv, D, ps = case["B"], case["H"], case["Hkv"], case["D"], case["page"]
    lens = _lengths(case)
    N = sum(n for n, _ in lens)
    counts = [-(-L // ps) for _, L in lens]
    P = sum(counts) + SPARE_PAGES
    order = torch.randperm(P, generator=g, device="cuda").to(torch.int32).cpu()
    table, at = torch.zeros(B, max(max(counts), 1), dtype=torch.int32), 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    ends = torch.tensor([0] + [n for n, _ in lens]).cumsum(0)
    s = {"case": case, "N": N, "max_n": max(n for n, _ in lens), "max_L": max(L for _, L in lens),
         "cu": ends.to(torch.int32).cuda(), "lens": torch.tensor([L for _, L in lens], dtype=torch.int32).cuda(),
         "table": table.cuda(), "scale": 1.0 / math.sqrt(D)}

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    channel = 0.5 + 1.5 * torch.rand(Hkv, D, generator=g, device="cuda")      # keys: channels of different size
    for name in ("k", "v"):
        x = normal(P, ps, Hkv, D)
        if name == "k":
            x *= channel
        if case["bits"] == 16:
            s[name] = _strided((P, ps, Hkv, D), case["layout"], dt, x)
        else:
            codes, scales = _quantize(x)
            s[name] = _strided((P, ps, Hkv, D // 2), case["layout"], torch.uint8, codes)
            s[name + "_scale"] = _strided((P, ps, Hkv, D // 32), case["layout"], torch.uint8, scales)
    if case["kind"] == "attend":
        s["q"] = (1.5 * normal(N, H, D)).to(dt)
    elif case["kind"].startswith("append"):
        s["q"], s["new_v"] = normal(N, H, D).to(dt), normal(N, Hkv, D).to(dt)
        s["new_k"] = (normal(N, Hkv, D) * channel).to(dt)
        if case["rot"]:
            freq = 10000.0 ** (-torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64) / (case["rot"] // 2))
            angle = torch.arange(s["max_L"], device="cuda", dtype=torch.float64)[:, None] * freq
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


# ── the plain forms ──────────────────────────────────────────────────────────


def _quantize(x):
    """(codes, scales) of values ``[..., D]``: for every 32 the smallest 2^e with 6 * 2^e >= all of them (e from -23 to
    13, kept as e + 127), and the nearest E2M1 number of each quotient, ties to even, two to a byte, the even one low."""
    D = x.shape[-1]
    x = x.unflatten(-1, (D // 32, 32))
    mant, e = torch.frexp(x.abs().amax(-1))                          # amax = mant * 2^e, mant in [0.5, 1)
    e = torch.where(mant > 0, e - 3 + (mant > 0.75), -23).clamp(-23, 13)
    a = x.abs() * _power(-e).to(x.dtype)[..., None]
    up = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (up + 8 * torch.signbit(x)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _power(e):
    """2^e as fp32, from the bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _dequantize(codes, scales):
    levels = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=codes.device)
    x = torch.stack((levels[(codes & 15).int()], levels[(codes >> 4).int()]), -1).flatten(-2)
    return x * _power(scales.to(torch.int32) - 127).repeat_interleave(32, -1)


def _slots(s, pos):
    """Page and slot of position ``pos[b, i]`` of sequence b; positions behind the end: its first page's."""
    ps = s["case"]["page"]
    pos = torch.where((pos >= 0) & (pos < s["lens"][:, None]), pos, 0)
    return torch.gather(s["table"].long(), 1, pos // ps), pos % ps


def _cached(s):
    """Keys and values of every sequence in 32 bits, ``[B, max_L, Hkv, D]``."""
    pos = torch.arange(s["max_L"], device="cuda").expand(s["lens"].numel(), -1)
    page, slot = _slots(s, pos)
    if s["case"]["bits"] == 16:
        return s["k"][page, slot].float(), s["v"][page, slot].float()
    return (_dequantize(s["k"][page, slot], s["k_scale"][page, slot]),
            _dequantize(s["v"][page, slot], s["v_scale"][page, slot]))


def _token_places(s):
    """Sequence and position of each new token."""
    t = torch.arange(s["N"], device="cuda")
    b = torch.searchsorted(s["cu"].long(), t, right=True) - 1
    return b, t, s["lens"].long()[b] - s["cu"].long()[b + 1] + t


def _rotate(x, s, pos):
    """The first ``rot`` dimensions turned by the token's angles: pairs (2i, 2i + 1), or (i, i + rot / 2)."""
    rot = s["case"]["rot"]
    x = x.double()
    if not rot:
        return x
    cos, sin = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
    if s["case"]["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _append(s):
    case, dt = s["case"], s["q"].dtype
    b, _, pos = _token_places(s)
    page, slot = s["table"].long()[b, pos // case["page"]], pos % case["page"]
    k, v, q = _rotate(s["new_k"], s, pos), s["new_v"], _rotate(s["q"], s, pos).to(dt)
    if case["bits"] == 16:
        s["k"][page, slot], s["v"][page, slot] = k.to(dt), v
        return {"k": s["k"], "v": s["v"], "q": q}
    s["k"][page, slot], s["k_scale"][page, slot] = _quantize(k)
    s["v"][page, slot], s["v_scale"][page, slot] = _quantize(v.double())
    return {"q": q} | _gather(s)


def _gather(s):
    k, v = _cached(s)
    inside = (torch.arange(s["max_L"], device="cuda") < s["lens"][:, None])[..., None, None]
    dt = DTYPES[s["case"]["dtype"]]
    return {"k": torch.where(inside, k, 0.0).to(dt), "v": torch.where(inside, v, 0.0).to(dt)}


def _attend(s):
    case, q = s["case"], s["q"]
    B, H, Hkv, D, n = case["B"], case["H"], case["Hkv"], case["D"], s["max_n"]
    k, v = _cached(s)
    lens, cu = s["lens"].long(), s["cu"].long()
    row = torch.arange(n, device="cuda")
    last = (lens - (cu[1:] - cu[:-1]))[:, None] + row if case["causal"] else (lens - 1)[:, None].expand(B, n)
    qb = q[(cu[:-1, None] + row).clamp(max=s["N"] - 1)].float()                         # [B, n, H, D]
    qb = qb.unflatten(2, (Hkv, H // Hkv)).permute(0, 2, 3, 1, 4).flatten(2, 3)          # [B, Hkv, g * n, D]
    p = torch.matmul(qb, k.permute(0, 2, 3, 1)) * s["scale"]
    j = torch.arange(s["max_L"], device="cuda")
    seen = (j < lens[:, None, None]) & (j <= last[:, :, None])                          # [B, n, max_L]
    p = p.unflatten(2, (H // Hkv, n)).masked_fill_(~seen[:, None, None], float("-inf")).flatten(2, 3)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.transpose(1, 2)) / torch.where(total > 0, total, 1.0)
    o = o.unflatten(2, (H // Hkv, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)              # [B, n, H, D]
    b, t, _ = _token_places(s)
    out = {"o": o[b, t - cu[b]].to(q.dtype)}
    if case["lse"]:
        lse = (top + total.log())[..., 0].unflatten(2, (H // Hkv, n)).permute(0, 3, 1, 2).flatten(2, 3)
        out["lse"] = lse[b, t - cu[b]]
    return out


# ── the calls ────────────────────────────────────────────────────────────────


def _run_own(s):
    import longvideosparseattention_amd as lv

    case, kind = s["case"], s["case"]["kind"]
    if "cache" not in s:                       # the handle that a program keeps beside its pages
        s["cache"] = lv.PagedKVCache(s["k"], s["v"], s.get("k_scale"), s.get("v_scale"))
    cache, out = s["cache"], {}
    if kind.startswith("append"):
        out["q"] = lv.paged_kv_append(cache, s["new_k"], s["new_v"], s["cu"], s["lens"], s["table"], q=s["q"],
                                      cos=s.get("cos"), sin=s.get("sin"), interleaved=case["interleaved"])
        if kind == "append":
            return out | {"k": s["k"], "v": s["v"]}
    if kind != "attend":
        k, v = lv.paged_kv_gather(cache, s["lens"], s["table"], s["max_L"], dtype=DTYPES[case["dtype"]])
        return out | {"k": k, "v": v}
    o = lv.paged_attention(s["q"], cache, s["cu"], s["lens"], s["table"], causal=case["causal"], scale=s["scale"],
                           return_lse=case["lse"], max_q_len=s["max_n"])
    return {"o": o[0], "lse": o[1]} if case["lse"] else {"o": o}


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    return _attend(state) if kind == "attend" else _gather(state) if kind == "gather" else _append(state)


def work(case):
    lens, kind = _lengths(case), case["kind"]
    N, L = sum(n for n, _ in lens), sum(x for _, x in lens)
    H, Hkv, D, rot = case["H"], case["Hkv"], case["D"], case["rot"]
    row = Hkv * (2 * D if case["bits"] == 16 else D // 2 + D // 32)             # one token's keys, or values
    if kind == "attend":
        pairs = sum(n * x - (n * (n - 1) // 2 if case["causal"] else 0) for n, x in lens)
        return {"bytes": 2 * L * row + 2 * 2 * N * H * D + 4 * N * H * case["lse"], "flops": 4 * D * H * pairs}
    padded = 2 * 2 * len(lens) * max(x for _, x in lens) * Hkv * D              # both gathered tensors
    if kind == "gather":
        return {"bytes": 2 * L * row + padded, "flops": 0}
    angles = 4 * rot * max(x for _, x in lens) if N > max(x for _, x in lens) else 4 * rot * N
    moved = 2 * N * (Hkv * D * 2 + row) + 2 * 2 * N * H * D + angles
    return {"bytes": moved + (2 * L * row + padded if kind == "append_gather" else 0), "flops": 3 * rot * N * (H + Hkv)}


# ── the same from the definitions, in 64 bits ────────────────────────────────


def _e2m1(nibble):
    """An E2M1 number from its bits: sign, two exponent bits (bias 1), one mantissa bit."""
    e, m = (nibble >> 1) & 3, (nibble & 1).double()
    size = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * (1 << (e - 1).clamp(min=0)).double())
    return torch.where(nibble >= 8, -size, size)


def _wide(codes, scales):
    """``[L, Hkv, D]`` in 64 bits from a sequence's codes and scales."""
    c = codes.long()
    x = torch.empty(*c.shape[:-1], 2 * c.shape[-1], dtype=torch.float64, device=c.device)
    x[..., 0::2], x[..., 1::2] = _e2m1(c & 15), _e2m1(c >> 4)
    step = (scales.long() + 896 << 52).view(torch.float64)                       # 2^(scale - 127)
    return (x.unflatten(-1, (-1, 32)) * step[..., None]).flatten(-2)


def _nearest(x):
    """What 4 bits hold of ``x [..., D]``."""
    D = x.shape[-1]
    groups = x.reshape(*x.shape[:-1], D // 32, 32)
    most = groups.abs().amax(-1, keepdim=True)
    step = torch.full_like(most, 2.0 ** 13)
    for e in range(12, -24, -1):                                                 # the smallest that reaches
        step = torch.where(6 * 2.0 ** e >= most, torch.full_like(step, 2.0 ** e), step)
    size = (groups.abs() / step).clamp(max=6.0)
    # numbers of two binades and the subnormals: spacing 0.5 below 2, 1 below 4, 2 up to 6; round() takes ties to even
    spacing = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0)).double()
    return (torch.copysign(torch.round(size / spacing) * spacing, groups) * step).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    lens, ps, kind = _lengths(case), case["page"], case["kind"]
    Hkv, group, D, rot = case["Hkv"], case["H"] // case["Hkv"], case["D"], case["rot"]
    out, t0 = {}, 0
    if kind.startswith("append"):
        out["q"] = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        if kind == "append":
            out |= {"k": s["k"].double(), "v": s["v"].double()}
    if kind in ("gather", "append_gather"):
        out |= {x: torch.zeros(len(lens), s["max_L"], Hkv, D, dtype=torch.float64, device="cuda") for x in "kv"}
    if kind == "attend":
        out["o"] = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        if case["lse"]:
            out["lse"] = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")

    def turned(x, first):
        x = x.double().clone()
        if rot:
            c, d = (s[w][first:first + x.shape[0]].double().unsqueeze(1) for w in ("cos", "sin"))
            i = torch.arange(rot // 2, device="cuda")
            i, j = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
            a, b = x[..., i], x[..., j]
            x[..., i], x[..., j] = c * a - d * b, d * a + c * b
        return x

    for b, (n, L) in enumerate(lens):
        pages = s["table"][b, :-(-L // ps)].long()
        rows = {w: s[w][pages].flatten(0, 1)[:L] for w in ("k", "v", "k_scale", "v_scale") if w in s}
        new = slice(t0, t0 + n)
        if kind.startswith("append"):
            k, v = turned(s["new_k"][new], L - n), s["new_v"][new].double()
            out["q"][new] = turned(s["q"][new], L - n)
            if kind == "append":
                at = torch.arange(L - n, L, device="cuda")
                out["k"][pages[at // ps], at % ps], out["v"][pages[at // ps], at % ps] = k, v
        if kind in ("gather", "append_gather") or kind == "attend":
            K, V = ((rows[w].double() if case["bits"] == 16 else _wide(rows[w], rows[w + "_scale"])) for w in ("k", "v"))
        if kind == "append_gather" and n:
            K[L - n:], V[L - n:] = _nearest(k), _nearest(v)
        if kind in ("gather", "append_gather"):
            out["k"][b, :L], out["v"][b, :L] = K, V
        if kind == "attend" and n:
            for h in range(case["H"]):
                z = (s["q"][new, h].double() @ K[:, h // group].T) * s["scale"]
                if case["causal"]:
                    z += torch.full_like(z, float("-inf")).triu(L - n + 1)
                out["o"][new, h] = torch.softmax(z, -1) @ V[:, h // group]
                if case["lse"]:
                    out["lse"][new, h] = torch.logsumexp(z, -1)
        t0 += n
    return out
