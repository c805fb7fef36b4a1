"""What works on parts of the paged cache, from its definitions, in 64 bits and on the CPU (see paged_ref.py for
batches and dense attention)."""
import math

import torch

from paged_ref import F32, U


def tiles(b, tile):
    """``(list, sequence, first row, end of rows, position of the first row)`` of every tile, and how many lists there are."""
    got = []
    for s, (n, L) in enumerate(b.seqs):
        for i in range(-(-n // tile)):
            at = b.ends[s] + i if tile == 1 else b.ends[s] // tile + s + i
            r0, r1 = b.ends[s] + i * tile, b.ends[s] + min(n, (i + 1) * tile)
            got.append((at, s, r0, r1, L - n + i * tile))
    return got, b.N if tile == 1 else b.N // tile + len(b.seqs)


def means(b, block):
    """``[L / block, Hkv, D]`` of every sequence."""
    return [torch.stack([K[j:j + block].double().mean(0) for j in range(0, K.shape[0], block)]) if K.shape[0] else K.double()
            for K in b.K]


def paged(b, rows, block, fill, like):
    """Per-sequence block rows ``[blocks, ...]`` put beside the pages as ``like`` is laid out."""
    out = torch.full(like.shape, fill, dtype=torch.float32)
    for s, x in enumerate(rows):
        for j in range(x.shape[0]):
            out[b.pages[s][j * block // b.ps], j * block % b.ps // block] = x[j].float()
    return out


def select(b, q, rows, block, top, tile, first, last, causal):
    """Lists from per-sequence means ``rows`` (what the call is given, fp32)."""
    todo, T = tiles(b, tile)
    g = b.H // b.Hkv
    out = torch.full((T, b.Hkv, top), -1, dtype=torch.int32)
    q = q.double().cpu()
    for at, s, r0, r1, p0 in todo:
        L = b.seqs[s][1]
        end = p0 + (r1 - r0)
        lim = max(0, min(L, end)) if causal else L
        blocks = -(-lim // block)
        Q = q[r0:r1].unflatten(1, (b.Hkv, g)).sum((0, 2))
        near = range(max(p0, 0) // block - (last - 1), (end - 1) // block + 1) if last and end > 0 else range(0)
        for h in range(b.Hkv):
            z = (rows[s][:blocks, h].double() @ Q[h]).tolist() if blocks else []
            rank = [math.inf if j < first or j in near else (-math.inf if math.isnan(x) else x) for j, x in enumerate(z)]
            nan = [not (j < first or j in near) and math.isnan(x) for j, x in enumerate(z)]
            order = sorted(range(blocks), key=lambda j: (not (j < first or j in near), nan[j], -rank[j], j))[:top]
            out[at, h, :len(order)] = torch.tensor(sorted(order), dtype=torch.int32)
    return out


def attention(b, q, lists, block, tile, causal, scale=None):
    """``(o, lse, tolerance of o, tolerance of lse)``: paged_ref.attention's arithmetic over the keys of the lists."""
    scale = 1.0 / math.sqrt(b.D) if scale is None else scale
    u, g = U[b.dtype], b.H // b.Hkv
    o = torch.zeros(b.N, b.H, b.D, dtype=torch.float64)
    tol = torch.zeros_like(o)
    lse = torch.full((b.N, b.H), float("-inf"), dtype=torch.float64)
    lse_tol = torch.zeros_like(lse)
    q, lists = q.double().cpu(), lists.cpu()
    for at, s, r0, r1, p0 in tiles(b, tile)[0]:
        L = b.seqs[s][1]
        for hk in range(b.Hkv):
            ids = [x for x in lists[at, hk].tolist()]
            ids = ids[:ids.index(-1)] if -1 in ids else ids
            pos = torch.tensor([p for j in ids for p in range(j * block, min(L, (j + 1) * block))], dtype=torch.long)
            for t in range(r0, r1):
                mine = pos[pos <= p0 + t - r0] if causal else pos
                if not mine.numel():
                    continue
                K, V = b.K[s][mine, hk].double(), b.V[s][mine, hk].double()
                Q = q[t, hk * g:(hk + 1) * g]
                z = Q @ K.T * scale
                size = (Q.abs() @ K.abs().T * scale).amax(-1, keepdim=True)
                top = z.amax(-1, keepdim=True)
                w = torch.exp(z - top)
                total = w.sum(-1, keepdim=True)
                row = w / total @ V
                A = w / total @ V.abs()
                d = (b.D + 4) * F32 * size + 4 * F32 * top.abs()
                h = slice(hk * g, (hk + 1) * g)
                o[t, h] = row
                tol[t, h] = u * row.abs() + A * (u + 2 * d + 2 * (L + 64) * F32)
                lse[t, h] = (top + total.log())[:, 0]
                lse_tol[t, h] = (d + (L + 64) * F32 + 8 * F32 * (top.abs() + total.log().abs()))[:, 0]
    return o, lse, tol, lse_tol


def weights(b, q, lse, causal, scale=None):
    """Per sequence ``([L, Hkv] sums, tolerances)`` for the lse that the call is given.

    A score is an fp32 sum of D exact products, off by D * 2^-24 of the sum of magnitudes; the exponent's argument, score *
    scale * log2(e) - lse * log2(e), rounds twice to fp32 at the size of its terms and the exponential is off by 2 * 2^-24;
    sums over the rows round in fp32 (as many times as there are rows, at most)."""
    scale = 1.0 / math.sqrt(b.D) if scale is None else scale
    g, got = b.H // b.Hkv, []
    q, lse = q.double().cpu(), lse.double().cpu()
    for s, (n, L) in enumerate(b.seqs):
        w, tol = torch.zeros(L, b.Hkv, dtype=torch.float64), torch.zeros(L, b.Hkv, dtype=torch.float64)
        for h in range(b.H if n else 0):
            r = slice(b.ends[s], b.ends[s + 1])
            K = b.K[s][:, h // g].double()
            z = q[r, h] @ K.T * scale
            size = q[r, h].abs() @ K.abs().T * scale
            l = lse[r, h][:, None]
            fine = torch.isfinite(l)
            l = torch.where(fine, l, torch.zeros_like(l))
            seen = fine & (torch.arange(L)[None] <= torch.arange(L - n, L)[:, None] if causal else torch.ones(n, L, dtype=torch.bool))
            p = torch.where(seen, torch.exp(z - l), torch.zeros_like(z))
            d = (b.D + 4) * F32 * size + 4 * F32 * (z.abs() + l.abs()) + 4 * F32
            w[:, h // g] += p.sum(0)
            tol[:, h // g] += torch.where(seen, p * d, torch.zeros_like(p)).sum(0)
        rows = n * g
        got.append((w, tol * 1.01 + w * (rows + 8) * F32))
    return got


def kept(w, L, keep, first, last):
    """Positions that stay of one head's weights ``w [L]``."""
    if L <= keep:
        return list(range(L))
    x = w.double().tolist()
    always = [j < first or j >= L - last for j in range(L)]
    order = sorted(range(L), key=lambda j: (not always[j], not always[j] and math.isnan(x[j]),
                                            0.0 if always[j] or math.isnan(x[j]) else -x[j], j))
    return sorted(order[:keep])
