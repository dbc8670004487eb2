"""Rotary positions, attention weights and eviction written plainly, in 64 bits, and how far
a kernel may be from them."""

from __future__ import annotations

import math

import torch

D = 128
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def rope(x, positions, frequencies, layout, scale=1.0, inverse=False):
    """(turned rows, what each may be off by).  Pair by pair, each coordinate by itself."""
    n = frequencies.numel()
    y, big = x.double().clone(), x.double().abs()
    angle = positions.double()[:, None, None] * frequencies
    cos, sin = torch.cos(angle) * scale, torch.sin(angle) * scale
    if inverse:
        sin = -sin
    pairs = torch.arange(n, device=x.device)
    i, j = (pairs, pairs + n) if layout == "half" else (2 * pairs, 2 * pairs + 1)
    a, b = x[..., i].double(), x[..., j].double()
    y[..., i], y[..., j] = a * cos - b * sin, b * cos + a * sin
    both = (a.abs() + b.abs()) * abs(scale)
    big[..., i], big[..., j] = both, both
    # sine and cosine: 2^-21.19 and 2^-21.41 (CUDA's documents, for [-pi, pi]), the angle's
    # reduction (two roundings of a part of a turn: 2^-24 turns, 2 pi's: 2^-24 of pi, and
    # 2^-53 of the 64-bit angle), scale, product, sum: 3 roundings; then the rounding to the type
    turns = (positions.double().abs()[:, None, None] * frequencies.abs().max().clamp(min=1e-9)
             if n else 0.0)
    arithmetic = big * (2.0 ** -21.19 + 3 * math.pi * 2.0 ** -24 + 3 * 2.0 ** -24
                        + turns * 4 * 2.0 ** -53)
    tol = y.abs() * UNIT[x.dtype] + arithmetic * (1 + UNIT[x.dtype]) + smallest(x.dtype)
    tol[..., 2 * n:] = 0.0
    return y, tol


def smallest(dtype):
    """Half a step of the subnormal numbers."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134


def dense(pages, row, n, head):
    size = pages.shape[2]
    j = torch.arange(n, device=pages.device)
    return pages[row[j // size].long(), head, j % size]


def attention_lse(q, k_pages, table, cu_q, kv_lens, window=0, scale=None):
    """log-sum-exp [T, q_heads], 64 bits rounded to 32; -inf where nothing is seen."""
    out = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    for b, s, seen, rows, heads, _ in _scores(q, k_pages, table, cu_q, kv_lens, window, scale):
        s = s.masked_fill(~seen[:, None], -math.inf)
        out[rows, heads] = torch.logsumexp(s, -1)
    return out.float()


def _scores(q, k_pages, table, cu_q, kv_lens, window, scale):
    """Per request and KV head: scores [n, R, kv], who sees whom [n, kv], and where from."""
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    G = k_pages.shape[1]
    R = q.shape[1] // G
    cu, kvs = cu_q.tolist(), kv_lens.tolist()
    for b, kv in enumerate(kvs):
        n = cu[b + 1] - cu[b]
        if n <= 0 or kv <= 0:
            continue
        p = kv - n + torch.arange(n, device=q.device)
        j = torch.arange(kv, device=q.device)
        seen = j <= p[:, None]
        if window:
            seen &= j > p[:, None] - window
        for g in range(G):
            k = dense(k_pages, table[b], kv, g).double()
            x = q[cu[b]:cu[b + 1], g * R:(g + 1) * R].double()
            size = (x.abs() @ k.abs().T) * scale
            yield (b, (x @ k.T) * scale, seen, slice(cu[b], cu[b + 1]),
                   slice(g * R, (g + 1) * R), (g, size))


def weights(q, k_pages, table, cu_q, kv_lens, lse, before, *, window=0, last=0, scale=None):
    """(row weights after the call, what each may be off by).

    A weight exp(d), d = s - lse: the score's sum of 128 products is off by 128 steps of its
    terms' sum (2^-23 each: the tensor cores cut where others round), d by its rounding, the
    scale's and that of the product with log2(e) and of log2(e) itself, 2^x by 2^-22.  A sum
    of n weights by one rounding for each number that goes into one place: 32 of a tile's
    128 columns, the tiles, the parts of a cluster, 6 more."""
    out = before.double().clone()
    tol = torch.zeros_like(out)
    eps = 2.0 ** -24
    size_of = k_pages.shape[2]
    for b, s, seen, rows, heads, (g, size) in _scores(q, k_pages, table, cu_q, kv_lens, window,
                                                      scale):
        n, R, kv = s.shape
        z = lse[rows, heads].double()[..., None]
        d = s - z
        e = torch.exp(d)
        e = torch.where(z == -math.inf, torch.zeros_like(e), e)
        counted = torch.arange(n, device=q.device) >= (n - last if last else 0)
        use = (seen & counted[:, None])[:, None].expand_as(e)
        e = torch.where(use, e, torch.zeros_like(e))
        off = 256 * eps * size + eps * (s.abs() + 4 * d.abs()) + 4 * eps
        off = torch.where(use & torch.isfinite(off), torch.expm1(off.clamp(max=50.0)),
                          torch.zeros_like(off))
        total = e.sum((0, 1))
        adds = 32 + n * R / (128 // R * R) + 8 + 6
        err = (e * off).sum((0, 1)) + total * adds * eps + n * R * 2.0 ** -126
        j = torch.arange(kv, device=q.device)
        at = (table[b][j // size_of].long(), torch.full_like(j, g), j % size_of)
        out[at] += total
        tol[at] += err + (out[at].abs() * eps).nan_to_num(0.0)
    return out, tol


def evict(pools, row_weights, row_positions, table, lens, keep, offsets, *, sink, recent, page):
    """Python lists and loops: every tensor [layers, pages, heads, page(, D)] on the CPU is
    changed in place; returns (lens, offsets, pages that come back)."""
    back, lens_out, offsets_out = [], [], []
    layers, _, heads, _ = row_weights.shape
    for b, (n, budget) in enumerate(zip(lens, keep)):
        if budget < 0 or n <= budget:
            lens_out.append(n)
            offsets_out.append(offsets[b])
            continue
        spot = [(table[b][j // page], j % page) for j in range(n)]
        for l in range(layers):
            for g in range(heads):
                def rank(j):
                    p = int(row_positions[l, spot[j][0], g, spot[j][1]])
                    w = float(row_weights[l, spot[j][0], g, spot[j][1]])
                    if p < sink or p >= n + offsets[b] - recent:
                        return (0, 0.0, j)
                    return (1, -math.inf, j) if math.isnan(w) else (2, -w, j)
                stays = sorted(sorted(range(n), key=rank)[:budget])
                holes = sorted(set(range(budget)) - set(stays))
                movers = [j for j in stays if j >= budget]
                assert len(holes) == len(movers)
                for to, source in zip(holes, movers):
                    (tp, to_row), (sp, so) = spot[to], spot[source]
                    for t in (*pools, row_weights, row_positions):
                        t[l, tp, g, to_row] = t[l, sp, g, so]
        back += table[b][-(-budget // page):-(-n // page)]
        lens_out.append(budget)
        offsets_out.append(offsets[b] + n - budget)
    return lens_out, offsets_out, back
