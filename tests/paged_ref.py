"""The paged cache's operators written plainly: the step plan over Python lists,
attention in 64 bits, and how far a 16-bit kernel may be from it."""

from __future__ import annotations

import math

import torch

# unit roundoff of the types (p bits of significand: 2^-p)
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def step(lens, new, table, stack, count, *, page, tokens_cap, num_pages):
    """(table, stack, kv_lens, cu_q, slots, positions, count, error) of one step."""
    table = [list(r) for r in table]
    stack = list(stack)
    width = len(table[0])
    cdiv = lambda a: -(-a // page)  # noqa: E731
    error = 0
    for b, x in enumerate(new):
        if x < 0:
            for i in range(cdiv(lens[b])):
                stack[count] = table[b][i]
                count += 1
    top = count
    wanted, kv, cu, slots, positions = 0, [], [0], [], []
    for b, x in enumerate(new):
        if x < 0:
            kv.append(0)
            cu.append(cu[-1])
            continue
        have = cdiv(lens[b])
        need = cdiv(lens[b] + x) - have
        ok = have + need <= width
        if ok:
            wanted += need
            ok = need == 0 or wanted <= top
        if ok:
            for i in range(need):
                count -= 1
                table[b][have + i] = stack[count]
        else:
            error = 3
        kv.append(lens[b] + x if ok else lens[b])
        cu.append(cu[-1] + x)
        for i in range(x):
            p = lens[b] + i
            positions.append(p)
            slots.append(table[b][p // page] * page + p % page if ok else -1)
    if len(slots) > tokens_cap:
        error = 3
    slots = (slots + [-1] * tokens_cap)[:tokens_cap]
    positions = (positions + [0] * tokens_cap)[:tokens_cap]
    return table, stack, kv, cu, slots, positions, count, error


def dense(pages, table_row, n, head):
    """Rows 0 .. n of one head of a request: [n, D] in 64 bits."""
    size = pages.shape[2]
    ids = table_row[:-(-n // size)].long()
    return pages[ids, head].reshape(-1, pages.shape[-1])[:n].double()


def attention(q, k_pages, v_pages, table, cu_q, kv_lens, *, window=0, scale=None,
              out_dtype=None):
    """(out, lse, out tolerance, lse tolerance), all [T, heads, ...] in 64 bits.

    Tolerances, from the kernel's arithmetic (16-bit products are exact in 32
    bits):
    * a score sums 128 products in 32 bits and is scaled: its error is at most
      e = 130 * 2^-24 * scale * sum|q k| + 2^-22 * |s| (the last for the
      exponent's argument), which changes each weight by a factor of at most 1 +- 2e
      against the others (2e: error of the score and of the row's maximum);
    * exp2 and the running rescaling: 2^-20 relative;
    * weights are rounded to the 16-bit type for the product with V: unit u each,
      and fp16 loses what is below 2^-25 of the row's largest weight;
    * sums over n keys in 32 bits: n * 2^-24 relative;
    * the result is rounded once to its type."""
    T, H, D = q.shape
    r = H // k_pages.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    unit = UNIT[q.dtype]
    unit_out = UNIT[out_dtype or q.dtype]
    out = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    tol_lse = torch.zeros_like(lse)
    cu, kv = cu_q.tolist(), kv_lens.tolist()
    for b, n_kv in enumerate(kv):
        first, n = cu[b], cu[b + 1] - cu[b]
        if n == 0 or n_kv == 0:
            continue
        p = torch.arange(n, device=q.device)[:, None] + n_kv - n
        j = torch.arange(n_kv, device=q.device)
        seen = (j <= p) & ((j > p - window) if window else torch.ones_like(j, dtype=torch.bool))
        for h in range(H):
            x = q[first:first + n, h].double()
            k = dense(k_pages, table[b], n_kv, h // r)
            v = dense(v_pages, table[b], n_kv, h // r)
            s = (x @ k.T) * scale
            # what a row does not see is not part of its sums, whatever it holds
            s = torch.where(seen, s, -math.inf)
            top = s.amax(-1, keepdim=True)
            top = torch.where(top == -math.inf, 0.0, top)
            w = torch.exp(s - top)
            total = w.sum(-1, keepdim=True)
            some = total > 0
            w = w / torch.where(some, total, 1.0)
            clean = torch.where(torch.isfinite(v), v, 0.0)
            o = w @ clean
            bad = (seen & (w > 0)).double() @ (~torch.isfinite(v)).double() > 0
            o = torch.where(bad, math.nan, o)
            out[first:first + n, h] = o
            z = (top + torch.log(total))[:, 0]
            lse[first:first + n, h] = z
            mag = (x.abs() @ k.abs().T) * scale
            e = torch.where(seen, 130 * 2.0 ** -24 * mag + 2.0 ** -22 * s.abs(), 0.0)
            e = torch.nan_to_num(e.amax(-1, keepdim=True), posinf=0.0)
            spread = w @ clean.abs()
            t = spread * (unit + 2 * e + 2.0 ** -20 + n_kv * 2.0 ** -24) + unit_out * o.abs()
            if q.dtype == torch.float16:
                t = t + 2.0 ** -25 * n_kv * clean.abs().amax(0)
            tol[first:first + n, h] = t + 1e-30
            tol_lse[first:first + n, h] = (e[:, 0] + 2.0 ** -20 + n_kv * 2.0 ** -24
                                           + 2.0 ** -22 * torch.nan_to_num(z.abs(), posinf=0.0))
    return out, lse, tol, tol_lse
