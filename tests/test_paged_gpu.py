"""Paged KV cache on the GPU: step plan, row write and attention against the
plain forms of paged_ref.py (lists of integers; 64-bit arithmetic)."""

from __future__ import annotations

import math
import random

import pytest
import torch

import paged_ref

pytestmark = pytest.mark.gpu

D = 128


# -------------------------------------------------------------- step plan --

def run_step(tw, dev, lens, new, table, stack, count, *, page, cap):
    i32 = dict(dtype=torch.int32, device=dev)
    B = len(lens)
    t = torch.tensor(table, **i32)
    f = torch.tensor(stack, **i32)
    kv, cu = torch.full((B,), -7, **i32), torch.full((B + 1,), -7, **i32)
    slots = torch.full((cap,), -7, dtype=torch.int64, device=dev)
    pos = torch.full((cap,), -7, **i32)
    left, error = torch.full((1,), -7, **i32), torch.zeros(1, **i32)
    args = (torch.tensor(lens, **i32), torch.tensor(new, **i32), t, f,
            torch.tensor([count], **i32))
    kw = dict(page_size=page, kv_lens=kv, cu_q=cu, slots=slots, positions=pos,
              free_count_out=left, error_flag=error)
    tw.ops.paged_step(*args, **kw)
    once = [x.tolist() for x in (t, f, kv, cu, slots, pos)] + [left.item(), error.item()]
    tw.ops.paged_step(*args, **kw)  # the same inputs again: the same outputs
    again = [x.tolist() for x in (t, f, kv, cu, slots, pos)] + [left.item(), error.item()]
    assert once == again
    return tuple(once)


def make_step(rng, B, *, page, max_ctx, max_new, width_slack, finished, spare):
    lens = [rng.randint(0, max_ctx) for _ in range(B)]
    new = [rng.choice((0, 1, 1, rng.randint(0, max_new))) for _ in range(B)]
    for b in rng.sample(range(B), min(finished, B)):
        new[b] = -1 - rng.randint(0, 3)
    cdiv = lambda a: -(-a // page)  # noqa: E731
    width = max(1, max(cdiv(a + max(x, 0)) for a, x in zip(lens, new)) + width_slack,
                max(cdiv(a) for a in lens))
    held = sum(cdiv(a) for a in lens)
    num = held + spare
    ids = list(range(num))
    rng.shuffle(ids)
    table, at = [], 0
    for a in lens:
        n = cdiv(a)
        table.append(ids[at:at + n] + [-5] * (width - n))
        at += n
    stack = ids[held:] + [-1] * held
    return lens, new, table, stack, spare


@pytest.mark.parametrize("B,page,max_ctx,max_new,finished,spare,slack", [
    (1, 16, 0, 1, 0, 4, 0),          # a first token
    (1, 16, 40, 0, 1, 0, 0),         # one request, ended
    (3, 1, 9, 5, 1, 40, 0),          # pages of one row
    (16, 16, 300, 1, 0, 100, 2),     # decode
    (33, 8, 100, 200, 4, 1000, 0),
    (700, 24, 500, 60, 50, 3000, 0),  # more requests than threads of a block
    (64, 16, 200, 90, 8, 30, 0),     # the stack runs out
    (64, 16, 200, 90, 0, 0, 0),      # an empty stack
    (40, 16, 200, 90, 3, 400, -4),   # rows of the table run out
])
def test_step_matches_lists(tw, cuda, B, page, max_ctx, max_new, finished, spare, slack):
    for seed in range(3):
        rng = random.Random(1000 * B + seed)
        lens, new, table, stack, count = make_step(rng, B, page=page, max_ctx=max_ctx,
                                                   max_new=max_new, width_slack=slack,
                                                   finished=finished, spare=spare)
        total = sum(max(0, x) for x in new)
        for cap in {total, total + 5, max(0, total - 3)}:
            want = paged_ref.step(lens, new, table, stack, count, page=page, tokens_cap=cap,
                                  num_pages=len(stack))
            got = run_step(tw, cuda, lens, new, table, stack, count, page=page, cap=cap)
            names = ("table", "stack", "kv_lens", "cu_q", "slots", "positions", "count", "error")
            for name, w, g in zip(names, want, got):
                assert g == w, (seed, cap, name)


def test_step_flags_pages_outside_the_pool(tw, cuda):
    # request 0 continues on a page that is none, request 1 is given one from the stack
    got = run_step(tw, cuda, [3, 0], [1, 1], [[99, 0], [-1, -1]], [0, 77, -1, -1], 2, page=4, cap=2)
    assert got[4] == [-1, -1] and got[7] == tw._lib.TW_ERR_INVALID_INDEX
    assert got[2] == [4, 1] and got[6] == 1


def test_step_refusals(tw, cuda):
    i32 = dict(dtype=torch.int32, device=cuda)
    z = lambda *s: torch.zeros(s, **i32)  # noqa: E731
    good = dict(lens=z(2), new_lens=z(2), block_table=z(2, 3), free_pages=z(4), free_count=z(1))
    outs = dict(page_size=16, kv_lens=z(2), cu_q=z(3),
                slots=torch.zeros(4, dtype=torch.int64, device=cuda), positions=z(4),
                free_count_out=z(1))
    tw.ops.paged_step(*good.values(), **outs)
    for name, value in (("lens", z(2).long()), ("new_lens", z(3)), ("block_table", z(3, 3)),
                        ("block_table", z(3, 2).T), ("free_count", z(2)), ("lens", z(2).cpu())):
        with pytest.raises(ValueError):
            tw.ops.paged_step(*{**good, name: value}.values(), **outs)
    for name, value in (("page_size", 0), ("kv_lens", z(1)), ("cu_q", z(2)),
                        ("slots", z(4)), ("positions", z(3)), ("kv_lens", good["lens"]),
                        ("free_count_out", good["free_count"])):
        with pytest.raises(ValueError):
            tw.ops.paged_step(*good.values(), **{**outs, name: value})
    with pytest.raises(ValueError):  # more requests than one launch scans
        n = 8193
        tw.ops.paged_step(z(n), z(n), z(n, 1), z(4), z(1),
                          **{**outs, "kv_lens": z(n), "cu_q": z(n + 1)})


# -------------------------------------------------------------- row write --

def make_pool(pages, heads, page, dtype, dev, layout, fill=math.nan):
    if layout == "head":
        both = [torch.full((pages, heads, page, D), fill, dtype=dtype, device=dev)
                for _ in range(2)]
    elif layout == "token":
        both = [torch.full((pages, page, heads, D), fill, dtype=dtype, device=dev).transpose(1, 2)
                for _ in range(2)]
    else:  # K and V of a page side by side
        x = torch.full((pages, 2, heads, page, D), fill, dtype=dtype, device=dev)
        both = [x[:, 0], x[:, 1]]
    return both


def put(pages, table_row, rows):
    """rows [n, heads, D] as tokens 0 .. n of a request."""
    n, size = rows.shape[0], pages.shape[2]
    j = torch.arange(n, device=rows.device)
    pages[table_row[(j // size)].long(), :, j % size] = rows


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,heads,page,layout,fused", [
    (1, 1, 1, "head", False), (5, 8, 16, "head", True), (130, 3, 24, "token", False),
    (1000, 8, 64, "paired", True), (33, 2, 5, "token", True)])
def test_write_puts_rows(tw, cuda, dtype, T, heads, page, layout, fused):
    g = torch.Generator().manual_seed(T + heads)
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[T // 2] = -1
    x = torch.randn(T, 4 * heads, D, generator=g).to(dtype).to(cuda)
    k, v = x[:, -2 * heads:-heads], x[:, -heads:]
    if not fused:
        k, v = k.contiguous(), v.contiguous()
    kp, vp = make_pool(pages, heads, page, dtype, cuda, layout, fill=7.0)
    want_k, want_v = kp.clone(), vp.clone()
    for i, s in enumerate(slots.tolist()):
        if s >= 0:
            want_k[s // page, :, s % page] = k[i]
            want_v[s // page, :, s % page] = v[i]
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    tw.ops.paged_write(k, v, slots.to(cuda), kp, vp, error_flag=error)
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
    assert error.item() == 0


def test_write_flags_slots_outside_the_pool(tw, cuda):
    kp, vp = make_pool(2, 1, 4, torch.float16, cuda, "head", fill=0.0)
    rows = torch.ones(4, 1, D, dtype=torch.float16, device=cuda)
    error = torch.zeros(1, dtype=torch.int32, device=cuda)
    slots = torch.tensor([8, -2, 3, 1 << 40], device=cuda)
    tw.ops.paged_write(rows, rows, slots, kp, vp, error_flag=error)
    assert error.item() == tw._lib.TW_ERR_INVALID_INDEX
    assert kp.sum().item() == D and kp[0, 0, 3].sum().item() == D


def test_write_refusals(tw, cuda):
    kp, vp = make_pool(2, 2, 4, torch.float16, cuda, "head")
    rows = torch.zeros(3, 2, D, dtype=torch.float16, device=cuda)
    slots = torch.zeros(3, dtype=torch.int64, device=cuda)
    odd = torch.zeros(3 * 2 * D + 1, dtype=torch.float16, device=cuda)[1:].view(3, 2, D)
    for args in ((rows[:, :1], rows[:, :1], slots, kp, vp), (rows.bfloat16(), rows, slots, kp, vp),
                 (rows, rows, slots.int(), kp, vp), (rows, rows, slots[:2], kp, vp),
                 (odd, rows, slots, kp, vp), (rows, rows, slots, kp, vp[:1]),
                 (rows, rows, slots, kp.float(), vp.float()),
                 (rows, rows, slots, kp, vp.transpose(1, 2).contiguous().transpose(1, 2)),
                 (rows.cpu(), rows, slots, kp, vp)):
        with pytest.raises(ValueError):
            tw.ops.paged_write(*args)
    empty = torch.zeros(0, 2, D, dtype=torch.float16, device=cuda)
    tw.ops.paged_write(empty, empty, slots[:0], kp, vp)  # nothing to write is no error


# -------------------------------------------------------------- attention --

class Batch:
    """Requests with `new` tokens each, `kv` tokens in all, in a pool whose every
    other row holds NaN or infinity, behind a table whose other entries are no pages."""

    def __init__(self, dev, new, kv, *, q_heads, kv_heads, page, dtype, layout="head", seed=0,
                 q_scale=1.0, extra_pages=3):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        need = [-(-n // page) for n in kv]
        pages = sum(need) + extra_pages
        ids = torch.randperm(pages, generator=g).to(torch.int32).to(dev)
        self.k_pages, self.v_pages = make_pool(pages, kv_heads, page, dtype, dev, layout)
        self.v_pages[::2] = math.inf
        width = max(1, max(need)) + 2
        self.table = torch.full((len(kv), width), 2 ** 30, dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
            put(self.k_pages, self.table[b], r(kv[b], kv_heads, D).to(dtype).to(dev))
            put(self.v_pages, self.table[b], r(kv[b], kv_heads, D).to(dtype).to(dev))
        total = sum(new)
        self.q = (r(total, q_heads, D) * q_scale).to(dtype).to(dev)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        self.cu = torch.tensor(cu, dtype=torch.int32, device=dev)
        self.kv = torch.tensor(kv, dtype=torch.int32, device=dev)
        self.max_q, self.max_kv = max(new), max(kv)

    def run(self, tw, q=None, **kw):
        q = self.q if q is None else q
        error = torch.zeros(1, dtype=torch.int32, device=q.device)
        lse = torch.full(q.shape[:2], math.nan, device=q.device)
        out = tw.ops.paged_attention(q, self.k_pages, self.v_pages, self.table, self.cu, self.kv,
                                     max_q_len=kw.pop("max_q_len", self.max_q),
                                     max_kv_len=kw.pop("max_kv_len", self.max_kv), lse=lse,
                                     error_flag=error, **kw)
        return out, lse, error.item()

    def check(self, out, lse, *, window=0, scale=None):
        ref, ref_lse, tol, tol_lse = paged_ref.attention(
            self.q, self.k_pages, self.v_pages, self.table, self.cu, self.kv, window=window,
            scale=scale, out_dtype=out.dtype)
        bad = (out.double() - ref).abs() > tol
        # NaN in the reference has to be NaN or infinite here, and nothing else may be
        fine = torch.isfinite(ref)
        assert bool((torch.isfinite(out.double()) == fine).all()), "finite where it should not be"
        worst = ((out.double() - ref).abs() / tol)[fine]
        assert not bool(bad[fine].any()), f"{float(worst.max()):.3f} of the tolerance"
        empty = ref_lse == -math.inf
        assert bool((lse[empty] == -math.inf).all()) and bool((out[empty] == 0).all())
        known = torch.isfinite(ref_lse)
        assert bool(((lse.double() - ref_lse).abs() <= tol_lse)[known].all())


HEADS = [(8, 8), (8, 2), (6, 2), (14, 2), (16, 1)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page,layout", [(16, "head"), (8, "token"), (24, "paired"), (256, "head")])
def test_single_tokens(tw, cuda, dtype, heads, page, layout):
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 700]
    b = Batch(cuda, [1] * len(kv), kv, q_heads=heads[0], kv_heads=heads[1], page=page,
              dtype=dtype, layout=layout, seed=page)
    out, lse, error = b.run(tw)
    assert error == 0
    b.check(out, lse)


@pytest.mark.parametrize("heads", HEADS + [(64, 1)])
@pytest.mark.parametrize("page,layout", [(16, "head"), (8, "token"), (40, "paired"), (128, "token")])
def test_chunks(tw, cuda, heads, page, layout):
    new = [1, 2, 5, 16, 17, 33, 64, 100, 129, 257]
    kv = [1, 40, 5, 130, 17, 500, 64, 227, 129, 700]
    b = Batch(cuda, new, kv, q_heads=heads[0], kv_heads=heads[1], page=page,
              dtype=torch.bfloat16, layout=layout, seed=page)
    out, lse, error = b.run(tw)
    assert error == 0
    b.check(out, lse)


@pytest.mark.parametrize("window", [1, 7, 16, 100, 128, 129, 5000])
@pytest.mark.parametrize("new,kv", [([1, 1, 1], [1, 90, 900]), ([40, 300, 1], [40, 700, 350])])
def test_window(tw, cuda, window, new, kv):
    b = Batch(cuda, new, kv, q_heads=8, kv_heads=2, page=16, dtype=torch.float16, seed=window)
    out, lse, error = b.run(tw, window=window)
    assert error == 0
    b.check(out, lse, window=window)


@pytest.mark.parametrize("page", [8, 16, 128])
def test_pages_before_the_window_may_be_gone(tw, cuda, page):
    new, kv, window = [1, 1, 40], [900, 300, 640], 100
    b = Batch(cuda, new, kv, q_heads=8, kv_heads=2, page=page, dtype=torch.bfloat16)
    whole, lse, _ = b.run(tw, window=window)
    b.check(whole, lse, window=window)
    for r in range(3):
        b.table[r, :(kv[r] - new[r] - window + 1) // page] = -1
    out, again, error = b.run(tw, window=window)
    assert error == 0 and torch.equal(out, whole) and torch.equal(again, lse)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("new,kv", [([1], [5000]), ([3], [5003]), ([200], [3200]), ([8], [2048])])
def test_long_contexts_with_few_rows(tw, cuda, out_dtype, new, kv):
    """Few rows and many keys: the work is split over the keys and joined."""
    b = Batch(cuda, new, kv, q_heads=8, kv_heads=2, page=16, dtype=torch.bfloat16, seed=kv[0],
              q_scale=3.0)
    out, lse, error = b.run(tw, out_dtype=out_dtype)
    assert error == 0 and out.dtype == out_dtype
    b.check(out, lse)


@pytest.mark.parametrize("scale", [1.0, 0.02])
def test_scale_and_growing_scores(tw, cuda, scale):
    """Scores that grow along the keys (the running maximum moves again and again)."""
    b = Batch(cuda, [1, 150], [900, 900], q_heads=8, kv_heads=2, page=16, dtype=torch.float16)
    for r in range(2):
        ramp = torch.linspace(0.05, 4.0, 900, device=cuda)[:, None, None]
        put(b.k_pages, b.table[r], (b.q[r][:2].float()[None] * ramp / 8).to(torch.float16))
    out, lse, error = b.run(tw, softmax_scale=scale)
    assert error == 0
    b.check(out, lse, scale=scale)


@pytest.mark.parametrize("new,kv", [([5, 1, 3], [3, 0, 0]), ([200, 40], [70, 0]),
                                    ([0, 4, 0], [9, 4, 0]), ([0], [5])])
def test_rows_that_see_nothing(tw, cuda, new, kv):
    b = Batch(cuda, new, kv, q_heads=8, kv_heads=2, page=16, dtype=torch.bfloat16)
    out, lse, error = b.run(tw)
    assert error == 0
    b.check(out, lse)


@pytest.mark.parametrize("new,kv", [([1, 1], [30, 300]), ([90, 20], [90, 200])])
def test_padding_rows(tw, cuda, new, kv):
    b = Batch(cuda, new, kv, q_heads=8, kv_heads=2, page=16, dtype=torch.bfloat16)
    real = b.q.shape[0]
    b.q = torch.cat((b.q, torch.full((77, 8, D), math.nan, dtype=b.q.dtype, device=cuda)))
    out, lse, error = b.run(tw)
    assert error == 0
    assert bool((out[real:] == 0).all()) and bool((lse[real:] == -math.inf).all())
    b.q, out, lse = b.q[:real], out[:real], lse[:real]
    b.check(out, lse)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("window", [0, 60])
def test_values_that_a_row_does_not_see_stay_out(tw, cuda, value, where, window):
    """A later token of the same chunk, or one before the window, that is not finite."""
    new, kv = [100, 3, 1], [190, 64, 120]
    b = Batch(cuda, new, kv, q_heads=8, kv_heads=2, page=16, dtype=torch.bfloat16, seed=3)
    pages = b.k_pages if where == "k" else b.v_pages
    for r, j in ((0, 150), (1, 62), (2, 20), (0, 93)):
        pages[b.table[r, j // 16].long(), :, j % 16, 5:7] = value
    if where == "k":  # a row that sees the key has a score of NaN or infinity
        b.q[..., 5:7] = 1.0
    out, lse, error = b.run(tw, window=window)
    assert error == 0
    if where == "v":
        b.check(out, lse, window=window)
        return
    # rows that do not see those keys are those of the clean cache
    for r, j in ((0, 150), (1, 62), (2, 20), (0, 93)):
        pages[b.table[r, j // 16].long(), :, j % 16, 5:7] = 0.0
    ref, _, tol, _ = paged_ref.attention(b.q, b.k_pages, b.v_pages, b.table, b.cu, b.kv,
                                         window=window)
    for r, keys in ((0, (150, 93)), (1, (62,)), (2, (20,))):
        p = kv[r] - new[r] + torch.arange(new[r], device=cuda)
        blind = torch.ones_like(p, dtype=torch.bool)
        for j in keys:
            blind &= (p < j) | ((p - window >= j) if window else torch.zeros_like(blind))
        rows = int(b.cu[r]) + torch.arange(new[r], device=cuda)[blind]
        assert bool(((out[rows].double() - ref[rows]).abs() <= tol[rows]).all())


@pytest.mark.parametrize("where", ["q", "k", "v"])
def test_values_that_a_row_sees_reach_it(tw, cuda, where):
    """NaN in what a row attends with is NaN in its result, and in no other row's."""
    b = Batch(cuda, [90, 1, 2], [200, 70, 40], q_heads=8, kv_heads=2, page=16,
              dtype=torch.float16)
    if where == "q":
        b.q[30, 3, 7] = math.nan
    else:
        pages = b.k_pages if where == "k" else b.v_pages
        pages[b.table[0, 150 // 16].long(), 0, 150 % 16, 3] = math.nan
        pages[b.table[1, 0].long(), :, 5] = math.nan
    out, lse, error = b.run(tw)
    assert error == 0
    bad = torch.isnan(out).any(-1)
    want = torch.zeros_like(bad)
    if where == "q":
        want[30, 3] = True
    else:
        want[40:90, :4] = True  # positions 150 .. 199, the four heads of KV head 0
        want[90] = True
    assert torch.equal(bad, want)


def test_requests_longer_than_max_q_len_are_flagged(tw, cuda):
    for new, most in (([3, 1], 1), ([100, 60], 60)):
        b = Batch(cuda, new, [150, 150], q_heads=8, kv_heads=2, page=16, dtype=torch.float16)
        good, _, _ = b.run(tw)
        out, _, error = b.run(tw, max_q_len=most)
        assert error == tw._lib.TW_ERR_BAD_ARG
        assert torch.equal(out[new[0]:], good[new[0]:])


@pytest.mark.parametrize("requests", [33, 150, 1500])
def test_many_requests(tw, cuda, requests):
    rng = random.Random(requests)
    new = [rng.choice((0, 1, 1, 1, 3, rng.randint(10, 70))) for _ in range(requests)]
    kv = [n + rng.randint(0, 60) for n in new]
    b = Batch(cuda, new, kv, q_heads=6, kv_heads=1, page=16, dtype=torch.bfloat16, seed=requests)
    out, lse, error = b.run(tw)
    assert error == 0
    ref = torch.empty_like(out)
    for r in range(requests):  # each request alone
        first, n = int(b.cu[r]), new[r]
        if n:
            ref[first:first + n] = tw.ops.paged_attention(
                b.q[first:first + n], b.k_pages, b.v_pages, b.table[r:r + 1],
                torch.tensor([0, n], dtype=torch.int32, device=cuda), b.kv[r:r + 1], max_q_len=n,
                max_kv_len=kv[r])
    # one kernel or the other, one range or several: the same within both roundings
    assert (out.float() - ref.float()).abs().max().item() <= 4 * 2.0 ** -8 * ref.abs().max().item()
    for r in rng.sample(range(requests), 10):
        first, n = int(b.cu[r]), new[r]
        if n == 0:
            continue
        o, z, tol, _ = paged_ref.attention(
            b.q[first:first + n], b.k_pages, b.v_pages, b.table[r:r + 1],
            torch.tensor([0, n], device=cuda), b.kv[r:r + 1])
        assert bool(((out[first:first + n].double() - o).abs() <= tol).all())


@pytest.mark.parametrize("most", [0, 1, 10 ** 6, 2 ** 31 - 1])
def test_max_kv_len_only_sizes_the_launch(tw, cuda, most):
    b = Batch(cuda, [1, 50], [3000, 700], q_heads=8, kv_heads=2, page=16, dtype=torch.bfloat16)
    out, lse, error = b.run(tw, max_kv_len=most)
    assert error == 0
    b.check(out, lse)


def test_strided_rows_and_another_stream(tw, cuda):
    b = Batch(cuda, [1, 70], [33, 170], q_heads=8, kv_heads=2, page=16, dtype=torch.float16)
    T = b.q.shape[0]
    wide = torch.full((T, 12, D), math.nan, dtype=torch.float16, device=cuda)
    wide[:, 2:10] = b.q
    out = torch.full((T, 20, D), 5.0, dtype=torch.float16, device=cuda)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        view, lse, error = b.run(tw, q=wide[:, 2:10], out=out[:, ::2][:, 1:9])
    torch.cuda.current_stream().wait_stream(stream)
    assert error == 0
    b.check(view, lse)
    assert bool((out[:, 1::2] == 5.0).all()) and bool((out[:, 0] == 5.0).all())
    assert bool((out[:, 18] == 5.0).all())


def test_same_bits_every_time(tw, cuda):
    b = Batch(cuda, [1, 1, 130], [3000, 70, 900], q_heads=8, kv_heads=2, page=16,
              dtype=torch.bfloat16)
    first = b.run(tw)
    for _ in range(5):
        out, lse, _ = b.run(tw)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


def test_graph_replay_follows_the_lengths(tw, cuda):
    """A captured step reads tables and lengths at replay."""
    b = Batch(cuda, [1, 1], [200, 300], q_heads=8, kv_heads=2, page=16, dtype=torch.bfloat16)
    out = torch.empty_like(b.q)
    lse = torch.empty(b.q.shape[:2], device=cuda)
    need = tw.ops.paged_attention_workspace_bytes(2, 2, 8, 2, 1, 300)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=cuda)
    call = lambda: tw.ops.paged_attention(b.q, b.k_pages, b.v_pages, b.table, b.cu, b.kv,  # noqa: E731
                                          max_q_len=1, max_kv_len=300, out=out, lse=lse,
                                          workspace=ws)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    b.kv.copy_(torch.tensor([100, 17], dtype=torch.int32))
    b.q.normal_()
    graph.replay()
    torch.cuda.synchronize()
    b.check(out, lse)


@pytest.mark.parametrize("new,kv", [([1, 1], [100, 100]), ([100, 60], [100, 100])])
def test_bad_pages_and_lengths_are_flagged(tw, cuda, new, kv):
    L = tw._lib
    b = Batch(cuda, new, kv, q_heads=8, kv_heads=2, page=16, dtype=torch.float16)
    good, _, _ = b.run(tw)
    for bad in (-1, 2 ** 30, b.k_pages.shape[0]):
        b.table[0, 2], keep = bad, b.table[0, 2].clone()
        out, _, error = b.run(tw)
        assert error == L.TW_ERR_INVALID_INDEX
        assert torch.equal(out[new[0]:], good[new[0]:])  # the other request is served
        b.table[0, 2] = keep
    # longer than the table: cut, flagged
    b.table = b.table[:, :7].contiguous()
    b.kv[0] = 2000
    out, _, error = b.run(tw)
    assert error == L.TW_ERR_INVALID_INDEX and torch.equal(out[new[0]:], good[new[0]:])


def test_pool_beyond_32_bit_offsets(tw, cuda):
    """Pages whose rows lie more than 2^32 elements into the pool."""
    page, heads, pages = 64, 8, 70000  # 4.6e9 elements, 9.2 GB for K and V together in one
    x = torch.empty(pages, heads, page, D, dtype=torch.bfloat16, device=cuda)
    g = torch.Generator().manual_seed(9)
    new, kv = [1, 90], [200, 300]
    table = torch.randperm(2000, generator=g)[:10].to(torch.int32).to(cuda).view(2, 5) + 68000
    b = Batch(cuda, new, [1, 1], q_heads=32, kv_heads=heads, page=page, dtype=torch.bfloat16)
    b.k_pages, b.v_pages, b.table = x, x, table
    b.q = torch.randn(91, 32, D, generator=g).to(torch.bfloat16).to(cuda)
    b.cu = torch.tensor([0, 1, 91], dtype=torch.int32, device=cuda)
    b.kv = torch.tensor(kv, dtype=torch.int32, device=cuda)
    rows = torch.randn(500, heads, D, generator=g).to(torch.bfloat16).to(cuda)
    slots = torch.cat([table[r, torch.arange(n, device=cuda) // page].long() * page
                       + torch.arange(n, device=cuda) % page for r, n in enumerate(kv)])
    assert int(slots.max()) * heads * D > 2 ** 32
    tw.ops.paged_write(rows, rows, slots, x, x)
    for r, n in enumerate(kv):
        j = torch.arange(n, device=cuda)
        first = 0 if r == 0 else kv[0]
        assert torch.equal(x[table[r, j // page].long(), :, j % page], rows[first:first + n])
    out, lse, error = b.run(tw, max_q_len=90, max_kv_len=300)
    assert error == 0
    b.check(out, lse)


@pytest.mark.parametrize("new,kv", [([1], [5000]), ([200], [4000])])
def test_workspace(tw, cuda, new, kv):
    """A workspace that the caller brings: as large as asked for, whatever it holds."""
    b = Batch(cuda, new, kv, q_heads=8, kv_heads=2, page=16, dtype=torch.bfloat16)
    need = tw.ops.paged_attention_workspace_bytes(1, new[0], 8, 2, new[0], kv[0])
    assert need > 0
    out, lse, _ = b.run(tw)
    for fill in (0, 255):
        ws = torch.full((need,), fill, dtype=torch.uint8, device=cuda)
        again, _, error = b.run(tw, workspace=ws)
        assert error == 0 and torch.equal(again, out)
    with pytest.raises(RuntimeError, match="capacity"):
        b.run(tw, workspace=ws[:need - 1])
    with pytest.raises(ValueError):
        b.run(tw, workspace=torch.empty(need + 4, dtype=torch.uint8, device=cuda)[4:])
    with pytest.raises(ValueError):
        b.run(tw, workspace=torch.empty(need, dtype=torch.uint8))


def test_attention_refusals(tw, cuda):
    b = Batch(cuda, [2, 1], [20, 30], q_heads=8, kv_heads=2, page=16, dtype=torch.float16)
    args = dict(q=b.q, k_pages=b.k_pages, v_pages=b.v_pages, block_table=b.table, cu_q=b.cu,
                kv_lens=b.kv, max_q_len=2, max_kv_len=30)
    tw.ops.paged_attention(**args)
    odd = torch.zeros(3 * 8 * D + 1, dtype=torch.float16, device=cuda)[1:].view(3, 8, D)
    bad = [dict(q=b.q.bfloat16()), dict(q=b.q[:, :7]), dict(q=odd), dict(q=b.q[..., :64]),
           dict(q=b.q.cpu()), dict(cu_q=b.cu.long()), dict(cu_q=b.cu[:2]),
           dict(kv_lens=b.kv.cpu()), dict(block_table=b.table[:1]),
           dict(block_table=b.table.T.contiguous().T), dict(out=torch.empty_like(b.q[:2])),
           dict(out_dtype=torch.bfloat16), dict(out=b.q.double()),
           dict(lse=torch.empty(8, 3, device=cuda)), dict(window=-1), dict(softmax_scale=0.0),
           dict(softmax_scale=-1.0), dict(softmax_scale=math.nan), dict(max_q_len=-1),
           dict(max_kv_len=-1), dict(k_pages=b.k_pages[:, :, :12], v_pages=b.v_pages[:, :, :12]),
           dict(k_pages=b.k_pages.float(), v_pages=b.v_pages.float()),
           dict(k_pages=b.k_pages[..., :64], v_pages=b.v_pages[..., :64])]
    for change in bad:
        with pytest.raises(ValueError):
            tw.ops.paged_attention(**{**args, **change})
    with pytest.raises(ValueError):  # 65 query heads per KV head
        many = torch.zeros(3, 130, D, dtype=torch.float16, device=cuda)
        tw.ops.paged_attention(**{**args, "q": many})
    empty = tw.ops.paged_attention(**{**args, "q": b.q[:0]})
    assert empty.shape == (0, 8, D)
