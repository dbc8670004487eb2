"""Eviction against the ranking written over Python lists: rows that stay, where they go,
lengths, offsets and pages."""

from __future__ import annotations

import random

import pytest
import torch

import evict_ref

pytestmark = pytest.mark.gpu

D = 128


def state(dev, seed, lens, *, layers=1, heads=2, page=16, dtype=torch.float16, gone=None,
          pool="head", ties=0.3, extra=3):
    """A cache in random order: pools, records, table, stack."""
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    held = [-(-n // page) for n in lens]
    pages = sum(held) + extra
    ids = list(range(pages))
    rng.shuffle(ids)
    width = max(held + [1]) + 1
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    stack = torch.full((pages,), -1, dtype=torch.int32)
    stack[:pages - at] = torch.tensor(ids[at:], dtype=torch.int32)
    shape = (layers, pages, heads, page) if pool == "head" else (layers, pages, page, heads)
    turn = (lambda t: t) if pool == "head" else (lambda t: t.transpose(2, 3))
    kv = [turn(torch.randn(*shape, D, generator=g).to(dtype).to(dev)) for _ in range(2)]
    w = torch.exp(2 * torch.randn(layers, pages, heads, page, generator=g))
    w[torch.rand(w.shape, generator=g) < ties] = 0.25  # many that are equal
    gone = [0] * len(lens) if gone is None else gone
    p = torch.zeros(layers, pages, heads, page, dtype=torch.int32)
    for b, n in enumerate(lens):
        j = torch.arange(n)
        for l in range(layers):
            for h in range(heads):
                spots = torch.randperm(n + gone[b], generator=g)[:n]
                p[l, table[b, j // page].long(), h, j % page] = spots.int()
    i32 = dict(dtype=torch.int32, device=dev)
    return dict(k=kv[0], v=kv[1], w=w.to(dev), p=p.to(dev), table=table.to(dev),
                stack=stack.to(dev), count=torch.tensor([pages - at], **i32),
                lens=torch.tensor(lens, **i32), gone=torch.tensor(gone, **i32), page=page,
                err=torch.zeros(1, **i32), layers=layers)


def call(tw, s, keep, sink, recent, *, max_len=None, flat=None, stack=True):
    n = s["lens"].numel()
    i32 = dict(dtype=torch.int32, device=s["lens"].device)
    lens_out, gone_out, left = (torch.full((m,), -9, **i32) for m in (n, n, 1))
    flat = s["layers"] == 1 if flat is None else flat
    pick = (lambda t: t[0]) if flat else (lambda t: t)
    tw.ops.paged_evict(pick(s["k"]), pick(s["v"]), pick(s["w"]), pick(s["p"]), s["table"],
                       s["lens"], torch.tensor(keep, **i32), s["gone"],
                       max_len=int(s["lens"].max()) if max_len is None else max_len, sink=sink,
                       recent=recent, lens_out=lens_out, offsets_out=gone_out,
                       error_flag=s["err"],
                       **(dict(free_pages=s["stack"], free_count=s["count"], free_count_out=left)
                          if stack else {}))
    return lens_out, gone_out, left


def check(tw, s, keep, sink, recent, **kw):
    """The call against the lists, on copies; every place that is not named stays."""
    cpu = {n: s[n].cpu().clone() for n in ("k", "v", "w", "p", "stack")}
    table = s["table"].tolist()
    count = int(s["count"])
    table_before = s["table"].clone()
    lens_out, gone_out, left = call(tw, s, keep, sink, recent, **kw)
    want_lens, want_gone, back = evict_ref.evict(
        (cpu["k"], cpu["v"]), cpu["w"], cpu["p"], table, s["lens"].tolist(), keep,
        s["gone"].tolist(), sink=sink, recent=recent, page=s["page"])
    assert lens_out.tolist() == want_lens
    assert gone_out.tolist() == want_gone
    cpu["stack"][count:count + len(back)] = torch.tensor(back, dtype=torch.int32)
    assert torch.equal(s["stack"].cpu(), cpu["stack"])
    assert int(left) == count + len(back)
    for n in ("p", "w", "k", "v"):
        a, b = s[n].cpu(), cpu[n]
        if n != "p":  # (NaN equals itself here)
            kind = torch.int32 if n == "w" else torch.int16
            a, b = a.contiguous().view(kind), b.contiguous().view(kind)
        assert torch.equal(a, b), n
    assert torch.equal(s["table"], table_before)
    assert int(s["err"]) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pool", ["head", "token"])
@pytest.mark.parametrize("page", [8, 16, 24, 64])
def test_small(tw, cuda, dtype, pool, page):
    rng = random.Random(page)
    for seed in range(3):
        lens = [0, 1, page, page + 1, 3 * page, 100, 333]
        keep = [rng.randint(0, n + 2) for n in lens]
        keep[-2] = -1
        s = state(cuda, seed, lens, page=page, dtype=dtype, pool=pool,
                  gone=[rng.choice((0, 500)) for _ in lens])
        check(tw, s, keep, rng.choice((0, 3)), rng.choice((0, 1, 20)))


@pytest.mark.parametrize("n,keep", [(2048, 2047), (2049, 1), (4097, 2000), (4160, 4096),
                                    (9000, 6500), (17001, 16000), (20011, 5)])
def test_cluster_sizes(tw, cuda, n, keep):
    """One CTA, two, four, eight a cluster; segments that end inside a word of rows."""
    s = state(cuda, n, [n, 70], heads=1, page=16, gone=[n // 3, 0])
    check(tw, s, [keep, 50], 4, min(64, keep))


def test_layers(tw, cuda):
    s = state(cuda, 9, [300, 40, 513], layers=3, heads=3, page=16, gone=[0, 7, 1000])
    check(tw, s, [100, 39, 64], 4, 32)
    s = state(cuda, 10, [300], layers=1, heads=2)
    check(tw, s, [100], 4, 32, flat=False)  # a leading dimension of one layer


@pytest.mark.parametrize("fill", [0.0, -0.0, float("nan"), float("inf"), -1.0, 1e-42])
def test_equal_weights(tw, cuda, fill):
    """All the same: the first rows stay and nothing moves.  Among a few larger ones: those,
    then the first."""
    s = state(cuda, 3, [5000], heads=2)
    s["w"].fill_(fill)
    before = s["k"].clone()
    s["p"].fill_(10)
    s["gone"].fill_(100000)
    check(tw, s, [3000], 0, 0)
    assert torch.equal(before, s["k"])
    s = state(cuda, 4, [5000], heads=2, ties=0.0)
    s["w"][:, ::3] = fill
    check(tw, s, [3000], 0, 0)


def test_ranking_of_values(tw, cuda):
    """NaN above infinity above numbers, -0 like 0, negative ones last; the protected rows
    above all."""
    s = state(cuda, 6, [64], heads=1, page=16, ties=0.0)
    values = [float("nan"), float("inf"), 1e30, 1.0, 1e-44, 0.0, -0.0, -1e-44, -1.0, -float("inf")]
    flat = torch.tensor([values[i % 10] for i in range(64)])
    j = torch.arange(64)
    s["w"][0, s["table"][0, j // 16].long().cpu(), 0, j % 16] = flat.to(cuda)
    for keep in (1, 7, 8, 20, 35, 45, 60, 63):
        t = {n: (x.clone() if isinstance(x, torch.Tensor) else x) for n, x in s.items()}
        check(tw, t, [keep], 0, 1)


def test_all_rows_protected(tw, cuda):
    """More protected rows than places: the first of them stay."""
    s = state(cuda, 8, [400], heads=2)
    check(tw, s, [100], 200, 300)
    s = state(cuda, 8, [400], heads=2)
    check(tw, s, [0], 4, 4)


def test_repeated_and_grown(tw, cuda):
    """Cut, grown and cut again, as a decoding loop does: positions stay those of the rows."""
    s = state(cuda, 12, [130], heads=2, ties=0.1, page=16, extra=4)
    for turn in range(3):
        check(tw, s, [96], 4, 16)
        s["lens"], s["gone"] = torch.tensor([96], dtype=torch.int32, device=cuda), s["gone"] + (
            s["lens"] - 96)
        # 34 more rows (the pages past the end are still in the table)
        j = torch.arange(96, 130, device=cuda)
        at = s["table"][0, j // 16].long()
        s["w"][:, at, :, j % 16] = torch.rand(34, 1, 2, device=cuda)
        s["p"][:, at, :, j % 16] = (j + s["gone"]).int()[:, None, None]
        s["lens"] = torch.tensor([130], dtype=torch.int32, device=cuda)
        s["count"].zero_()
        places = s["p"][0, s["table"][0, torch.arange(130) // 16].long(), 0, torch.arange(130) % 16]
        assert len(set(places.tolist())) == 130


def test_no_stack(tw, cuda):
    s = state(cuda, 13, [200, 100])
    stack = s["stack"].clone()
    lens, gone, _ = call(tw, s, [50, 100], 0, 8, stack=False)
    assert lens.tolist() == [50, 100] and gone.tolist() == [150, 0]
    assert torch.equal(stack, s["stack"])


def test_many_requests(tw, cuda):
    """Requests past a warp's and a CTA's first look, few of which are cut."""
    rng = random.Random(2)
    lens = [rng.choice((0, 1, 5, 17, 40)) for _ in range(1500)]
    keep = [rng.choice((-1, 50, 50, 50, n // 2)) for n in lens]
    s = state(cuda, 14, lens, heads=1, page=8)
    check(tw, s, keep, 1, 2)


def test_flags(tw, cuda):
    """Requests that are longer than max_len or their table row are left as they are; a page
    outside the pool is flagged and its rows do not move; a stack that is full is flagged."""
    L = tw._lib
    s = state(cuda, 15, [100, 40])
    k = s["k"].clone()
    lens, gone, left = call(tw, s, [50, 50], 0, 0, max_len=99)
    assert int(s["err"]) == L.TW_ERR_BAD_ARG
    assert lens.tolist() == [100, 40] and gone.tolist() == [0, 0] and torch.equal(k, s["k"])
    assert int(left) == int(s["count"])
    s = state(cuda, 16, [100, 40])
    s["lens"][0] = 5000
    k = s["k"].clone()
    lens, _, _ = call(tw, s, [50, 30], 0, 0, max_len=6000)
    assert int(s["err"]) == L.TW_ERR_INVALID_INDEX
    assert lens.tolist() == [5000, 30]
    s = state(cuda, 17, [100], heads=1)
    for bad in (-1, s["stack"].numel(), 1 << 30):
        t = {n: (x.clone() if isinstance(x, torch.Tensor) else x) for n, x in s.items()}
        page = int(t["table"][0, 5])
        t["table"][0, 5] = bad
        before = t["k"].clone()
        lens, _, _ = call(tw, t, [60], 0, 0)
        assert int(t["err"]) == L.TW_ERR_INVALID_INDEX and lens.tolist() == [60]
        assert torch.equal(t["k"][:, page], before[:, page])
    s = state(cuda, 18, [100])
    s["count"].fill_(s["stack"].numel())
    call(tw, s, [10], 0, 0)
    assert int(s["err"]) == L.TW_ERR_CAPACITY


def test_refusals(tw, cuda):
    s = state(cuda, 19, [100], layers=2)
    i32 = dict(dtype=torch.int32, device=cuda)
    good = dict(k_pages=s["k"], v_pages=s["v"], row_weights=s["w"], row_positions=s["p"],
                block_table=s["table"], lens=s["lens"], keep=torch.full((1,), 50, **i32),
                offsets=s["gone"], max_len=100, sink=0, recent=0,
                lens_out=torch.zeros(1, **i32), offsets_out=torch.zeros(1, **i32))
    for bad in (dict(k_pages=s["k"][0]), dict(v_pages=s["v"][:1]), dict(row_weights=s["w"].int()),
                dict(row_positions=s["p"][:, :1]), dict(row_weights=None), dict(sink=-1),
                dict(recent=-1), dict(max_len=-1), dict(lens_out=s["lens"]),
                dict(offsets_out=s["gone"]), dict(free_pages=s["stack"]),
                dict(keep=torch.zeros(2, **i32)), dict(block_table=s["table"].long()),
                dict(k_pages=s["k"].float(), v_pages=s["v"].float()),
                dict(row_weights=s["w"].expand(2, *s["w"].shape[1:]).flip(0)[:, :, :1])):
        with pytest.raises(ValueError):
            tw.ops.paged_evict(**{**good, **bad})
    tw.ops.paged_evict(**good)


def test_graph_and_stream(tw, cuda):
    """Captured once, replayed on other records; and on another stream."""
    a, b = (state(cuda, seed, [700, 90], heads=2) for seed in (20, 21))
    b["table"], b["stack"] = a["table"].clone(), a["stack"].clone()
    want = {n: (x.clone() if isinstance(x, torch.Tensor) else x) for n, x in b.items()}
    args = ([256, 90], 4, 32)
    i32 = dict(dtype=torch.int32, device=cuda)
    keep, lens_out, gone_out, left = (torch.tensor(args[0], **i32), torch.zeros(2, **i32),
                                      torch.zeros(2, **i32), torch.zeros(1, **i32))
    run = lambda s: tw.ops.paged_evict(  # noqa: E731
        s["k"][0], s["v"][0], s["w"][0], s["p"][0], s["table"], s["lens"], keep, s["gone"],
        max_len=700, sink=4, recent=32, lens_out=lens_out, offsets_out=gone_out,
        free_pages=s["stack"], free_count=s["count"], free_count_out=left, error_flag=s["err"])
    run({n: (x.clone() if isinstance(x, torch.Tensor) else x) for n, x in a.items()})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(a)
    for n in ("k", "v", "w", "p"):
        a[n].copy_(b[n])
    graph.replay()
    torch.cuda.synchronize()
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        run(want)
    side.synchronize()
    for n in ("k", "v", "w", "p", "stack"):
        assert torch.equal(a[n], want[n]), n


@pytest.mark.parametrize("n,keep,max_len", [(400_003, 399_700, None), (700_001, 350_000, None),
                                            (90_001, 60_000, 1 << 21), (5000, 2500, 1 << 21)])
def test_long_requests(tw, cuda, n, keep, max_len):
    """Keys that shared memory does not hold, lists that take several turns, a bound far above
    the lengths: against a stable sort."""
    page = 64
    g = torch.Generator(cuda).manual_seed(n)
    pages = -(-n // page) + 2
    i32 = dict(dtype=torch.int32, device=cuda)
    table = torch.randperm(pages, generator=g, device=cuda)[:-2].to(torch.int32)[None].contiguous()
    k, v = (torch.randint(-30000, 30000, (pages, 1, page, D), generator=g, device=cuda,
                          dtype=torch.int16) for _ in range(2))
    w = torch.rand(pages, 1, page, generator=g, device=cuda)
    w[torch.rand(w.shape, generator=g, device=cuda) < 0.2] = 0.5
    p = torch.randint(0, 2 * n, (pages, 1, page), generator=g, device=cuda, dtype=torch.int32)
    j = torch.arange(n, device=cuda)
    at = table[0, j // page].long(), torch.zeros_like(j), j % page
    fixed = (p[at] < 50) | (p[at] >= 2 * n - 100)
    order = torch.where(fixed, 2.0, w[at].double()).sort(descending=True, stable=True).indices
    stays = torch.zeros(n, dtype=torch.bool, device=cuda)
    stays[order[:keep]] = True
    to, source = torch.nonzero(~stays[:keep])[:, 0], torch.nonzero(stays[keep:])[:, 0] + keep
    spot = lambda x: (table[0, x // page].long(), torch.zeros_like(x), x % page)  # noqa: E731
    want = [t.clone() for t in (k, v, w, p)]
    for t in want:
        t[spot(to)] = t[spot(source)]
    lens_out, gone_out = torch.zeros(1, **i32), torch.zeros(1, **i32)
    err = torch.zeros(1, **i32)
    tw.ops.paged_evict(k.view(torch.float16), v.view(torch.float16), w, p, table,
                       torch.tensor([n], **i32), torch.tensor([keep], **i32),
                       torch.tensor([n], **i32), max_len=n if max_len is None else max_len, sink=50,
                       recent=100, lens_out=lens_out, offsets_out=gone_out, error_flag=err)
    assert int(err) == 0 and int(lens_out) == keep and int(gone_out) == 2 * n - keep
    for got, t in zip((k, v, w, p), want):
        assert torch.equal(got, t)


def test_far_pages(tw, cuda):
    """Places beyond 2^31 elements of a pool: written, weighed and moved there."""
    heads, page, pages = 8, 16, 140_000  # 2.3e9 elements
    g = torch.Generator().manual_seed(1)
    i32 = dict(dtype=torch.int32, device=cuda)
    k, v = (torch.zeros(pages, heads, page, D, dtype=torch.float16, device=cuda) for _ in range(2))
    w = torch.zeros(pages, heads, page, device=cuda)
    p = torch.zeros(pages, heads, page, **i32)
    ids = torch.tensor([pages - 1, 3, pages - 7, pages - 2], **i32)
    table = ids[None].contiguous()
    rows = torch.randn(60, 2 * heads, D, generator=g).to(torch.float16).to(cuda)
    kk, vv = rows[:, :heads], rows[:, heads:]
    j = torch.arange(60, device=cuda)
    slots = table[0, j // page].long() * page + j % page
    f, _ = tw.ops.rope_frequencies(128, device=cuda)
    q = tw.ops.paged_rope_write(kk, kk, vv, j.int(), slots, f, k, v, row_weights=w,
                                row_positions=p)
    at = table[0, j // page].long(), slice(None), j % page
    assert torch.equal(k[at], q) and torch.equal(v[at], vv)
    cu, kv = torch.tensor([0, 60], **i32), torch.tensor([60], **i32)
    lse = evict_ref.attention_lse(q, k, table, cu, kv)
    ref, tol = evict_ref.weights(q, k, table, cu, kv, lse, w)
    tw.ops.paged_weights(q, k, table, cu, kv, lse, w, max_q_len=60, max_kv_len=60)
    assert bool(((w.double() - ref).abs() <= tol).all()) and bool((w[at] > 0).all())
    had = [w[at].T.clone(), k[at].transpose(0, 1).clone(), v[at].transpose(0, 1).clone()]
    out = [torch.zeros(1, **i32) for _ in range(2)]
    tw.ops.paged_evict(k, v, w, p, table, kv, torch.tensor([33], **i32), torch.zeros(1, **i32),
                       max_len=60, sink=2, recent=5, lens_out=out[0], offsets_out=out[1])
    at = table[0, j[:33] // page].long(), slice(None), j[:33] % page
    places = p[at].T.long()  # [heads, 33]
    for h in range(heads):
        fixed = (j < 2) | (j >= 55)
        best = torch.where(fixed, torch.inf, had[0][h]).sort(descending=True, stable=True).indices
        assert sorted(places[h].tolist()) == sorted(best[:33].tolist())
        assert torch.equal(k[at][:, h], had[1][h][places[h]])
        assert torch.equal(v[at][:, h], had[2][h][places[h]])
