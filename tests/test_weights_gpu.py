"""Accumulated attention weights against the formula in 64 bits."""

from __future__ import annotations

import math
import random

import pytest
import torch

import evict_ref

pytestmark = pytest.mark.gpu

D = 128


def state(dev, seed, new, before, *, q_heads=8, kv_heads=2, page=16, dtype=torch.bfloat16,
          pool="head", pad=0, loud=1.0):
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    kv = [b + x for b, x in zip(before, new)]
    held = [-(-n // page) for n in kv]
    pages = sum(held) + 3
    ids = list(range(pages))
    rng.shuffle(ids)
    table = torch.full((len(new), max(held + [1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    shape = (pages, kv_heads, page, D) if pool == "head" else (pages, page, kv_heads, D)
    k = torch.randn(shape, generator=g)
    if pool == "token":
        k = k.transpose(1, 2)
    k[..., 3] *= loud
    if pool == "token":  # [pages, rows, heads, D] in memory
        k = k.transpose(1, 2).to(dtype).to(dev).transpose(1, 2)
    else:
        k = k.to(dtype).to(dev)
    q = torch.randn(sum(new) + pad, q_heads, D, generator=g).to(dtype).to(dev)
    i32 = dict(dtype=torch.int32, device=dev)
    cu = torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], **i32)
    s = dict(q=q, k_pages=k, block_table=table.to(dev), cu_q=cu, kv_lens=torch.tensor(kv, **i32),
             row_weights=torch.rand(pages, kv_heads, page, generator=g).to(dev))
    s["max"] = dict(max_q_len=max(new), max_kv_len=max(kv))
    return s


def check(tw, s, *, window=0, last=0, scale=None, lse=None):
    if lse is None:
        lse = evict_ref.attention_lse(s["q"], s["k_pages"], s["block_table"], s["cu_q"],
                                      s["kv_lens"], window, scale)
    ref, tol = evict_ref.weights(s["q"], s["k_pages"], s["block_table"], s["cu_q"], s["kv_lens"],
                                 lse, s["row_weights"], window=window, last=last, scale=scale)
    got = s["row_weights"].clone()
    err = torch.zeros(1, dtype=torch.int32, device=got.device)
    tw.ops.paged_weights(s["q"], s["k_pages"], s["block_table"], s["cu_q"], s["kv_lens"], lse, got,
                         window=window, last=last, softmax_scale=scale, error_flag=err, **s["max"])
    assert int(err) == 0
    # a sum beyond the largest 32-bit number (2^128 (1 - 2^-24)) is infinite in 32 bits: its
    # terms are not negative, so no order of additions brings it back
    ref = torch.where(torch.isinf(ref.float()), ref * math.inf, ref)
    odd = ~torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got[odd & ~torch.isnan(ref)].double(), ref[odd & ~torch.isnan(ref)])
    apart = (got.double() - ref).abs()[~odd]
    assert bool((apart <= tol[~odd]).all()), (apart - tol[~odd]).max()
    again = s["row_weights"].clone()  # the same bits whatever ran when
    tw.ops.paged_weights(s["q"], s["k_pages"], s["block_table"], s["cu_q"], s["kv_lens"], lse,
                         again, window=window, last=last, softmax_scale=scale, **s["max"])
    assert torch.equal(got.view(torch.int32), again.view(torch.int32))
    return got


@pytest.mark.parametrize("q_heads,kv_heads", [(8, 8), (8, 2), (6, 2), (14, 2), (5, 1), (16, 1),
                                              (64, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_single_tokens(tw, cuda, q_heads, kv_heads, dtype):
    s = state(cuda, q_heads, [1] * 6, [0, 1, 127, 128, 300, 1500], q_heads=q_heads,
              kv_heads=kv_heads, dtype=dtype)
    check(tw, s)


@pytest.mark.parametrize("q_heads,kv_heads", [(8, 8), (8, 2), (6, 2), (14, 2), (16, 1), (64, 1)])
@pytest.mark.parametrize("page,pool", [(8, "head"), (16, "token"), (24, "head"), (64, "head"),
                                       (128, "token")])
def test_chunks(tw, cuda, q_heads, kv_heads, page, pool):
    s = state(cuda, page, [33, 1, 130, 0, 2, 255], [100, 700, 0, 50, 5, 513], q_heads=q_heads,
              kv_heads=kv_heads, page=page, pool=pool, dtype=torch.float16)
    check(tw, s)


@pytest.mark.parametrize("n,before", [(1, 4000), (2, 0), (3, 255), (5, 256), (17, 1000), (127, 1),
                                      (128, 128), (129, 900), (500, 0), (700, 333), (1024, 1024)])
def test_one_request(tw, cuda, n, before):
    """Clusters of every size: a single request's few blocks of keys."""
    s = state(cuda, n, [n], [before], q_heads=4, kv_heads=1)
    check(tw, s)


@pytest.mark.parametrize("window", [1, 5, 64, 128, 129, 300, 2 ** 31 - 1])
@pytest.mark.parametrize("last", [0, 1, 40])
def test_windows(tw, cuda, window, last):
    s = state(cuda, window % 1000, [150, 1, 3, 400], [0, 900, 256, 300], q_heads=6, kv_heads=2)
    check(tw, s, window=window, last=last)
    one = state(cuda, window % 1000 + 1, [400], [700], q_heads=8, kv_heads=2)
    check(tw, one, window=window, last=last)


@pytest.mark.parametrize("last", [1, 2, 31, 32, 33, 200, 5000])
def test_last(tw, cuda, last):
    s = state(cuda, last, [150, 1, 33, 257], [10, 900, 256, 0], q_heads=8, kv_heads=2)
    check(tw, s, last=last)


def test_sums_to_rows(tw, cuda):
    """Every counted row gives one in all: the weights of a head sum to the number of rows."""
    s = state(cuda, 4, [300], [500], q_heads=8, kv_heads=2)
    s["row_weights"].zero_()
    got = check(tw, s)
    assert got.double().sum((0, 2)).tolist() == pytest.approx([300 * 4] * 2, rel=1e-5)


def test_lse_of_the_attention(tw, cuda):
    """With paged_attention's own lse, as a serving step calls them."""
    s = state(cuda, 8, [64, 1, 200], [0, 700, 90], q_heads=8, kv_heads=2)
    lse = torch.empty(s["q"].shape[:2], device=cuda)
    tw.ops.paged_attention(s["q"], s["k_pages"], s["k_pages"], s["block_table"], s["cu_q"],
                           s["kv_lens"], lse=lse, **s["max"])
    check(tw, s, lse=lse)


def test_values_that_are_not_finite(tw, cuda):
    """What the mask hides does not count, in K or in the rows beside: NaN and infinities in
    rows no one sees, in later requests' q, in unused places of pages."""
    s = state(cuda, 2, [40, 1, 130], [60, 300, 20], q_heads=6, kv_heads=2, pad=5)
    lse = evict_ref.attention_lse(s["q"], s["k_pages"], s["block_table"], s["cu_q"], s["kv_lens"])
    lse[int(s["cu_q"][-1]):] = float("nan")
    s["q"][int(s["cu_q"][-1]):] = float("nan")
    # rows past each request's end, and pages no request has
    used = torch.zeros(s["k_pages"].shape[:3], dtype=torch.bool, device=cuda)
    for b, kv in enumerate(s["kv_lens"].tolist()):
        j = torch.arange(kv, device=cuda)
        used[s["block_table"][b, j // 16].long(), :, j % 16] = True
    s["k_pages"][~used] = float("nan")
    got = check(tw, s, lse=lse)
    assert bool(torch.isfinite(got).all())
    # a NaN row of q counts where it is seen, and only there
    s["q"][10] = float("nan")
    lse[10] = float("nan")
    got = check(tw, s, lse=lse)
    assert bool(torch.isnan(got).any()) and not bool(torch.isnan(got).all())
    # a key that is infinite in places; rows whose group does not fill 128 columns
    s = state(cuda, 3, [130], [20], q_heads=6, kv_heads=2)
    lse = evict_ref.attention_lse(s["q"], s["k_pages"], s["block_table"], s["cu_q"], s["kv_lens"])
    s["q"][..., 7] = s["q"][..., 7].abs() + 1
    s["k_pages"][int(s["block_table"][0, 2]), :, 5, 7] = -float("inf")
    check(tw, s, lse=lse)  # its scores are -inf: no weight


def test_rows_that_see_nothing(tw, cuda):
    """More new rows than rows held (positions below 0): they see nothing and count nothing,
    and so does a row whose lse is -inf, whatever its scores."""
    s = state(cuda, 5, [40], [0], q_heads=4, kv_heads=1)
    s["kv_lens"].fill_(25)
    check(tw, s)
    s = state(cuda, 5, [40, 1], [20, 100], q_heads=4, kv_heads=1)
    lse = evict_ref.attention_lse(s["q"], s["k_pages"], s["block_table"], s["cu_q"], s["kv_lens"])
    lse[3:30] = -math.inf
    lse[40] = -math.inf
    check(tw, s, lse=lse)
    lse[5] = math.inf
    check(tw, s, lse=lse)


@pytest.mark.parametrize("loud,scale", [(30.0, None), (300.0, None), (1.0, 1.0), (1.0, 1e-3),
                                        (3000.0, 1.0)])
def test_large_scores(tw, cuda, loud, scale):
    s = state(cuda, 6, [50, 1], [200, 600], q_heads=4, kv_heads=2, loud=loud)
    check(tw, s, scale=scale)


def test_any_lse(tw, cuda):
    """A log-sum-exp of other scores: the formula holds, up to infinity."""
    s = state(cuda, 7, [50, 1], [200, 600], q_heads=4, kv_heads=2)
    lse = torch.randn(s["q"].shape[:2], device=cuda) * 20
    lse[::7] -= 60
    check(tw, s, lse=lse)
    lse.fill_(-200.0)
    got = check(tw, s, lse=lse)
    assert bool(torch.isinf(got).any())


def test_flags(tw, cuda):
    L = tw._lib
    s = state(cuda, 9, [5, 40], [100, 30], q_heads=4, kv_heads=1)
    lse = evict_ref.attention_lse(s["q"], s["k_pages"], s["block_table"], s["cu_q"], s["kv_lens"])

    def run(**change):
        got = s["row_weights"].clone()
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        args = {**{n: s[n] for n in ("q", "k_pages", "block_table", "cu_q", "kv_lens")},
                **s["max"], **change}
        tw.ops.paged_weights(lse=lse, row_weights=got, error_flag=err, **args)
        return got, int(err)

    good, err = run()
    assert err == 0
    # a request with more rows than max_q_len is not counted
    got, err = run(max_q_len=39)
    assert err == L.TW_ERR_BAD_ARG
    mine = torch.zeros_like(got, dtype=torch.bool)
    j = torch.arange(70, device=cuda)
    mine[s["block_table"][1, j // 16].long(), :, j % 16] = True
    assert torch.equal(got[~mine], good[~mine]) and torch.equal(got[mine], s["row_weights"][mine])
    # a longer one than max_kv_len is, all the same
    got, err = run(max_kv_len=3)
    assert err == 0 and torch.equal(got, good)
    # pages outside the pool: flagged, their keys left out
    for bad in (-1, s["k_pages"].shape[0], 1 << 30):
        table = s["block_table"].clone()
        page = int(table[0, 2])
        table[0, 2] = bad
        got, err = run(block_table=table)
        assert err == L.TW_ERR_INVALID_INDEX
        assert torch.equal(got[page], s["row_weights"][page])
        rest = torch.arange(got.shape[0], device=cuda) != page
        assert torch.equal(got[rest], good[rest])
    # more rows held than the table has places for
    got, err = run(kv_lens=torch.tensor([5000, 70], dtype=torch.int32, device=cuda))
    assert err == L.TW_ERR_INVALID_INDEX
    # rows that q does not have
    got, err = run(cu_q=torch.tensor([0, 5, 99], dtype=torch.int32, device=cuda), max_q_len=99)
    assert err == L.TW_ERR_BAD_ARG


def test_refusals(tw, cuda):
    s = state(cuda, 10, [5], [100], q_heads=4, kv_heads=2)
    lse = torch.zeros(5, 4, device=cuda)
    good = {**{n: s[n] for n in ("q", "k_pages", "block_table", "cu_q", "kv_lens", "row_weights")},
            **s["max"], "lse": lse}
    w = s["row_weights"]
    for bad in (dict(q=s["q"].float()), dict(q=s["q"][:, :3]), dict(q=s["q"][..., :64]),
                dict(lse=lse.double()), dict(lse=lse[:4]), dict(lse=None),
                dict(lse=lse.t().contiguous().t()), dict(row_weights=w.half()),
                dict(row_weights=w[:2]), dict(row_weights=None),
                dict(row_weights=w.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(cu_q=s["cu_q"].long()), dict(kv_lens=s["kv_lens"][:0]), dict(window=-1),
                dict(last=-1), dict(softmax_scale=0.0), dict(max_q_len=-1),
                dict(k_pages=s["k_pages"][:, :, :12]), dict(block_table=s["block_table"].t())):
        with pytest.raises(ValueError):
            tw.ops.paged_weights(**{**good, **bad})
    tw.ops.paged_weights(**good)


def test_shared_pages(tw, cuda):
    """Two requests over the same pages: both count (in either order: two additions)."""
    s = state(cuda, 11, [1, 1], [200, 200], q_heads=4, kv_heads=1)
    s["block_table"][1] = s["block_table"][0]
    lse = evict_ref.attention_lse(s["q"], s["k_pages"], s["block_table"], s["cu_q"], s["kv_lens"])
    ref, tol = evict_ref.weights(s["q"], s["k_pages"], s["block_table"], s["cu_q"], s["kv_lens"],
                                 lse, s["row_weights"])
    tw.ops.paged_weights(s["q"], s["k_pages"], s["block_table"], s["cu_q"], s["kv_lens"], lse,
                         s["row_weights"], **s["max"])
    assert bool(((s["row_weights"].double() - ref).abs() <= 2 * tol).all())


def test_many_requests(tw, cuda):
    """More requests than a warp looks at in one go; many of them wait."""
    rng = random.Random(1)
    new = [rng.choice((0, 0, 0, 1, 1, 7)) for _ in range(150)]
    before = [rng.randint(0, 400) if n else 0 for n in new]
    s = state(cuda, 12, new, before, q_heads=4, kv_heads=2)
    check(tw, s)


def test_graph_and_stream(tw, cuda):
    s = state(cuda, 13, [70, 1], [200, 900], q_heads=8, kv_heads=2)
    lse = evict_ref.attention_lse(s["q"], s["k_pages"], s["block_table"], s["cu_q"], s["kv_lens"])
    call = lambda w: tw.ops.paged_weights(  # noqa: E731
        s["q"], s["k_pages"], s["block_table"], s["cu_q"], s["kv_lens"], lse, w, **s["max"])
    w = torch.zeros_like(s["row_weights"])
    call(w.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(w)
    s["q"].mul_(0.5)
    lse.copy_(evict_ref.attention_lse(s["q"], s["k_pages"], s["block_table"], s["cu_q"],
                                      s["kv_lens"]))
    side, want = torch.cuda.Stream(cuda), torch.zeros_like(w)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        call(want)
        call(want)
    side.synchronize()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(w, want)


@pytest.mark.parametrize("q_heads,kv_heads", [(4, 1), (8, 2), (6, 2), (32, 2)])
def test_clusters_of_several_items(tw, cuda, q_heads, kv_heads):
    """Few items that clusters take, more of them than clusters, so that each takes several:
    a tile or two for a CTA, or none.  Many times, for what depends on who is first."""
    new = [70, 1, 257, 33, 0, 129, 300, 2, 90, 65, 40, 128]
    s = state(cuda, 14, new, [3, 500, 40, 256, 9, 0, 200, 700, 1, 511, 90, 128], q_heads=q_heads,
              kv_heads=kv_heads, dtype=torch.float16)
    first = check(tw, s)
    for _ in range(20):
        assert torch.equal(first, check(tw, s))
    for seed in range(8):
        rng = random.Random(seed)
        new = [rng.choice((0, 1, rng.randint(2, 300))) for _ in range(rng.randint(4, 14))]
        check(tw, state(cuda, seed, new + [64], [rng.randint(0, 600) for _ in new] + [5],
                        q_heads=q_heads, kv_heads=kv_heads), last=rng.choice((0, 0, 100)))
