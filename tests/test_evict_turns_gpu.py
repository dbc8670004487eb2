"""Eviction whose clusters take several tasks (a request, layer and head) one after another, as
they do for a whole model: against a stable sort of each."""

from __future__ import annotations

import random

import pytest
import torch

import test_evict_gpu

pytestmark = pytest.mark.gpu

D = 128


def launched(max_len, tasks):
    """(CTAs a cluster, clusters) of a call, by the rule that the launch goes by."""
    C = 1
    while C < 8 and max_len > C * 4096 and (2 * C * tasks <= 296 or max_len > C * 16384):
        C *= 2
    return C, min(tasks, 592 // C)


def reference(s, keep, sink, recent):
    """The call on copies, a stable sort for each request, layer and head: (k, v, w, p, lens,
    offsets, stack, count)."""
    kv, w, p = [t.clone() for t in s["kv"]], s["w"].clone(), s["p"].clone()
    page, stack, at = s["page"], s["stack"].clone(), int(s["count"])
    lens, gone = s["lens"].tolist(), s["gone"].tolist()
    lens_out, gone_out = list(lens), list(gone)
    for b, (n, m) in enumerate(zip(lens, keep)):
        if m < 0 or n <= m:
            continue
        j = torch.arange(n, device=w.device)
        pages, row = s["table"][b, j // page].long(), j % page
        for l in range(w.shape[0]):
            for h in range(w.shape[2]):
                place = p[l, pages, h, row]
                fixed = (place < sink) | (place >= n + gone[b] - recent)
                rank = torch.where(fixed, torch.inf, w[l, pages, h, row].double())
                best = rank.sort(descending=True, stable=True).indices[:m]
                stays = torch.zeros(n, dtype=torch.bool, device=w.device)
                stays[best] = True
                to = torch.nonzero(~stays[:m])[:, 0]
                source = torch.nonzero(stays[m:])[:, 0] + m
                for t in (*kv, w, p):
                    t[l, pages[to], h, row[to]] = t[l, pages[source], h, row[source]]
        first, last = -(-m // page), -(-n // page)
        stack[at:at + last - first] = s["table"][b, first:last]
        at += last - first
        lens_out[b], gone_out[b] = m, gone[b] + n - m
    return [*kv, w, p], lens_out, gone_out, stack, at


def state(dev, seed, lens, *, layers, heads, page=16):
    """A cache with pages in any order.  Weights below 1, a third of them equal; every fourth
    head's fall with the row (nothing moves), every fourth's rise (all that stays moves)."""
    g = torch.Generator(dev).manual_seed(seed)
    held = [-(-n // page) for n in lens]
    pages = sum(held) + 3
    ids = torch.randperm(pages, generator=g, device=dev).int()
    i32 = dict(dtype=torch.int32, device=dev)
    table, at = torch.full((len(lens), max(held) + 1), -1, **i32), 0
    w = torch.rand(layers, pages, heads, page, generator=g, device=dev)
    w[torch.rand(w.shape, generator=g, device=dev) < 0.3] = 0.5
    p = torch.zeros(layers, pages, heads, page, **i32)
    gone = [(7 * b) % 40 for b in range(len(lens))]
    for b, n in enumerate(held):
        table[b, :n] = ids[at:at + n]
        at += n
        j = torch.arange(lens[b], device=dev)
        where = table[b, j // page].long()
        p[:, where, :, j % page] = (j + gone[b]).int()[:, None, None]
        for h in range(heads):
            if h % 4 == 2:
                w[:, where, h, j % page] = (1 - (j + 1) / (lens[b] + 1)).float()
            elif h % 4 == 3:
                w[:, where, h, j % page] = ((j + 1) / (lens[b] + 1)).float()
    stack = torch.full((pages,), -1, **i32)
    stack[:pages - at] = ids[at:]
    kv = [torch.randint(-30000, 30000, (layers, pages, heads, page, D), generator=g, device=dev,
                        dtype=torch.int16) for _ in range(2)]
    return dict(kv=kv, w=w, p=p, table=table, stack=stack, page=page,
                count=torch.tensor([pages - at], **i32), lens=torch.tensor(lens, **i32),
                gone=torch.tensor(gone, **i32))


def check(tw, s, keep, sink, recent, max_len):
    want, lens_out, gone_out, stack, count = reference(s, keep, sink, recent)
    i32 = dict(dtype=torch.int32, device=s["w"].device)
    got_lens, got_gone, left, err = (torch.zeros(n, **i32) for n in (len(keep), len(keep), 1, 1))
    k, v = (t.view(torch.float16) for t in s["kv"])
    tw.ops.paged_evict(k, v, s["w"], s["p"], s["table"], s["lens"], torch.tensor(keep, **i32),
                       s["gone"], max_len=max_len, sink=sink, recent=recent, lens_out=got_lens,
                       offsets_out=got_gone, free_pages=s["stack"], free_count=s["count"],
                       free_count_out=left, error_flag=err)
    assert int(err) == 0
    assert got_lens.tolist() == lens_out and got_gone.tolist() == gone_out
    assert int(left) == count and torch.equal(s["stack"], stack)
    for got, t in zip((s["p"], s["w"], *s["kv"]), (want[3], want[2], want[0], want[1])):
        assert torch.equal(got, t)


@pytest.mark.parametrize("max_len,cluster", [(700, 1), (20_000, 2), (40_000, 4), (1 << 18, 8),
                                             (1 << 21, 8)])
def test_tasks_in_turn(tw, cuda, max_len, cluster):
    """Short requests under a far bound: each cluster takes four tasks and more, among them
    such without rows that move, with equal weights at the border, with nothing to keep, and
    requests that are left as they are or hold nothing."""
    rng = random.Random(max_len)
    layers, heads = 8, 8
    lens = [rng.choice((0, 1, 31, 64, 100, 333, 700)) for _ in range(12)] * 4
    keep = [rng.choice((-1, 0, n // 2, n // 3, max(n - 3, 0), n, n + 1)) for n in lens]
    C, clusters = launched(max_len, len(lens) * layers * heads)
    assert C == cluster and len(lens) * layers * heads >= 4 * clusters
    for sink, recent in ((0, 0), (3, 20)):
        s = state(cuda, max_len + sink, lens, layers=layers, heads=heads)
        check(tw, s, keep, sink, recent, max_len)


@pytest.mark.parametrize("lens,keep,layers,heads", [
    # (clusters of two, of four, of eight)
    ([20_000, 300, 17_001, 5000], [9000, 100, 17_000, 2500], 16, 8),
    ([40_000, 500, 39_999], [2048, 200, 30_000], 10, 8),
    ([70_001, 64], [2048, 33], 12, 8)])
def test_long_requests_in_turn(tw, cuda, lens, keep, layers, heads):
    """Rows in all CTAs of a cluster, several tasks each, short ones after long ones."""
    C, clusters = launched(max(lens), len(lens) * layers * heads)
    assert C > 1 and len(lens) * layers * heads > clusters
    s = state(cuda, len(lens), lens, layers=layers, heads=heads)
    check(tw, s, keep, 4, 64, max(lens))


def test_lists_in_several_turns(tw, cuda):
    """More rows that move than the cluster's memory lists (32768 of them under the largest
    bound), in tasks that a cluster takes before and after others."""
    lens = [72_000 if b in (0, 19, 37) else 40 + b for b in range(40)]
    keep = [36_000 if n > 70_000 else 30 for n in lens]
    max_len = 1 << 21
    C, clusters = launched(max_len, 4 * len(lens))
    assert C == 8 and clusters == 74 and 4 * len(lens) > 2 * clusters
    s = state(cuda, 5, lens, layers=1, heads=4, page=64)
    check(tw, s, keep, 0, 0, max_len)


def test_against_the_lists(tw, cuda):
    """The same, against the ranking over Python lists."""
    rng = random.Random(4)
    lens = [rng.randint(0, 60) for _ in range(90)]
    keep = [rng.randint(0, n) for n in lens]
    layers = 4
    C, clusters = launched(1 << 18, len(lens) * layers * 2)
    assert C == 8 and len(lens) * layers * 2 >= 9 * clusters
    s = test_evict_gpu.state(cuda, 6, lens, layers=layers, heads=2, page=8,
                             gone=[rng.randint(0, 9) for _ in lens])
    test_evict_gpu.check(tw, s, keep, 2, 6, max_len=1 << 18)
