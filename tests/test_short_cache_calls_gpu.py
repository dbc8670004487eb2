"""PagedKVCache kept short: windows beside requests that wait, budgets as numbers of any kind,
a run in which rows are lost, and two caches whose kernels run at the same time."""

from __future__ import annotations

import pytest
import torch

import evict_ref
import paged_ref

pytestmark = pytest.mark.gpu

D = 128


def make(tw, dev, **kw):
    args = dict(num_layers=1, num_kv_heads=2, num_pages=60, max_requests=3,
                max_tokens_per_request=320, page_size=16, dtype=torch.float16, device=dev,
                track_weights=True)
    return tw.PagedKVCache(**{**args, **kw})


def rows(g, dev, n, heads=8):
    return torch.randn(n, heads, D, generator=g).to(torch.float16).to(dev)


def feed(cache, g, dev, new, **kw):
    """A step of random rows; (plan, q, out)."""
    plan = cache.step(new)
    x = rows(g, dev, plan.tokens)
    cache.write(0, x[:, :2], x[:, 2:4])
    return plan, x[:, 4:], cache.attend(0, x[:, 4:], **kw)


def test_window_while_a_cut_request_waits(tw, cuda):
    """A window is refused for tokens of a request that has lost rows, not for those of others
    while it waits; and outputs and weights are then those of the window."""
    g = torch.Generator().manual_seed(1)
    cache = make(tw, cuda)
    feed(cache, g, cuda, [90, 40])
    cache.evict([50], sink=2, recent=8)
    assert cache.evicted == [40, 0, 0]
    weights = cache.row_weights[0].clone()
    plan = cache.step([0, 30, 25])
    x = rows(g, cuda, 55)
    cache.write(0, x[:, :2], x[:, 2:4])
    for r, i, n in ((1, 40, 30), (2, 0, 25)):
        j = torch.arange(i, i + n, device=cuda)
        weights[cache.block_table[r, j // 16].long(), :, j % 16] = 0
    q, lse = x[:, 4:], torch.empty(55, 4, device=cuda)
    out = cache.attend(0, q, window=20, lse=lse)
    args = (q, cache.pool[0, 0], cache.pool[0, 1], cache.block_table, plan.cu_q, plan.kv_lens)
    ref, _, tol, _ = paged_ref.attention(*args, window=20)
    assert bool(((out.double() - ref).abs() <= tol).all())
    wref, wtol = evict_ref.weights(args[0], args[1], *args[3:], lse, weights, window=20)
    assert bool(((cache.row_weights[0].double() - wref).abs() <= wtol).all())
    cache.step([1, 1])  # now it has a token
    x = rows(g, cuda, 2)
    cache.write(0, x[:, :2], x[:, 2:4])
    with pytest.raises(ValueError, match="window"):
        cache.attend(0, x[:, 4:], window=20)
    cache.attend(0, x[:, 4:])
    cache.step([-1, 1])  # it ends, another begins in its place
    cache.step([5])
    x = rows(g, cuda, 5)
    cache.write(0, x[:, :2], x[:, 2:4])
    cache.attend(0, x[:, 4:], window=3)
    cache.synchronize()


def test_budgets_of_any_kind(tw, cuda):
    """One number for all requests, also one of NumPy's; numbers for each, in any sequence."""
    np = pytest.importorskip("numpy")
    for keep, want in ((np.int64(40), [40, 30, 40]), (np.int32(40), [40, 30, 40]),
                       (np.array([40, -1], dtype=np.int64), [40, 30, 70]),
                       (torch.tensor([-1, 20]), [90, 20, 70]), ((50,), [50, 30, 70])):
        cache = make(tw, cuda)
        feed(cache, torch.Generator().manual_seed(2), cuda, [90, 30, 70])
        cache.evict(keep, sink=2, recent=8)
        assert cache.lengths == want
        cache.synchronize()
        assert cache._lens.tolist() == want
    cache = make(tw, cuda)
    with pytest.raises(TypeError):
        cache.evict(40.0, sink=2, recent=8)


def test_a_run_loses_rows(tw, cuda):
    """Steps and evictions in turn: every request loses rows, in every turn some do."""
    g = torch.Generator().manual_seed(3)
    cache = make(tw, cuda)
    lost = [0, 0, 0]
    for turn in range(6):
        plan, q, out = feed(cache, g, cuda, [60, 1 + 30 * (turn % 2), 45])
        args = (q, cache.pool[0, 0], cache.pool[0, 1], cache.block_table, plan.cu_q, plan.kv_lens)
        ref, _, tol, _ = paged_ref.attention(*args)
        assert bool(((out.double() - ref).abs() <= tol).all())
        before = list(cache.lengths)
        cache.evict(50, sink=2, recent=12)
        gone = [a - b for a, b in zip(before, cache.lengths)]
        assert any(gone)
        lost = [a + b for a, b in zip(lost, gone)]
        assert cache.evicted == lost
    assert all(lost)
    cache.synchronize()
    assert cache._lens.tolist() == cache.lengths and cache._offsets.tolist() == cache.evicted


class Turn:
    """One cache's operators over device tensors that are all there beforehand: a round writes
    a chunk and single tokens, attends, weighs and evicts, with no word from the host."""

    def __init__(self, tw, dev, seed, lens, new, page=16, heads=2, q_heads=8):
        g = torch.Generator().manual_seed(seed)
        i32 = dict(dtype=torch.int32, device=dev)
        held = [-(-n // page) for n in lens]
        pages, B = sum(held) + 2, len(lens)
        ids = torch.randperm(pages, generator=g)
        table, at = torch.zeros(B, max(held), dtype=torch.int32), 0
        for b, n in enumerate(held):
            table[b, :n] = ids[at:at + n].int()
            at += n
        T = sum(new)
        self.tw, self.new, self.lens = tw, max(new), max(lens)
        self.kv = [torch.randn(pages, heads, page, D, generator=g).to(torch.float16).to(dev)
                   for _ in range(2)]
        self.w = torch.rand(pages, heads, page, generator=g).to(dev)
        self.p = torch.randint(0, 3 * max(lens), (pages, heads, page), generator=g,
                               dtype=torch.int32).to(dev)
        qkv = torch.randn(T, q_heads + 2 * heads, D, generator=g).to(torch.float16).to(dev)
        self.qkv = qkv.split((q_heads, heads, heads), 1)
        j = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)])
        b = torch.cat([torch.full((m,), i) for i, m in enumerate(new)])
        self.positions = j.int().to(dev)
        self.slots = (table[b, j // page].long() * page + j % page).to(dev)
        self.table = table.to(dev)
        self.cu_q = torch.tensor([sum(new[:i]) for i in range(B + 1)], **i32)
        self.kv_lens = torch.tensor(lens, **i32)
        self.keep = torch.tensor([n * 2 // 3 for n in lens], **i32)
        self.offsets = torch.tensor([n // 2 for n in lens], **i32)
        self.lens_out, self.gone_out = torch.zeros(B, **i32), torch.zeros(B, **i32)
        self.lse = torch.empty(T, q_heads, device=dev)
        self.err = torch.zeros(1, **i32)
        self.f, _ = tw.ops.rope_frequencies(96, device=dev)
        self.outs = []

    def operators(self):
        """The round's calls, one by one."""
        ops, (q, k, v), (kp, vp) = self.tw.ops, self.qkv, self.kv
        how = dict(max_q_len=self.new, max_kv_len=self.lens, error_flag=self.err)
        q = ops.paged_rope_write(q, k, v, self.positions, self.slots, self.f, kp, vp,
                                 row_weights=self.w, row_positions=self.p, error_flag=self.err)
        yield
        out = ops.paged_attention(q, kp, vp, self.table, self.cu_q, self.kv_lens, lse=self.lse,
                                  **how)
        yield
        ops.paged_weights(q, kp, self.table, self.cu_q, self.kv_lens, self.lse, self.w, **how)
        yield
        ops.paged_evict(kp, vp, self.w, self.p, self.table, self.kv_lens, self.keep, self.offsets,
                        max_len=self.lens, sink=4, recent=16, lens_out=self.lens_out,
                        offsets_out=self.gone_out, error_flag=self.err)
        yield
        self.outs += [q, out, self.lse.clone(), self.w.clone(), self.p.clone()]

    def state(self):
        return [*self.outs, *self.kv, self.lens_out, self.gone_out]


def test_two_caches_at_the_same_time(tw, cuda):
    """The operators of two caches, launched in turn on two streams that begin together, with
    enough of them that both are at work: each cache gets what it gets alone."""
    plans = ((11, [2000, 700, 901], [300, 1, 40]), (12, [5000, 90], [1, 1]))
    rounds = 12

    def launch(turns, streams):
        """All operators of the rounds, one of each cache in turn; when each stream was busy."""
        begin = torch.cuda.Event()
        hold = torch.empty(1 << 28, dtype=torch.int32, device=cuda)
        torch.cuda.synchronize()
        for _ in range(20):  # the streams start behind this: several ms
            hold.add_(1)
        begin.record()
        times = []
        for s in streams:
            s.wait_event(begin)
            with torch.cuda.stream(s):
                times.append([torch.cuda.Event(enable_timing=True) for _ in range(2)])
                times[-1][0].record()
        for _ in range(rounds):
            calls = [t.operators() for t in turns]
            for _ in range(5):  # (the last: what the round leaves is copied)
                for s, call in zip(streams, calls):
                    with torch.cuda.stream(s):
                        next(call, None)
        for s, t in zip(streams, times):
            with torch.cuda.stream(s):
                t[1].record()
        torch.cuda.synchronize()
        return times

    make_all = lambda: [Turn(tw, cuda, *plan) for plan in plans]  # noqa: E731
    alone = make_all()
    for t in alone:
        launch([t], [torch.cuda.Stream(cuda)])
    for _ in range(3):
        both = make_all()
        a, b = launch(both, [torch.cuda.Stream(cuda) for _ in both])
        assert a[0].elapsed_time(b[1]) > 0 and b[0].elapsed_time(a[1]) > 0  # side by side
        for x, y in zip(alone, both):
            assert int(x.err) == 0 and int(y.err) == 0
            assert len(y.state()) == 5 * rounds + 4
            assert all(torch.equal(s, t) for s, t in zip(x.state(), y.state()))
    assert any(not torch.equal(s, t) for s, t in zip(alone[0].outs, alone[0].outs[5:]))
