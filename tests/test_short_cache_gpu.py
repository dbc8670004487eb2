"""PagedKVCache with rotary positions, weights and eviction: a run of them together against
the same in 64 bits, row by row, and what is refused."""

from __future__ import annotations

import math
import random
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import evict_ref
import paged_ref

pytestmark = pytest.mark.gpu

REPO = Path(__file__).resolve().parents[1]
D = 128


def make(tw, dev, **kw):
    args = dict(num_layers=2, num_kv_heads=2, num_pages=60, max_requests=3,
                max_tokens_per_request=320, page_size=16, dtype=torch.float16, device=dev,
                track_weights=True)
    return tw.PagedKVCache(**{**args, **kw})


def test_a_run_of_steps(tw, cuda):
    """Chunks, single tokens, evictions, ends and new requests.  After each step: outputs and
    weights as the rows in the cache give them; rows, positions and weights of each head are
    those of tokens that were written (each at most once, protected ones among them); pages
    are held once or free."""
    rng, g = random.Random(3), torch.Generator().manual_seed(3)
    cache = make(tw, cuda)
    rotary = tw.RotaryPositions(96, base=5000.0, layout="interleaved", device=cuda)
    written = [{}, {}, {}]  # per request: position -> (k, v) per layer, k turned
    for turn in range(14):
        new = []
        for r in range(3):
            n = rng.choice((0, 1, 1, rng.randint(2, 80)))
            if cache.lengths[r] + n > 300 or (cache.lengths[r] and rng.random() < 0.12):
                n = -1
            new.append(n)
        seen = [l + e for l, e in zip(cache.lengths, cache.evicted)]
        plan = cache.step(new)
        total, cu = plan.tokens, plan.cu_q.tolist()
        for r, n in enumerate(new):
            if n < 0:
                written[r] = {}
                assert cache.evicted[r] == 0
            elif n:
                assert plan.positions[cu[r]:cu[r + 1]].tolist() == list(range(seen[r], seen[r] + n))
        for layer in range(2):
            rows = torch.randn(total, 10, D, generator=g).to(torch.float16).to(cuda)
            q, k, v = rows.split((6, 2, 2), 1)
            before = cache.row_weights[layer].clone()
            turned = cache.write_rotated(layer, q, k, v, rotary)
            assert torch.equal(turned, rotary(q, plan.positions))
            kt = rotary(k, plan.positions)
            for r in range(3):
                for i in range(cu[r], cu[r + 1]):
                    written[r].setdefault(int(plan.positions[i]), {})[layer] = (kt[i], v[i])
            out = cache.attend(layer, turned)
            if not total:
                continue
            args = (cache.block_table, plan.cu_q, plan.kv_lens)
            ref, _, tol, _ = paged_ref.attention(turned, cache.pool[layer, 0],
                                                 cache.pool[layer, 1], *args)
            assert bool(((out.double() - ref).abs() <= tol).all())
            for r in range(3):
                for i in range(cu[r], cu[r + 1]):
                    s = int(plan.slots[i])
                    before[s // 16, :, s % 16] = 0
            lse = torch.empty(total, 6, device=cuda)
            tw.ops.paged_attention(turned, cache.pool[layer, 0], cache.pool[layer, 1], *args,
                                   max_q_len=plan.max_q_len, max_kv_len=plan.max_kv_len, lse=lse)
            wref, wtol = evict_ref.weights(turned, cache.pool[layer, 0], *args, lse, before)
            assert bool(((cache.row_weights[layer].double() - wref).abs() <= wtol).all())
        if turn % 3 == 2:
            sums = {}
            for layer in range(2):
                for r in range(3):
                    j = torch.arange(cache.lengths[r], device=cuda)
                    sums[layer, r] = (cache.request_positions(layer, r), cache.row_weights[layer][
                        cache.block_table[r, j // 16].long(), :, j % 16].T.clone())
            lengths, evicted = list(cache.lengths), list(cache.evicted)
            cache.evict(100, sink=3, recent=20)
            assert cache.lengths == [min(l, 100) for l in lengths]
            for r in range(3):
                assert cache.evicted[r] - evicted[r] == lengths[r] - cache.lengths[r]
                tokens = lengths[r] + evicted[r]
                for layer in range(2):
                    for h in range(2):
                        had, weight = (x[h].tolist() for x in sums[layer, r])
                        place = cache.request_positions(layer, r)[h].tolist()
                        if lengths[r] <= 100:
                            assert place == had
                            continue
                        order = sorted(range(len(had)), key=lambda j: (
                            not (had[j] < 3 or had[j] >= tokens - 20),
                            0 if (had[j] < 3 or had[j] >= tokens - 20) else -weight[j], j))
                        assert sorted(place) == sorted(had[j] for j in order[:100])
        for r in range(3):
            for layer in range(2):
                if not cache.lengths[r]:
                    continue
                k, v = cache.request_kv(layer, r)
                places = cache.request_positions(layer, r)
                for h in range(2):
                    p = places[h].tolist()
                    assert len(set(p)) == len(p)
                    want_k = torch.stack([written[r][x][layer][0][h] for x in p])
                    want_v = torch.stack([written[r][x][layer][1][h] for x in p])
                    assert torch.equal(k[h], want_k) and torch.equal(v[h], want_v)
        used = [p for r in range(3)
                for p in cache.block_table[r, :-(-cache.lengths[r] // 16)].tolist()]
        free = cache._free_pages[:cache.free_pages].tolist()
        assert int(cache._free_count[cache._turn]) == cache.free_pages
        assert sorted(used + free) == list(range(cache.num_pages))
        assert cache._lens.tolist() == cache.lengths
        assert cache._offsets.tolist() == cache.evicted
    cache.synchronize()
    assert any(cache.evicted) or turn


def test_plain_write_keeps_records(tw, cuda):
    """write() of rows that the caller turned: K and V as without tracking, records set."""
    g = torch.Generator().manual_seed(4)
    a, b = make(tw, cuda), make(tw, cuda, track_weights=False)
    k, v = (torch.randn(70, 2, D, generator=g).to(torch.float16).to(cuda) for _ in range(2))
    for cache in (a, b):
        cache.pool.zero_()
        if cache is a:
            cache.row_weights.fill_(5)
        cache.step([50, 0, 20])
        cache.write(1, k, v)
    assert torch.equal(a.pool, b.pool)
    assert a.request_positions(1, 0).tolist() == [list(range(50))] * 2
    assert a.request_positions(1, 2).tolist() == [list(range(20))] * 2
    j = torch.arange(50, device=cuda)
    assert not bool(a.row_weights[1][a.block_table[0, j // 16].long(), :, j % 16].any())


def test_last_and_window(tw, cuda):
    g = torch.Generator().manual_seed(5)
    cache = make(tw, cuda, num_layers=1)
    rows = torch.randn(90, 8, D, generator=g).to(torch.float16).to(cuda)
    cache.step([90])
    cache.write(0, rows[:, :2], rows[:, 2:4])
    cache.attend(0, rows[:, 4:], window=30, last=10)
    weights = cache.row_weights[0][cache.block_table[0, torch.arange(90, device=cuda) // 16].long(),
                                   :, torch.arange(90, device=cuda) % 16]
    assert not bool(weights[:90 - 10 - 29].any()) and bool((weights[52:] > 0).all())
    assert weights.double().sum(0).tolist() == pytest.approx([20.0, 20.0], rel=1e-5)
    cache.evict(64, sink=2, recent=8)
    cache.step([1])
    cache.write(0, rows[:1, :2], rows[:1, 2:4])
    with pytest.raises(ValueError, match="window"):
        cache.attend(0, rows[:1, 4:], window=30)
    cache.attend(0, rows[:1, 4:])


def test_refusals(tw, cuda):
    plain, cache = make(tw, cuda, track_weights=False), make(tw, cuda)
    q = torch.zeros(40, 4, D, dtype=torch.float16, device=cuda)
    for c in (plain, cache):
        c.step([40])
        for layer in range(2):
            c.write(layer, q[:, :2], q[:, :2])
    with pytest.raises(ValueError, match="track"):
        plain.evict(8, sink=0, recent=0)
    with pytest.raises(ValueError, match="track"):
        plain.attend(0, q, last=3)
    with pytest.raises(ValueError, match="track"):
        plain.request_positions(0, 0)
    with pytest.raises(ValueError, match="sink"):
        cache.evict(67)
    with pytest.raises(ValueError, match="requests"):
        cache.evict([80] * 4)
    with pytest.raises(ValueError, match="negative"):
        cache.evict(80, sink=-1)
    with pytest.raises(ValueError, match="40 tokens"):
        cache.write_rotated(0, q[:3], q[:, :2], q[:, :2], tw.RotaryPositions(device=cuda))
    with pytest.raises(ValueError):
        tw.RotaryPositions(layout="other", device=cuda)
    cache.evict([-1, 10], sink=1, recent=2)  # nothing to do: the step goes on
    cache.attend(0, q)
    cache.evict([16], sink=1, recent=2)
    assert cache.lengths == [16, 0, 0] and cache.evicted == [24, 0, 0]
    with pytest.raises(ValueError, match="step"):
        cache.attend(0, q)
    assert cache.request_kv(0, 0)[0].shape == (2, 16, D)
    with pytest.raises(ValueError, match="lost"):
        cache.to_offloaded(0, None)
    cache.step([-1])
    assert cache.evicted == [0, 0, 0] and cache.free_pages == cache.num_pages
    cache.synchronize()


def test_rotary_positions(tw, cuda):
    """A score of two turned rows depends on the distance of their positions alone."""
    g = torch.Generator().manual_seed(6)
    rotary = tw.RotaryPositions(128, base=10000.0, device=cuda)
    a, b = (torch.randn(1, 1, D, generator=g).to(torch.float16).to(cuda).expand(40, 1, D)
            .contiguous() for _ in range(2))
    at = torch.arange(40, dtype=torch.int32, device=cuda) * 1000
    x, y = rotary(a, at + 77).double(), rotary(b, at).double()
    scores = (x * y).sum(-1)
    size = (a.double().abs() * b.double().abs()).sum(-1) * 2
    assert bool(((scores - scores[0]).abs() <= size * 4 * 2.0 ** -11).all())
    assert math.isfinite(float(scores[0]))


def test_example(tw, cuda):
    done = subprocess.run([sys.executable, str(REPO / "examples" / "short_cache.py"), "--prompt",
                           "900", "--decode", "90", "--keep", "400", "--chunk", "300"],
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    assert "rows of 990 tokens" in done.stdout


def test_two_caches_at_once(tw, cuda):
    """Two caches on two streams, their kernels side by side: each gets what it gets alone."""
    rotary = tw.RotaryPositions(128, base=10000.0, device=cuda)

    def run(seed, stream):
        g = torch.Generator().manual_seed(seed)
        rows = torch.randn(700, 10, D, generator=g).to(torch.float16).to(cuda)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            cache = make(tw, cuda, num_layers=3, num_pages=120, max_tokens_per_request=800)
            cache.pool.zero_()
            at, outs = 0, []
            for new in ([300, 1], [5, 260], [1, 1], [1, 40]):
                n = sum(new)
                cache.step(new)
                for layer in range(3):
                    q, k, v = rows[at:at + n].split((6, 2, 2), 1)
                    q = cache.write_rotated(layer, q, k, v, rotary)
                    outs.append(cache.attend(layer, q))
                at += n
                cache.evict(160, sink=2, recent=30)
            return cache, outs

    alone = [run(seed, torch.cuda.Stream(cuda)) for seed in (1, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in range(2)]
    for _ in range(3):
        both = [run(seed, s) for seed, s in zip((1, 2), streams)]
        torch.cuda.synchronize()
        for (a, x), (b, y) in zip(alone, both):
            b.synchronize()
            assert all(torch.equal(s, t) for s, t in zip(x, y))
            assert torch.equal(a.row_weights, b.row_weights) and torch.equal(a.pool, b.pool)
            assert torch.equal(a.row_positions, b.row_positions)
            assert a.lengths == b.lengths and a.evicted == b.evicted
