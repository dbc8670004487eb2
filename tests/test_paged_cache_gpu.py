"""PagedKVCache: serving steps over pages against dense attention in 64 bits, pages that
come back, capacity, the hand-over to the offloaded cache, and the example."""

from __future__ import annotations

import random
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import paged_ref

pytestmark = pytest.mark.gpu

REPO = Path(__file__).resolve().parents[1]
D = 128


def make(tw, dev, **kw):
    args = dict(num_layers=2, num_kv_heads=2, num_pages=64, max_requests=4,
                max_tokens_per_request=320, page_size=16, dtype=torch.float16, device=dev)
    return tw.PagedKVCache(**{**args, **kw})


def rows(n, heads, dev, g, dtype=torch.float16):
    return torch.randn(n, heads, D, generator=g).to(dtype).to(dev)


@pytest.mark.parametrize("page_size", [8, 16, 64])
def test_serving_steps(tw, cuda, page_size):
    """Random steps: chunks, single tokens, pauses, ends and new requests in their place."""
    rng = random.Random(page_size)
    g = torch.Generator().manual_seed(page_size)
    cache = make(tw, cuda, page_size=page_size, num_pages=24 * 64 // page_size)
    held = [[], [], [], []]  # per request: (k, v) per layer of all its tokens
    for _ in range(12):
        new = []
        for r in range(4):
            n = rng.choice((0, 1, 1, rng.randint(2, 90)))
            if cache.lengths[r] + n > 300 or (cache.lengths[r] and rng.random() < 0.15):
                n = -1
            new.append(n)
        plan = cache.step(new)
        total = sum(max(0, n) for n in new)
        assert plan.tokens == total == int(plan.cu_q[-1])
        for r, n in enumerate(new):
            held[r] = [] if n < 0 else held[r]
        fresh = [(rows(total, 2, cuda, g), rows(total, 2, cuda, g)) for _ in range(2)]
        cu = plan.cu_q.tolist()
        for r, n in enumerate(new):
            if n > 0:
                held[r].append([(k[cu[r]:cu[r + 1]], v[cu[r]:cu[r + 1]]) for k, v in fresh])
                assert plan.positions[cu[r]:cu[r + 1]].tolist() == \
                    list(range(cache.lengths[r] - n, cache.lengths[r]))
        assert plan.kv_lens.tolist() == cache.lengths
        assert int(cache._free_count[cache._turn]) == cache.free_pages
        for layer, (k, v) in enumerate(fresh):
            cache.write(layer, k, v)
            q = rows(total, 6, cuda, g)
            out = cache.attend(layer, q)
            if total == 0:
                assert out.shape == (0, 6, D)
                continue
            ref, _, tol, _ = paged_ref.attention(q, cache.pool[layer, 0], cache.pool[layer, 1],
                                                 cache.block_table, plan.cu_q, plan.kv_lens)
            assert bool(((out.double() - ref).abs() <= tol).all())
            for r in range(4):
                if held[r]:
                    kk, vv = cache.request_kv(layer, r)
                    assert torch.equal(kk, torch.cat([t[layer][0] for t in held[r]]).transpose(0, 1))
                    assert torch.equal(vv, torch.cat([t[layer][1] for t in held[r]]).transpose(0, 1))
        # no page is held twice
        used = [p for r in range(4)
                for p in cache.block_table[r, :-(-cache.lengths[r] // page_size)].tolist()]
        free = cache._free_pages[:cache.free_pages].tolist()
        assert sorted(used + free) == list(range(cache.num_pages))
    cache.synchronize()


def test_capacity_is_checked_before_anything_changes(tw, cuda):
    cache = make(tw, cuda, num_pages=10)
    cache.step([100, 20])
    before = (list(cache.lengths), cache.free_pages, cache.block_table.clone())
    for new in ([0, 0, 60], [0, 301], [29, 0, 0, 16]):
        with pytest.raises(RuntimeError, match="capacity"):
            cache.step(new)
        assert (cache.lengths, cache.free_pages) == before[:2]
        assert torch.equal(cache.block_table, before[2])
    cache.step([-1, 0, 60])  # the pages of request 0 serve request 2
    assert cache.lengths == [0, 20, 60, 0] and cache.free_pages == 10 - 2 - 4
    cache.synchronize()


def test_a_plan_keeps_its_numbers(tw, cuda):
    """Plans that are held while later steps are planned."""
    cache = make(tw, cuda)
    plans, want = [], []
    for new in ([3, 40], [1, 1, 17], [20, -1, 1], [1, 5, 1, 2], [-1, 1, 0, 30]):
        plans.append(cache.step(new))
        want.append(list(cache.lengths))
    for plan, lengths in zip(plans, want):
        assert plan.kv_lens.tolist() == lengths
        assert int(plan.cu_q[-1]) == plan.tokens == plan.slots.numel() == plan.positions.numel()
    cache.synchronize()


def test_refusals(tw, cuda):
    for bad in (dict(page_size=12), dict(head_dim=64), dict(dtype=torch.float32), dict(num_pages=0),
                dict(device="cpu"), dict(max_requests=9000)):
        with pytest.raises(ValueError):
            make(tw, cuda, **bad)
    cache = make(tw, cuda)
    g = torch.Generator().manual_seed(0)
    with pytest.raises(ValueError):
        cache.write(0, rows(1, 2, cuda, g), rows(1, 2, cuda, g))  # no step yet
    with pytest.raises(ValueError):
        cache.step([1] * 5)
    cache.step([3])
    with pytest.raises(ValueError):
        cache.write(0, rows(2, 2, cuda, g), rows(2, 2, cuda, g))
    with pytest.raises(ValueError):
        cache.attend(0, rows(4, 2, cuda, g))
    with pytest.raises(IndexError):
        cache.attend(2, rows(3, 2, cuda, g))


def test_device_errors_are_raised_by_synchronize(tw, cuda):
    cache = make(tw, cuda)
    g = torch.Generator().manual_seed(0)
    cache.step([3])
    cache.block_table[0, 0] = 1 << 20
    cache.attend(0, rows(3, 4, cuda, g))
    with pytest.raises(ValueError, match="out of bounds"):
        cache.synchronize()
    cache.synchronize()  # raised once


def test_hand_over_to_the_offloaded_cache(tw, cuda):
    layers, G, R, n = 2, 2, 4, 1000
    cache = make(tw, cuda, num_pages=80, max_tokens_per_request=1024)
    g = torch.Generator().manual_seed(5)
    for at in range(0, n, 250):
        cache.step([250])
        for layer in range(layers):
            cache.write(layer, rows(250, G, cuda, g), rows(250, G, cuda, g))
    off = tw.TwilightMatchedBudgetOffloadedCache(
        num_cache_entries=layers * G, max_cache_len=n + 8, head_dim=D, num_query_heads_per_kv=R,
        dtype=torch.float16, device=cuda, sink_tokens=64, recent_tokens=256, block_size=16,
        candidate_token_budget=256, top_p=0.95, budget_mode="dynamic",
        layer_batched_selection=True, gqa_groupwise_execution=True, qk_backend="cuda",
        int4_group_size=32)
    cache.to_offloaded(0, off)
    torch.cuda.synchronize()
    for layer in range(layers):
        k, v = cache.request_kv(layer, 0)
        for h in range(G):
            assert torch.equal(off.entry_kv("key", layer * G + h)[:n].to(cuda), k[h])
            assert torch.equal(off.entry_kv("value", layer * G + h)[:n].to(cuda), v[h])
    off.close()


def test_example_runs(tw, cuda):
    run = subprocess.run([sys.executable, str(REPO / "examples" / "paged_prompts.py"), "--long",
                          "2500"], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    assert "apart" in run.stdout
