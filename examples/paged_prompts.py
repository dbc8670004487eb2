"""Prompts in chunks over a paged cache, then decoding: dense for short requests,
sparse and offloaded for the long one.

    python examples/paged_prompts.py [--long 6000] [--chunk 512]

A stack of attention layers with random weights serves three prompts.  Each step
takes a chunk of the prompts that are still being read and one token of those that
are done.  Then the longest request moves to the offloaded cache
(TwilightMatchedBudgetOffloadedCache), which decodes it sparsely, while the others go on
over their pages.  The script checks that chunks give what whole prompts give, and
how far the sparse decode is from the dense one.
"""

from __future__ import annotations

import argparse
import importlib
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
tw = importlib.import_module("twilight-cpu-gpu-offloading_b200")

LAYERS, HIDDEN, Q_HEADS, KV_HEADS, D = 2, 1024, 8, 2, 128


class Stack:
    """Attention layers with random weights, rotary positions."""

    def __init__(self, dev: torch.device, dtype: torch.dtype) -> None:
        g = torch.Generator(dev).manual_seed(1)
        rows = (Q_HEADS + 2 * KV_HEADS) * D
        self.w_qkv = [(torch.randn(rows, HIDDEN, generator=g, device=dev) / HIDDEN ** 0.5).to(dtype)
                      for _ in range(LAYERS)]
        self.w_out = [(torch.randn(HIDDEN, Q_HEADS * D, generator=g, device=dev)
                       / (Q_HEADS * D) ** 0.5).to(dtype) for _ in range(LAYERS)]
        self.rotary = tw.RotaryPositions(D, base=500000.0, device=dev)

    def qkv(self, layer: int, x: torch.Tensor, positions: torch.Tensor):
        """q, k (rotated) and v, views of one projection."""
        y = (x @ self.w_qkv[layer].T).view(-1, Q_HEADS + 2 * KV_HEADS, D)
        self.rotary(y[:, :-KV_HEADS], positions, out=y[:, :-KV_HEADS])
        return y[:, :Q_HEADS], y[:, Q_HEADS:-KV_HEADS], y[:, -KV_HEADS:]

    def step(self, cache, plan, x: torch.Tensor) -> torch.Tensor:
        for layer in range(LAYERS):
            q, k, v = self.qkv(layer, x, plan.positions)
            cache.write(layer, k, v)
            x = x + cache.attend(layer, q).flatten(1) @ self.w_out[layer].T
        return x


def serve(stack: Stack, prompts: list[torch.Tensor], chunk: int, decode: int):
    """All prompts in chunks, then `decode` tokens of each (its own last output, at unit
    size); returns the cache and the outputs of each request."""
    dev, dtype = prompts[0].device, prompts[0].dtype
    n = len(prompts)
    most = max(len(p) for p in prompts) + decode
    cache = tw.PagedKVCache(num_layers=LAYERS, num_kv_heads=KV_HEADS, max_requests=n,
                            num_pages=sum(-(-(len(p) + decode) // 16) for p in prompts),
                            max_tokens_per_request=most, dtype=dtype, device=dev)
    done = [0] * n
    outputs: list[list[torch.Tensor]] = [[] for _ in range(n)]
    while any(d < len(p) + decode for d, p in zip(done, prompts)):
        rows, new = [], []
        for r, p in enumerate(prompts):
            if done[r] < len(p):
                rows.append(p[done[r]:done[r] + chunk])
            elif done[r] < len(p) + decode:
                last = outputs[r][-1][-1:]
                rows.append(last / last.float().pow(2).mean().sqrt().to(dtype))
            else:
                rows.append(p[:0])
            new.append(len(rows[-1]))
        plan = cache.step(new)
        for r, y in enumerate(stack.step(cache, plan, torch.cat(rows)).split(new)):
            outputs[r].append(y)
            done[r] += new[r]
    cache.synchronize()
    return cache, [torch.cat(o) for o in outputs]


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--long", type=int, default=6000, help="tokens of the longest prompt")
    ap.add_argument("--chunk", type=int, default=512)
    args = ap.parse_args()
    dev, dtype = torch.device("cuda", torch.cuda.current_device()), torch.bfloat16
    g = torch.Generator(dev).manual_seed(2)
    prompts = [torch.randn(n, HIDDEN, generator=g, device=dev).to(dtype)
               for n in (args.long, 700, 45)]
    stack = Stack(dev, dtype)

    cache, chunked = serve(stack, prompts, args.chunk, decode=4)
    _, whole = serve(stack, prompts, 10 ** 9, decode=4)
    apart = max((a - b).float().norm().item() / b.float().norm().item()
                for a, b in zip(chunked, whole))
    print(f"chunks of {args.chunk} against whole prompts: {apart:.1e} apart")

    # the long request decodes one more token, sparsely from the offloaded cache
    long = cache.lengths[0]
    offloaded = tw.TwilightMatchedBudgetOffloadedCache(
        num_cache_entries=LAYERS * KV_HEADS, max_cache_len=long + 8, head_dim=D,
        num_query_heads_per_kv=Q_HEADS // KV_HEADS, dtype=dtype, device=dev, sink_tokens=64,
        recent_tokens=256, block_size=16, candidate_token_budget=min(4096, long // 32 * 16),
        top_p=0.95, budget_mode="dynamic", layer_batched_selection=True,
        gqa_groupwise_execution=True, qk_backend="cuda", int4_group_size=32)
    cache.to_offloaded(0, offloaded)
    x = torch.randn(1, HIDDEN, generator=g, device=dev).to(dtype)
    position = torch.full((1,), long, dtype=torch.int32, device=dev)
    q, k, v = stack.qkv(0, x, position)
    sparse = offloaded.decode_layer(queries=q.reshape(KV_HEADS, -1, D).contiguous(),
                                    key_states=k[0].contiguous(), value_states=v[0].contiguous(),
                                    entries=list(range(KV_HEADS)))
    # ... and densely over its pages; the others end, their pages are free
    cache.step([1, -1, -1])
    cache.write(0, k, v)
    dense = cache.attend(0, q)
    cache.synchronize()
    torch.cuda.synchronize()
    gap = (sparse.reshape(-1) - dense.reshape(-1)).float().norm() / dense.float().norm()
    print(f"one more token of the {long}-token request: sparse and dense {gap.item():.2f} apart; "
          f"{cache.free_pages} pages free")
    offloaded.close()
    return 0 if apart < 0.02 else 1


if __name__ == "__main__":
    sys.exit(main())
