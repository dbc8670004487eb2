"""A long conversation in a cache that is kept short: rotary positions, accumulated attention
weights, eviction.

    python examples/short_cache.py [--prompt 3000] [--decode 300] [--keep 1024]

A stack of attention layers with random weights reads a prompt in chunks and decodes.  Two
caches serve it: one that holds all rows, and one that is cut to `keep` rows per layer and
head whenever it has grown 64 beyond that.  A few keys of the prompt draw most of the
attention; the script shows how many of them the short cache still holds, how far its
outputs are from the full one's, and how many pages it gave back.
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
SLACK = 64


class Stack:
    def __init__(self, dev: torch.device, dtype: torch.dtype) -> None:
        g = torch.Generator(dev).manual_seed(1)
        rows = (Q_HEADS + 2 * KV_HEADS) * D
        self.w_qkv = [(torch.randn(rows, HIDDEN, generator=g, device=dev) / HIDDEN ** 0.5).to(dtype)
                      for _ in range(LAYERS)]
        self.w_out = [(torch.randn(HIDDEN, Q_HEADS * D, generator=g, device=dev)
                       / (Q_HEADS * D) ** 0.5).to(dtype) for _ in range(LAYERS)]
        # slow pairs only: what the tokens say counts more than where they are
        self.rotary = tw.RotaryPositions(64, base=500000.0, layout="interleaved", device=dev,
                                         scaling={"type": "linear", "factor": 64.0})

    def step(self, cache, x: torch.Tensor, **kw) -> torch.Tensor:
        for layer in range(LAYERS):
            y = (x @ self.w_qkv[layer].T).view(-1, Q_HEADS + 2 * KV_HEADS, D)
            q, k, v = y.split((Q_HEADS, KV_HEADS, KV_HEADS), 1)
            q = cache.write_rotated(layer, q, k, v, self.rotary)
            x = x + cache.attend(layer, q, **kw).flatten(1) @ self.w_out[layer].T
        return x


def serve(stack: Stack, prompt: torch.Tensor, decode: int, chunk: int, keep: int | None):
    """The cache at the end and the outputs of the decoded tokens."""
    cache = tw.PagedKVCache(num_layers=LAYERS, num_kv_heads=KV_HEADS, max_requests=1,
                            num_pages=-(-(len(prompt) + decode) // 16),
                            max_tokens_per_request=len(prompt) + decode, dtype=prompt.dtype,
                            device=prompt.device, track_weights=keep is not None)
    out, kw = [], {}
    for i in range(0, len(prompt), chunk):
        rows = prompt[i:i + chunk]
        cache.step([len(rows)])
        if keep is not None and i + chunk < len(prompt):
            kw = dict(last=64)  # the end of a chunk says what its rows look for
        x = stack.step(cache, rows, **kw)
        if keep is not None:
            cache.evict(keep, sink=4, recent=min(256, keep // 4))
    for _ in range(decode):
        x = x[-1:] / x[-1:].float().pow(2).mean().sqrt().to(x.dtype)
        plan = cache.step([1])
        x = stack.step(cache, x)
        out.append(x)
        if keep is not None and cache.lengths[0] >= keep + SLACK:
            cache.evict(keep, sink=4, recent=min(256, keep // 4))
    cache.synchronize()
    assert int(plan.positions) == len(prompt) + decode - 1
    return cache, torch.cat(out)


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--prompt", type=int, default=3000)
    ap.add_argument("--decode", type=int, default=300)
    ap.add_argument("--keep", type=int, default=1024)
    ap.add_argument("--chunk", type=int, default=512)
    args = ap.parse_args()
    dev, dtype = torch.device("cuda", torch.cuda.current_device()), torch.bfloat16
    g = torch.Generator(dev).manual_seed(2)
    common = torch.randn(HIDDEN, generator=g, device=dev)
    prompt = torch.randn(args.prompt, HIDDEN, generator=g, device=dev)
    loud = torch.randperm(args.prompt, generator=g, device=dev)[:32]
    prompt[loud] = 3 * prompt[loud] + 2 * common  # what draws attention
    prompt = (prompt + 0.5 * common).to(dtype)
    stack = Stack(dev, dtype)
    full, dense = serve(stack, prompt, args.decode, args.chunk, None)
    short, cut = serve(stack, prompt, args.decode, args.chunk, args.keep)
    gap = (dense - cut).float().norm() / dense.float().norm()
    held = [torch.isin(loud, short.request_positions(layer, 0)[h]).float().mean().item()
            for layer in range(LAYERS) for h in range(KV_HEADS)]
    print(f"{short.lengths[0]} rows of {full.lengths[0]} tokens held; of the {len(loud)} loud "
          f"ones {100 * min(held):.0f} to {100 * max(held):.0f} % in a head; outputs "
          f"{gap.item():.2f} apart; pages free: {short.free_pages} against {full.free_pages}")
    return 0 if short.lengths[0] < args.keep + SLACK else 1


if __name__ == "__main__":
    sys.exit(main())
