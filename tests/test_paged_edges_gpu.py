"""Paged attention at its edges: what may not reach a result, what a call must not cost, what
its buffers do not hold."""

from __future__ import annotations

import pytest
import torch

from test_paged_gpu import Batch, D

pytestmark = pytest.mark.gpu


# ------------------------------------------------------- workspace and order --

def test_inputs_that_the_kernel_before_writes(tw, cuda):
    """Chunks and single tokens in one call, right behind the kernels that write its rows of
    K and V, its table and its lengths."""
    new, kv = [200, 1, 1, 90, 1, 1, 1, 30], [1500, 900, 40, 90, 700, 1, 333, 30]
    b = Batch(cuda, new, kv, q_heads=8, kv_heads=2, page=16, dtype=torch.bfloat16)
    rows = sum(kv)
    g = torch.Generator().manual_seed(11)
    slots = torch.cat([b.table[r, torch.arange(n, device=cuda) // 16].long() * 16
                       + torch.arange(n, device=cuda) % 16 for r, n in enumerate(kv)])
    keep_table, keep_kv, keep_cu = b.table.clone(), b.kv.clone(), b.cu.clone()
    calls = []
    for turn in range(6):
        k, v = (torch.randn(rows, 2, D, generator=g).to(torch.bfloat16).to(cuda) for _ in range(2))
        b.q = torch.randn(b.q.shape, generator=g).to(torch.bfloat16).to(cuda)
        out, lse = torch.empty_like(b.q), torch.empty(b.q.shape[:2], device=cuda)
        b.table.fill_(-1), b.kv.zero_(), b.cu.zero_()
        torch.cuda.synchronize()
        b.table.copy_(keep_table), b.kv.copy_(keep_kv), b.cu.copy_(keep_cu)
        tw.ops.paged_write(k, v, slots, b.k_pages, b.v_pages)
        tw.ops.paged_attention(b.q, b.k_pages, b.v_pages, b.table, b.cu, b.kv, max_q_len=200,
                               max_kv_len=1500, out=out, lse=lse)
        b.check(out, lse)
        calls.append(out)
    assert not torch.equal(calls[0], calls[1])
