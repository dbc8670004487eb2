"""Paged attention at its edges: what may not reach a result, what a call must not cost, what
its buffers do not hold."""

from __future__ import annotations

import math

import pytest
import torch

from test_paged_gpu import Batch, D

pytestmark = pytest.mark.gpu


def alike(a, b):
    """The same bits (NaN included)."""
    return torch.equal(a.view(torch.int32), b.view(torch.int32))


# ---------------------------------------------------------- the same bits --

@pytest.mark.parametrize("heads", [(8, 2), (6, 2), (14, 2), (5, 1)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_bits_do_not_depend_on_rows_after_the_request(tw, cuda, heads, dtype):
    b = Batch(cuda, [50], [700], q_heads=heads[0], kv_heads=heads[1], page=16, dtype=dtype)
    first = None
    for fill in (0.0, math.nan, math.inf, 1e4):
        after = torch.full((77, heads[0], D), fill, dtype=dtype, device=cuda)
        out, lse, error = b.run(tw, q=torch.cat((b.q, after)), out_dtype=torch.float32)
        assert error == 0
        if first is None:
            first = out[:50].clone(), lse[:50].clone()
        assert alike(out[:50], first[0]) and alike(lse[:50], first[1]), fill


@pytest.mark.parametrize("heads", [(6, 2), (14, 2), (5, 1), (24, 8)])
def test_bits_do_not_depend_on_the_calls_before(tw, cuda, heads):
    """What earlier kernels left in shared memory stays out of the arithmetic."""
    b = Batch(cuda, [300], [900], q_heads=heads[0], kv_heads=heads[1], page=16,
              dtype=torch.bfloat16)
    filler = Batch(cuda, [2048], [2048], q_heads=32, kv_heads=8, page=64, dtype=torch.bfloat16)
    first = None
    for fill in (0.0, math.nan, math.inf, 3e38):
        filler.q.fill_(fill)
        filler.run(tw)
        out, lse, error = b.run(tw, out_dtype=torch.float32)
        assert error == 0
        if first is None:
            first = out.clone(), lse.clone()
        assert alike(out, first[0]) and alike(lse, first[1]), fill


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
