"""Paged attention at its edges: what may not reach a result, what a call must not cost, what
its buffers do not hold."""

from __future__ import annotations

import math

import pytest
import torch

import paged_ref
from test_paged_gpu import Batch, D, put

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


# -------------------------------------------------- values not finite in V --

def spoil(b, request, keys, value, dims=slice(5, 7)):
    page = b.v_pages.shape[2]
    for j in keys:
        b.v_pages[b.table[request, j // page].long(), :, j % page, dims] = value


def device_ms(call):
    call()
    best = math.inf
    for _ in range(3):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        call()
        end.record()
        end.synchronize()
        best = min(best, begin.elapsed_time(end))
    return best


@pytest.mark.parametrize("new,kv,window", [([256], [3000], 0), ([3, 1], [3000, 40], 0),
                                           ([256], [3000], 1500)])
@pytest.mark.parametrize("where", ["seen by all", "seen by some", "both", "everywhere"])
def test_values_not_finite_cost_little(tw, cuda, new, kv, window, where):
    """A call whose V holds NaN takes about as long as a clean one: at most ten times (rows
    of the few keys in question are looked at once more), not a pass per row."""
    b = Batch(cuda, new, kv, q_heads=8, kv_heads=2, page=16, dtype=torch.bfloat16)
    call = lambda: b.run(tw, window=window)  # noqa: E731
    clean = device_ms(call)
    early, late = kv[0] - new[0] - 9, kv[0] - 1
    spoil(b, 0, {"seen by all": [early], "seen by some": [late], "both": [early, late],
                 "everywhere": range(kv[0])}[where], math.nan)
    assert device_ms(call) < 10 * clean + 0.05
    out, lse, error = b.run(tw, window=window)
    assert error == 0
    b.check(out, lse, window=window)


@pytest.mark.parametrize("heads", [(8, 2), (6, 2), (2, 2), (64, 1)])
@pytest.mark.parametrize("window", [0, 1, 20, 150])
@pytest.mark.parametrize("new,kv", [([100, 3, 1], [190, 64, 120]), ([4], [4]), ([2, 4], [900, 5]),
                                    ([290], [1600])])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_infinities_and_nan_reach_the_rows_that_see_them(tw, cuda, heads, window, new, kv, dtype):
    """Signed infinities and NaN in some dimensions of V, seen by some rows of a request and
    hidden from others: each result is what the sum over the visible keys gives."""
    b = Batch(cuda, new, kv, q_heads=heads[0], kv_heads=heads[1], page=16, dtype=dtype, seed=7)
    marks = []
    for r, (n, m) in enumerate(zip(new, kv)):
        for at, value, dim in ((m - 1, math.inf, 3), (m - n // 2 - 1, -math.inf, 3),
                               (m - n, math.nan, 64), (max(0, m - n - 5), -math.inf, 127),
                               (max(0, m - n - window), math.inf, 40), (m - 2, math.nan, 0)):
            if at >= 0:
                spoil(b, r, [at], value, dim)
                marks.append((r, at, value, dim))
    out, lse, error = b.run(tw, window=window, out_dtype=torch.float32)
    assert error == 0
    b.check(out, lse, window=window)
    # which of them: with weights above zero the sum is the first infinity, NaN, or
    # NaN where both signs meet
    for r, (n, m) in enumerate(zip(new, kv)):
        first = int(b.cu[r])
        for i in range(n):
            p = m - n + i
            want = {}
            held = {(at, dim): value for q, at, value, dim in marks if q == r}  # the last one put
            for (at, dim), value in held.items():
                if at <= p and (not window or at > p - window):
                    want[dim] = want.get(dim, 0.0) + value
            for dim, value in want.items():
                got = out[first + i, :, dim]
                same = torch.isnan(got) if math.isnan(value) else got == value
                assert bool(same.all()), (r, i, dim, value)


# ------------------------------------------------------------ small weights --

@pytest.mark.parametrize("new,kv", [([1], [256]), ([64], [760])])
def test_small_fp16_weights_count(tw, cuda, new, kv):
    """One key of weight 1, all others of 2^-25.5 with large values: the others' share of the
    sum is not lost in the 16-bit weights.

    Tolerance: weights and V in 16 bits, 32-bit sums.  Weights are rounded relative to
    themselves (unit 2^-11) or, below the smallest normal value, by at most 2^-25 of the
    type, which is 2^-32 of the row's largest where that one stands at 2^7."""
    n = kv[0]
    b = Batch(cuda, new, kv, q_heads=4, kv_heads=1, page=16, dtype=torch.float16)
    rows = torch.zeros(n, 1, D, dtype=torch.float16, device=cuda)
    rows[0, 0, 0] = 17.6875  # 25.52 in log2 units
    put(b.k_pages, b.table[0], rows)
    values = torch.full((n, 1, D), 30000.0, dtype=torch.float16, device=cuda)
    values[0] = 1.0
    put(b.v_pages, b.table[0], values)
    b.q.zero_()
    b.q[..., 0] = 1.0
    out, lse, error = b.run(tw, softmax_scale=1.0, out_dtype=torch.float32)
    assert error == 0
    seen = (n - new[0] + 1 + torch.arange(new[0], device=cuda)).double()[:, None, None]
    small = math.exp(-17.6875)
    total = 1.0 + (seen - 1) * small
    ref = (1.0 + (seen - 1) * small * 30000.0) / total
    tol = 2.0 ** -11 * ref + (seen - 1) * 2.0 ** -32 * 30000.0 + 2.0 ** -18 * ref
    assert bool(((out.double() - ref).abs() <= tol).all()), \
        float(((out.double() - ref).abs() / tol).max())
    ref_lse = 17.6875 + torch.log(total[..., 0])
    assert bool(((lse.double() - ref_lse).abs() <= 2.0 ** -18).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [1e3, 1e5, 1e6, 1e7, 4e7, 1e8, 3e9, 1e30])
@pytest.mark.parametrize("new,kv", [([1], [200]), ([70], [400]), ([300], [2000])])
def test_large_scores(tw, cuda, dtype, size, new, kv):
    """Scores so large that their rounding moves an exponent by more than the types' range:
    a row whose largest score stands out by more than the scores' own error is the V row of
    that key, and any other row lies among the values it sees."""
    b = Batch(cuda, new, kv, q_heads=4, kv_heads=1, page=16, dtype=dtype)
    out, lse, error = b.run(tw, softmax_scale=size)
    assert error == 0
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    j = torch.arange(kv[0], device=cuda)
    rows = [pages[b.table[0, j // 16].long(), 0, j % 16].double() for pages in (b.k_pages,
                                                                                b.v_pages)]
    score = torch.einsum("thd,kd->thk", b.q.double(), rows[0]) * size
    seen = j <= kv[0] - new[0] + torch.arange(new[0], device=cuda)[:, None]
    score.masked_fill_(~seen[:, None], -math.inf)
    best = score.topk(2, -1)
    # as in paged_ref: a score's error in 32 bits, twice, and 40 for the others to vanish
    slack = 260 * 2.0 ** -24 * (b.q.double().abs() @ rows[0].abs().T).amax(-1) * size + 40
    alone = best.values[..., 0] - best.values[..., 1] > slack
    assert size < 1e6 or bool(alone.any())
    want = rows[1][best.indices[..., 0]]
    unit = paged_ref.UNIT[dtype]
    assert bool(((out.double() - want).abs() <= 2 * unit * want.abs())[alone].all())
    low, high = rows[1].amin(0), rows[1].amax(0)
    assert bool((out.double() >= low - 2 * unit * low.abs()).all())
    assert bool((out.double() <= high + 2 * unit * high.abs()).all())
    # lse: the largest score, but for log(keys)
    top = best.values[..., 0]
    assert bool(((lse.double() - top).abs() <= math.log(kv[0]) + slack).all())


# ------------------------------------------------------------------ lengths --

def test_a_bound_of_no_tokens_is_kept_to(tw, cuda):
    """max_q_len 0: a request with one token is longer than that."""
    b = Batch(cuda, [1, 0], [20, 30], q_heads=8, kv_heads=2, page=16, dtype=torch.float16)
    out = torch.full_like(b.q, 5.0)
    _, _, error = b.run(tw, max_q_len=0, out=out)
    assert error == tw._lib.TW_ERR_BAD_ARG
    assert bool((out == 5.0).all())
    b = Batch(cuda, [0, 0], [20, 30], q_heads=8, kv_heads=2, page=16, dtype=torch.float16)
    b.q = torch.zeros(3, 8, D, dtype=torch.float16, device=cuda)  # padding only
    out, _, error = b.run(tw)
    assert error == 0 and bool((out == 0).all())


@pytest.mark.parametrize("new,kv", [([1, 1, 3], [40, 50, 60]), ([40, 70], [50, 200]),
                                    ([40, 5], [50, 200]), ([300], [300])])
def test_requests_beyond_the_rows_of_q_are_flagged(tw, cuda, new, kv):
    """cu_q promises more rows than q has: that request is not computed (its positions would
    be wrong), the others are."""
    b = Batch(cuda, new, kv, q_heads=8, kv_heads=2, page=16, dtype=torch.bfloat16)
    good, _, error = b.run(tw)
    assert error == 0
    q = b.q[:-2].contiguous()
    out = torch.full_like(q, 5.0)
    _, _, error = b.run(tw, q=q, out=out)
    assert error == tw._lib.TW_ERR_BAD_ARG
    first = int(b.cu[-2])
    assert torch.equal(out[:first], good[:first])
    assert bool((out[first:] == 5.0).all())


@pytest.mark.parametrize("new", [1, 200])
def test_lengths_beyond_2_30_are_cut_and_flagged(tw, cuda, new):
    """Pages may be shared, so that a table can hold more positions than 32 bits count."""
    page, window = 1 << 20, 100
    b = Batch(cuda, [new], [1], q_heads=8, kv_heads=1, page=8, dtype=torch.bfloat16)
    g = torch.Generator(cuda).manual_seed(3)
    b.k_pages, b.v_pages = (torch.randn(1, 1, page, D, generator=g, device=cuda).to(torch.bfloat16)
                            for _ in range(2))
    b.table = torch.zeros(1, 2049, dtype=torch.int32, device=cuda)
    results = []
    for length in (1 << 30, (1 << 30) + 1, 2 ** 31 - 1):
        b.kv.fill_(length)
        out, lse, error = b.run(tw, window=window, max_kv_len=1 << 30)
        assert error == (tw._lib.TW_ERR_INVALID_INDEX if length > 1 << 30 else 0)
        results.append((out, lse))
    for out, lse in results[1:]:
        assert torch.equal(out, results[0][0]) and torch.equal(lse, results[0][1])
    # the same keys in a table of one page
    b.table, b.max_kv = b.table[:, :1].contiguous(), page
    b.kv.fill_(page)
    out, lse, error = b.run(tw, window=window)
    assert error == 0
    assert torch.equal(out, results[0][0]) and torch.equal(lse, results[0][1])


# ------------------------------------------------------- workspace and order --

def test_one_long_request_among_many(tw, cuda):
    """More partial results than the workspace's bound holds at the usual range length."""
    requests = 700
    new, kv = [1] * requests, [3] * requests
    new[1], kv[350], new[350] = 4, 70000, 4
    kv[1] = 4
    b = Batch(cuda, new, kv, q_heads=32, kv_heads=8, page=128, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    out, lse, error = b.run(tw)
    assert error == 0
    first = int(b.cu[350])
    for r, at, n in ((350, first, 4), (1, int(b.cu[1]), 4), (699, int(b.cu[699]), 1)):
        o, z, tol, tol_z = paged_ref.attention(
            b.q[at:at + n], b.k_pages, b.v_pages, b.table[r:r + 1],
            torch.tensor([0, n], device=cuda), b.kv[r:r + 1])
        assert bool(((out[at:at + n].double() - o).abs() <= tol).all())
        assert bool(((lse[at:at + n].double() - z).abs() <= tol_z).all())


def test_large_workspaces_go_back_to_the_allocator(tw, cuda):
    """What a call takes for itself and is large is not kept once it has been used."""
    b = Batch(cuda, [4] + [1] * 299, [70000] + [3] * 299, q_heads=32, kv_heads=8, page=128,
              dtype=torch.bfloat16)
    need = tw.ops.paged_attention_workspace_bytes(300, b.q.shape[0], 32, 8, 4, 70000)
    assert need > 1 << 27
    out = torch.empty_like(b.q)
    call = lambda: tw.ops.paged_attention(  # noqa: E731
        b.q, b.k_pages, b.v_pages, b.table, b.cu, b.kv, max_q_len=4, max_kv_len=70000, out=out)
    before = torch.cuda.memory_allocated()
    call()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before < 1 << 27


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
