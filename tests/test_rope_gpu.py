"""Rotary positions: rows by themselves and with the write to the paged cache, against the
formula in 64 bits; gradients against differences."""

from __future__ import annotations

import pytest
import torch

import evict_ref

pytestmark = pytest.mark.gpu

D = 128
LAYOUTS = ("half", "interleaved")


def normal(g, dev, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g).to(dtype).to(dev)


def within(got, ref, tol):
    return bool(((got.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dims", [0, 2, 10, 16, 36, 64, 80, 126, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows(tw, cuda, layout, dims, dtype):
    g = torch.Generator().manual_seed(dims)
    f, _ = tw.ops.rope_frequencies(dims, base=500000.0, device=cuda)
    for tokens, heads in ((1, 1), (3, 5), (37, 16), (18, 33), (5, 70)):
        x = normal(g, cuda, tokens, heads, D, dtype=dtype)
        pos = torch.randint(0, 1 << 20, (tokens,), generator=g, dtype=torch.int32).to(cuda)
        out = tw.ops.rope(x, pos, f, layout=layout, scale=1.25)
        ref, tol = evict_ref.rope(x, pos, f, layout, 1.25)
        assert within(out, ref, tol)
        assert torch.equal(out[..., dims:], x[..., dims:])


@pytest.mark.parametrize("layout", LAYOUTS)
def test_far_positions(tw, cuda, layout):
    """The angle is reduced in 64 bits: positions up to 2^31, negative ones, and pairs that
    turn by more than a turn a position."""
    g = torch.Generator().manual_seed(5)
    pos = torch.tensor([0, 1, -1, (1 << 24) + 1, 2 ** 31 - 1, -2 ** 31, 999_999_937],
                       dtype=torch.int32, device=cuda)
    x = normal(g, cuda, len(pos), 4, D, dtype=torch.float16)
    f = torch.cat((torch.tensor([7.5, 1.0, 0.3]), torch.rand(61, generator=g) / 100))
    f = f.double().to(cuda)
    ref, tol = evict_ref.rope(x, pos, f, layout)
    assert within(tw.ops.rope(x, pos, f, layout=layout), ref, tol)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dims", [128, 64, 36])
def test_views_and_in_place(tw, cuda, layout, dims):
    """q and k side by side in a projection's output, turned where they lie: nothing else
    changes, and the result is that of the call with another output."""
    g = torch.Generator().manual_seed(dims)
    f, _ = tw.ops.rope_frequencies(dims, device=cuda)
    y = normal(g, cuda, 21, 12, D)
    pos = torch.arange(100, 121, dtype=torch.int32, device=cuda)
    whole = y.clone()
    want = tw.ops.rope(y[:, 1:10], pos, f, layout=layout)
    out = tw.ops.rope(y[:, 1:10], pos, f, layout=layout, out=y[:, 1:10])
    assert out.data_ptr() == y[:, 1:10].data_ptr()
    assert torch.equal(y[:, 1:10], want)
    assert torch.equal(y[:, 0], whole[:, 0]) and torch.equal(y[:, 10:], whole[:, 10:])
    head_first = normal(g, cuda, 9, 21, D).transpose(0, 1)
    assert torch.equal(tw.ops.rope(head_first, pos, f, layout=layout),
                       tw.ops.rope(head_first.contiguous(), pos, f, layout=layout))


@pytest.mark.parametrize("layout", LAYOUTS)
def test_gradient(tw, cuda, layout):
    """inverse is the gradient: that of the formula, and differences along random directions
    (the rotation is linear: a difference is exact but for roundings)."""
    g = torch.Generator().manual_seed(11)
    f, scale = tw.ops.rope_frequencies(96, scaling={"type": "yarn", "factor": 4.0, "original": 64},
                                       device=cuda)
    pos = torch.arange(7, dtype=torch.int32, device=cuda) * 1000
    x, dy = (normal(g, cuda, 7, 3, D, dtype=torch.float16) for _ in range(2))
    dx = tw.ops.rope(dy, pos, f, layout=layout, scale=scale, inverse=True)
    leaf = x.double().requires_grad_()
    n = f.numel()
    i = torch.arange(n, device=cuda)
    a, b = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
    angle = pos.double()[:, None, None] * f
    turned = leaf.clone()
    turned[..., a] = scale * (leaf[..., a] * angle.cos() - leaf[..., b] * angle.sin())
    turned[..., b] = scale * (leaf[..., b] * angle.cos() + leaf[..., a] * angle.sin())
    (turned * dy.double()).sum().backward()
    _, tol = evict_ref.rope(dy, pos, f, layout, scale, inverse=True)
    assert within(dx, leaf.grad, tol)
    step = normal(g, cuda, 7, 3, D, dtype=torch.float16)
    y0, y1 = (tw.ops.rope(z, pos, f, layout=layout, scale=scale).double()
              for z in (x, (x + step)))
    moved = (x + step).double() - x.double()
    _, t0 = evict_ref.rope(x, pos, f, layout, scale)
    _, t1 = evict_ref.rope(x + step, pos, f, layout, scale)
    gap = ((y1 - y0) * dy.double()).sum() - (dx.double() * moved).sum()
    assert gap.abs() <= ((t0 + t1) * dy.double().abs()).sum() + (tol * moved.abs()).sum()


@pytest.mark.parametrize("layout,dims", [("half", 128), ("half", 20), ("interleaved", 64)])
@pytest.mark.parametrize("pool", ["head", "token"])
@pytest.mark.parametrize("tokens,q_heads,kv_heads,page", [(1, 32, 8, 16), (5, 3, 1, 8),
                                                          (70, 14, 2, 24), (33, 6, 6, 64)])
def test_write(tw, cuda, layout, dims, pool, tokens, q_heads, kv_heads, page):
    """q turned, k turned and v as it is at their slots, records of the slots; every other
    place of the pool and the records as it was."""
    g = torch.Generator().manual_seed(tokens + page)
    f, _ = tw.ops.rope_frequencies(dims, device=cuda)
    pages = -(-tokens // page) + 2
    y = normal(g, cuda, tokens, q_heads + 2 * kv_heads, D)
    q, k, v = y.split((q_heads, kv_heads, kv_heads), 1)
    make = lambda: (normal(g, cuda, pages, kv_heads, page, D) if pool == "head"  # noqa: E731
                    else normal(g, cuda, pages, page, kv_heads, D).transpose(1, 2))
    kp, vp = make(), make()
    k0, v0 = kp.clone(), vp.clone()
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(cuda)
    if tokens > 2:
        slots[1] = -1
    pos = torch.randint(0, 100000, (tokens,), generator=g, dtype=torch.int32).to(cuda)
    w = torch.full((pages, kv_heads, page), 3.0, device=cuda)
    p = torch.full((pages, kv_heads, page), -5, dtype=torch.int32, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    before = y.clone()
    out = tw.ops.paged_rope_write(q, k, v, pos, slots, f, kp, vp, layout=layout, row_weights=w,
                                  row_positions=p, error_flag=err)
    assert torch.equal(y, before)
    assert torch.equal(out, tw.ops.rope(q, pos, f, layout=layout))
    ref, tol = evict_ref.rope(q, pos, f, layout)
    assert within(out, ref, tol)
    turned = tw.ops.rope(k, pos, f, layout=layout)
    wanted_w, wanted_p = torch.full_like(w, 3.0), torch.full_like(p, -5)
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            k0[s // page, :, s % page] = turned[t]
            v0[s // page, :, s % page] = v[t]
            wanted_w[s // page, :, s % page] = 0.0
            wanted_p[s // page, :, s % page] = pos[t]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)
    assert torch.equal(w, wanted_w) and torch.equal(p, wanted_p)
    assert int(err) == 0
    # q in place, no records
    tw.ops.paged_rope_write(q, k, v, pos, slots, f, kp, vp, layout=layout, q_out=q)
    assert torch.equal(y[:, :q_heads], out) and torch.equal(y[:, q_heads:], before[:, q_heads:])


def test_write_flags_bad_slots(tw, cuda):
    g = torch.Generator().manual_seed(1)
    f, _ = tw.ops.rope_frequencies(128, device=cuda)
    q, k, v = (normal(g, cuda, 4, h, D) for h in (4, 2, 2))
    kp, vp = (torch.zeros(3, 2, 16, D, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    pos = torch.arange(4, dtype=torch.int32, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    slots = torch.tensor([0, 48, 1 << 40, -7], device=cuda)
    out = tw.ops.paged_rope_write(q, k, v, pos, slots, f, kp, vp, error_flag=err)
    assert int(err) == tw._lib.TW_ERR_INVALID_INDEX
    assert torch.equal(out, tw.ops.rope(q, pos, f))
    assert bool((vp[0, :, 0] == v[0]).all())
    vp[0, :, 0] = 0
    assert not bool(vp.any())


def test_no_rows(tw, cuda):
    f, _ = tw.ops.rope_frequencies(128, device=cuda)
    none = torch.empty(0, dtype=torch.int32, device=cuda)
    x = torch.empty(0, 4, D, dtype=torch.float16, device=cuda)
    assert tw.ops.rope(x, none, f).shape == (0, 4, D)
    pages = torch.zeros(1, 2, 16, D, dtype=torch.float16, device=cuda)
    assert tw.ops.paged_rope_write(x, x[:, :2], x[:, :2], none, none.long(), f, pages,
                                   pages.clone()).shape == (0, 4, D)
    one = torch.zeros(1, dtype=torch.int32, device=cuda)
    no_q = torch.empty(1, 0, D, dtype=torch.float16, device=cuda)
    k = torch.ones(1, 2, D, dtype=torch.float16, device=cuda)
    tw.ops.paged_rope_write(no_q, k, k, one, one.long(), f, pages, pages)  # k and v only
    assert bool((pages[0, :, 0] == 1).all())


def test_refusals(tw, cuda):
    ops = tw.ops
    f, _ = ops.rope_frequencies(128, device=cuda)
    x = torch.zeros(3, 4, D, dtype=torch.float16, device=cuda)
    pos = torch.zeros(3, dtype=torch.int32, device=cuda)
    for bad in (dict(x=x[..., :64]), dict(x=x.float()), dict(x=x[0]), dict(positions=pos[:2]),
                dict(positions=pos.long()), dict(frequencies=f.float()),
                dict(frequencies=torch.ones(65, dtype=torch.float64, device=cuda)),
                dict(frequencies=f.cpu()), dict(scale=float("nan")), dict(out=x[:2]),
                dict(out=x.bfloat16()), dict(x=x[..., 0:1].expand(3, 4, D)),
                dict(x=torch.zeros(3, 4 * D + 8, dtype=torch.float16, device=cuda)[:, 4:4 + 4 * D]
                     .view(3, 4, D))):
        args = {**dict(x=x, positions=pos, frequencies=f), **bad}
        with pytest.raises(ValueError):
            ops.rope(args.pop("x"), args.pop("positions"), args.pop("frequencies"), **args)
    pages = torch.zeros(2, 2, 16, D, dtype=torch.float16, device=cuda)
    k = torch.zeros(3, 2, D, dtype=torch.float16, device=cuda)
    good = dict(q=x, k=k, v=k, positions=pos, slots=pos.long() - 1, frequencies=f, k_pages=pages,
                v_pages=pages)
    w = torch.zeros(2, 2, 16, device=cuda)
    for bad in (dict(k=x), dict(v=k[:2]), dict(q=x.bfloat16()), dict(slots=pos),
                dict(positions=pos[:1]), dict(k_pages=pages[:1]), dict(q_out=x[:, :2]),
                dict(row_weights=w.int()), dict(row_weights=w[:1]),
                dict(row_weights=w.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(row_positions=w), dict(layout="both"), dict(error_flag=w)):
        with pytest.raises(ValueError):
            ops.paged_rope_write(**{**good, **bad})
    ops.paged_rope_write(**good)


def test_streams_and_graph(tw, cuda):
    """On another stream than the tensors' own, and replayed from a graph on new values."""
    g = torch.Generator().manual_seed(3)
    f, _ = tw.ops.rope_frequencies(64, device=cuda)
    x = normal(g, cuda, 40, 8, D)
    pos = torch.arange(40, dtype=torch.int32, device=cuda)
    want = tw.ops.rope(x, pos, f)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        got = tw.ops.rope(x, pos, f)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tw.ops.rope(x, pos, f, out=out)
    x.copy_(normal(g, cuda, 40, 8, D))
    pos.add_(7)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, tw.ops.rope(x, pos, f))
