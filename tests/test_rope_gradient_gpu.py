"""Rotary positions under autograd: gradients through ops.rope, and what is refused instead of
losing one."""

from __future__ import annotations

import pytest
import torch

import evict_ref

pytestmark = pytest.mark.gpu

D = 128
LAYOUTS = ("half", "interleaved")


def normal(g, dev, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g).to(dtype).to(dev)


def setting(tw, dev, tokens, dims=128):
    f, scale = tw.ops.rope_frequencies(dims, scaling={"type": "yarn", "factor": 4.0,
                                                      "original": 64}, device=dev)
    return torch.arange(tokens, dtype=torch.int32, device=dev) * 911, f, scale


def within(got, ref, tol):
    return bool(((got.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("layout,dims", [("half", 128), ("half", 36), ("interleaved", 64),
                                         ("half", 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_backward(tw, cuda, layout, dims, dtype, inverse):
    """backward() gives the gradient of the formula: the turn by the other angle."""
    g = torch.Generator().manual_seed(dims)
    for tokens, heads in ((1, 1), (7, 3), (33, 12)):
        pos, f, scale = setting(tw, cuda, tokens, dims)
        x, dy = (normal(g, cuda, tokens, heads, D, dtype=dtype) for _ in range(2))
        how = dict(layout=layout, scale=scale, inverse=inverse)
        want = tw.ops.rope(x, pos, f, **how)
        leaf = x.clone().requires_grad_()
        y = tw.ops.rope(leaf, pos, f, **how)
        assert torch.equal(y.detach(), want)
        y.backward(dy)
        ref, tol = evict_ref.rope(dy, pos, f, layout, scale, inverse=not inverse)
        assert within(leaf.grad, ref, tol)


def test_gradients_as_they_come(tw, cuda):
    """Incoming gradients with strides of 0, transposed, and off 16 bytes."""
    g = torch.Generator().manual_seed(1)
    pos, f, _ = setting(tw, cuda, 9)
    x = normal(g, cuda, 9, 4, D).requires_grad_()
    y = tw.ops.rope(x, pos, f)
    ones = torch.ones_like(x)
    got, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(got, tw.ops.rope(ones, pos, f, inverse=True))
    for dy in (normal(g, cuda, 4, 9, D).transpose(0, 1),
               normal(g, cuda, 9, 4, 2 * D)[..., ::2],
               normal(g, cuda, 9 * 4 * D + 1)[1:].view(9, 4, D)):
        got, = torch.autograd.grad(tw.ops.rope(x, pos, f), x, dy)
        assert torch.equal(got, tw.ops.rope(dy.contiguous().clone(), pos, f, inverse=True))


def test_projection(tw, cuda):
    """q and k side by side in a projection's output, v beside them: each part its own."""
    g = torch.Generator().manual_seed(2)
    pos, f, scale = setting(tw, cuda, 21)
    rotary = tw.RotaryPositions(128, scaling={"type": "yarn", "factor": 4.0, "original": 64},
                                device=cuda)
    y = normal(g, cuda, 21, 10, D).requires_grad_()
    q, k, v = y.split((6, 2, 2), 1)
    dq, dk, dv = normal(g, cuda, 21, 10, D).split((6, 2, 2), 1)
    torch.autograd.backward([rotary(q, pos), rotary(k, pos), v], [dq, dk, dv])
    dqk = tw.ops.rope(torch.cat((dq, dk), 1), pos, f, scale=scale, inverse=True)
    assert torch.equal(y.grad, torch.cat((dqk, dv), 1))


def test_twice(tw, cuda):
    """The gradient of the gradient: the call by itself again, as it is linear."""
    g = torch.Generator().manual_seed(3)
    pos, f, _ = setting(tw, cuda, 5)
    x = normal(g, cuda, 5, 2, D).requires_grad_()
    dy = normal(g, cuda, 5, 2, D).requires_grad_()
    z = normal(g, cuda, 5, 2, D)
    dx, = torch.autograd.grad(tw.ops.rope(x, pos, f), x, dy, create_graph=True)
    back, = torch.autograd.grad(dx, dy, z)
    assert torch.equal(back, tw.ops.rope(z, pos, f))


def test_refused_instead_of_lost(tw, cuda):
    """What would cut a gradient off: an output of the caller's, frequencies that are learnt."""
    g = torch.Generator().manual_seed(4)
    pos, f, _ = setting(tw, cuda, 5)
    x = normal(g, cuda, 5, 2, D)
    leaf, out = x.clone().requires_grad_(), torch.zeros_like(x)
    for bad in (dict(x=leaf, out=out), dict(x=leaf, out=leaf), dict(x=x, out=leaf),
                dict(x=x, frequencies=f.clone().requires_grad_())):
        args = {**dict(x=x, positions=pos, frequencies=f), **bad}
        with pytest.raises(ValueError, match="gradient"):
            tw.ops.rope(args.pop("x"), args.pop("positions"), args.pop("frequencies"), **args)
    assert not bool(out.any()) and torch.equal(leaf.detach(), x)
    want = tw.ops.rope(x, pos, f)
    with torch.no_grad():  # nothing to lose
        assert torch.equal(tw.ops.rope(leaf, pos, f, out=out), want)
        assert torch.equal(tw.ops.rope(x, pos, f.clone().requires_grad_()), want)
    assert not tw.ops.rope(leaf.detach(), pos, f).requires_grad
    with pytest.raises(ValueError, match="frequencies"):  # and what was wrong stays wrong
        tw.ops.rope(leaf, pos, f.float())


def test_positions_kept(tw, cuda):
    """Positions that change before the gradient is taken are told, not used."""
    g = torch.Generator().manual_seed(5)
    pos, f, _ = setting(tw, cuda, 5)
    x = normal(g, cuda, 5, 2, D).requires_grad_()
    y = tw.ops.rope(x, pos, f)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_stream_and_graph(tw, cuda):
    """Forward and backward on another stream, and both replayed from a graph."""
    g = torch.Generator().manual_seed(6)
    pos, f, _ = setting(tw, cuda, 40)
    x0, dy = (normal(g, cuda, 40, 8, D) for _ in range(2))
    want = tw.ops.rope(dy, pos, f, inverse=True)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        x = x0.clone().requires_grad_()
        got, = torch.autograd.grad(tw.ops.rope(x, pos, f), x, dy)
    side.synchronize()
    assert torch.equal(got, want)
    del x
    x = x0.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = tw.ops.rope(x, pos, f)
        got, = torch.autograd.grad(y, x, dy)
    dy.copy_(normal(g, cuda, 40, 8, D))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, tw.ops.rope(dy, pos, f, inverse=True))
    assert torch.equal(y.detach(), tw.ops.rope(x0, pos, f))
