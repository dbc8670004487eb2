"""Tensors that the rotary calls change in place: autograd learns that they have changed."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128


def calls(tw, cuda):
    """Each way in which a tensor x [5, 4, 128] is overwritten."""
    f, _ = tw.ops.rope_frequencies(128, device=cuda)
    pos = torch.arange(5, dtype=torch.int32, device=cuda)
    pages = torch.zeros(2, 4, 16, D, dtype=torch.float16, device=cuda)
    other = torch.ones(5, 4, D, dtype=torch.float16, device=cuda)
    return {
        "in place": lambda x: tw.ops.rope(x, pos, f, out=x),
        "output": lambda x: tw.ops.rope(other, pos, f, out=x),
        "q in place": lambda x: tw.ops.paged_rope_write(x, other, other, pos, pos.long(), f,
                                                        pages, pages.clone(), q_out=x),
        "q output": lambda x: tw.ops.paged_rope_write(other, other, other, pos, pos.long(), f,
                                                      pages, pages.clone(), q_out=x)}


@pytest.mark.parametrize("way", ["in place", "output", "q in place", "q output"])
def test_told(tw, cuda, way):
    """A product keeps x for its gradient; x changes; the gradient is refused, not wrong."""
    call = calls(tw, cuda)[way]
    x = torch.full((5, 4, D), 2.0, dtype=torch.float16, device=cuda)
    w = torch.ones_like(x).requires_grad_()
    y = (w * x).sum()
    before = x._version
    call(x[:, :])  # (a view of it: they share what counts the changes)
    assert x._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


@pytest.mark.parametrize("way", ["in place", "output", "q in place", "q output"])
def test_inference_tensors(tw, cuda, way):
    """They count no changes: overwritten as before, inside inference mode and outside."""
    call = calls(tw, cuda)[way]
    with torch.inference_mode():
        x = torch.ones(5, 4, D, dtype=torch.float16, device=cuda)
        want = call(x.clone()).clone()
        y = x.clone()
        assert torch.equal(call(y), want)
        y = x.clone()
    assert torch.equal(call(y), want)


def test_inputs_are_not_told(tw, cuda):
    """What a call only reads keeps its count."""
    f, _ = tw.ops.rope_frequencies(128, device=cuda)
    x = torch.ones(5, 4, D, dtype=torch.float16, device=cuda)
    pos = torch.arange(5, dtype=torch.int32, device=cuda)
    pages = torch.zeros(2, 4, 16, D, dtype=torch.float16, device=cuda)
    tw.ops.rope(x, pos, f)
    tw.ops.paged_rope_write(x, x, x, pos, pos.long(), f, pages, pages.clone())
    assert x._version == 0 and pos._version == 0 and f._version == 0
