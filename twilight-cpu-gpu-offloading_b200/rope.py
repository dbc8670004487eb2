"""A model's rotary positions on one device: the frequencies and factor of
ops.rope_frequencies and the layout, for ops.rope and PagedKVCache.write_rotated (no
counterpart in the reference, whose models bring their own, hi/mp.py:211-217)."""

from __future__ import annotations

from typing import Optional

import torch

from . import ops


class RotaryPositions:
    """Rotary positions of the first `dims` dimensions of each head.

    layout "half" pairs dimensions (n, n + dims / 2), "interleaved" (2n, 2n + 1); base and
    scaling as in ops.rope_frequencies."""

    def __init__(self, dims: int = ops.HEAD_DIM, *, base: float = 10000.0, layout: str = "half",
                 scaling: Optional[dict] = None, device: torch.device | str = "cuda") -> None:
        ops._interleaved(layout)
        self.dims, self.layout = dims, layout
        self.frequencies, self.scale = ops.rope_frequencies(dims, base=base, scaling=scaling,
                                                            device=device)

    def __call__(self, x: torch.Tensor, positions: torch.Tensor, *, inverse: bool = False,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Rows x [T, heads, 128] turned by positions [T] int32 (ops.rope, differentiable in x)."""
        return ops.rope(x, positions, self.frequencies, layout=self.layout, scale=self.scale,
                        inverse=inverse, out=out)
