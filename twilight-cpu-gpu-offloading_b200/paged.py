"""A paged KV cache in device memory for several requests, and for prompts that are
processed in chunks (no counterpart in the reference, whose cache is one
contiguous slab per head, hi/slab_cache.py:37-74, filled by one whole prompt).

A serving step is::

    step = cache.step([512, 1, 1, -1])          # a chunk, two decodes, one request ends
    for layer in range(layers):
        q, k, v = project(layer, hidden, step.positions)
        cache.write(layer, k, v)
        out = cache.attend(layer, q)             # [tokens, q_heads, 128]

Tables, slots and lengths are built on the device (ops.paged_step); the host keeps
the lengths it gave, so nothing is read back and capacity is checked before a
launch.  step() copies the numbers it is given to the device and waits for that copy,
and so for what the stream holds before it.  Kernels see all max_requests rows, those of
waiting requests too: a cache for many more requests than are served at a time divides
its work less well than one of the right size.  A finished prompt can move to an offloaded cache for sparse decoding
(to_offloaded).
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _lib, ops
from .ops import HEAD_DIM


@dataclass(frozen=True)
class PagedStep:
    """What one step() planned; device tensors, rows of the step's tokens in request order.
    Later steps leave them as they are (the cache's block_table moves on)."""

    tokens: int
    cu_q: torch.Tensor        # [requests + 1] int32
    kv_lens: torch.Tensor     # [requests] int32, the new tokens included
    slots: torch.Tensor       # [tokens] int64
    positions: torch.Tensor   # [tokens] int32
    max_q_len: int
    max_kv_len: int


class PagedKVCache:
    """Pages of `page_size` tokens for `num_layers` layers and up to `max_requests`
    requests of up to `max_tokens_per_request` tokens.  The pages of one request are
    the same in every layer."""

    def __init__(self, *, num_layers: int, num_kv_heads: int, num_pages: int,
                 max_requests: int, max_tokens_per_request: int, page_size: int = 16,
                 head_dim: int = HEAD_DIM, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda") -> None:
        device = torch.device(device)
        if device.type != "cuda" or not torch.cuda.is_available():
            raise ValueError("an operational CUDA device is required")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if head_dim != HEAD_DIM:
            raise ValueError(f"head_dim must be {HEAD_DIM} (the sm_100a kernels' tile)")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("K/V dtype must be float16 or bfloat16")
        if min(num_layers, num_kv_heads, num_pages, max_requests, max_tokens_per_request) <= 0:
            raise ValueError("sizes must be positive")
        if page_size <= 0 or page_size % 8:
            raise ValueError("page_size must be a multiple of 8")
        if max_requests > 8192:
            raise ValueError("at most 8192 requests")
        _lib.load()  # fail loudly without the extension
        self.device, self.dtype = device, dtype
        self.num_layers, self.num_kv_heads = num_layers, num_kv_heads
        self.num_pages, self.page_size = num_pages, page_size
        self.max_requests = max_requests
        width = -(-max_tokens_per_request // page_size)
        self.max_tokens_per_request = width * page_size
        # [layer][K, V][page][head][row][D]
        self.pool = torch.empty((num_layers, 2, num_pages, num_kv_heads, page_size, HEAD_DIM),
                                dtype=dtype, device=device)
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((max_requests, width), -1, **i32)
        self._free_pages = torch.arange(num_pages - 1, -1, -1, **i32)
        self._lens = torch.zeros(max_requests, **i32)  # those of the last plan
        # free count before and after a step, in turn
        self._free_count = [torch.full((1,), num_pages, **i32) for _ in range(2)]
        self._turn = 0
        self._error_flag = torch.zeros(1, **i32)
        self.lengths = [0] * max_requests  # the host's copy
        self.free_pages = num_pages
        self._step: Optional[PagedStep] = None

    def _pages(self, tokens: int) -> int:
        return -(-tokens // self.page_size)

    # ----------------------------------------------------------------- steps --
    def step(self, new_tokens: Sequence[int]) -> PagedStep:
        """Plans the next step: new_tokens[r] tokens for request r (0: it waits; negative:
        it has ended, and its pages are free from this step on).  Requests past the
        sequence wait.  RuntimeError when pages or a request's row would not suffice,
        with nothing changed."""
        new = [int(n) for n in new_tokens]
        if len(new) > self.max_requests:
            raise ValueError(f"{len(new)} requests in a cache for {self.max_requests}")
        new += [0] * (self.max_requests - len(new))
        free = self.free_pages + sum(self._pages(l) for l, n in zip(self.lengths, new) if n < 0)
        after = [0 if n < 0 else l + n for l, n in zip(self.lengths, new)]
        for r, (l, n, a) in enumerate(zip(self.lengths, new, after)):
            if a > self.max_tokens_per_request:
                raise RuntimeError(f"capacity exceeded: request {r} would hold {a} tokens of "
                                   f"{self.max_tokens_per_request}")
            if n > 0:
                free -= self._pages(a) - self._pages(l)
        if free < 0:
            raise RuntimeError(f"capacity exceeded: {-free} pages too few")
        tokens = sum(n for n in new if n > 0)
        i32 = dict(dtype=torch.int32, device=self.device)
        before, now = self._turn, self._turn ^ 1
        cu_q = torch.empty(self.max_requests + 1, **i32)
        kv_lens = torch.empty(self.max_requests, **i32)
        slots = torch.empty(tokens, dtype=torch.int64, device=self.device)
        positions = torch.empty(tokens, **i32)
        ops.paged_step(self._lens, torch.tensor(new, **i32), self.block_table,
                       self._free_pages, self._free_count[before], page_size=self.page_size,
                       kv_lens=kv_lens, cu_q=cu_q, slots=slots, positions=positions,
                       free_count_out=self._free_count[now], error_flag=self._error_flag)
        self._turn, self._lens = now, kv_lens
        self.lengths, self.free_pages = after, free
        self._step = PagedStep(tokens, cu_q, kv_lens, slots, positions,
                               max(0, *new), max(after))
        return self._step

    def _layer(self, layer: int) -> tuple[torch.Tensor, torch.Tensor, PagedStep]:
        if not 0 <= layer < self.num_layers:
            raise IndexError("layer out of range")
        if self._step is None:
            raise ValueError("plan a step first")
        return self.pool[layer, 0], self.pool[layer, 1], self._step

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """The step's new K / V rows [tokens, kv_heads, 128] of one layer."""
        k_pages, v_pages, step = self._layer(layer)
        if k.shape[0] != step.tokens:
            raise ValueError(f"the step has {step.tokens} tokens, got {k.shape[0]} rows")
        if step.tokens:
            ops.paged_write(k, v, step.slots, k_pages, v_pages, error_flag=self._error_flag)

    def attend(self, layer: int, q: torch.Tensor, *, window: int = 0, **kw) -> torch.Tensor:
        """Attention of the step's tokens, whose rows have been written: q and the result
        [tokens, q_heads, 128].  Keywords of ops.paged_attention (out, out_dtype, lse,
        softmax_scale, workspace)."""
        k_pages, v_pages, step = self._layer(layer)
        if q.shape[0] != step.tokens:
            raise ValueError(f"the step has {step.tokens} tokens, got {q.shape[0]} rows")
        return ops.paged_attention(q, k_pages, v_pages, self.block_table, step.cu_q, step.kv_lens,
                                   max_q_len=step.max_q_len, max_kv_len=step.max_kv_len,
                                   window=window, error_flag=self._error_flag, **kw)

    # ---------------------------------------------------------------- export --
    def request_kv(self, layer: int, request: int) -> tuple[torch.Tensor, torch.Tensor]:
        """K and V of one request and layer, [kv_heads, tokens, 128] each."""
        k_pages, v_pages, _ = self._layer(layer)
        n, G, P = self.lengths[request], self.num_kv_heads, self.page_size
        out = torch.empty((2, G, n, HEAD_DIM), dtype=self.dtype, device=self.device)
        if n:
            j = torch.arange(n, device=self.device)
            page = self.block_table[request, j // P].long()
            g = torch.arange(G, device=self.device)[:, None]
            rows = ((page * G + g) * P + j % P).reshape(-1)
            ops.gather_kv(k_pages.reshape(-1, HEAD_DIM), v_pages.reshape(-1, HEAD_DIM), rows,
                          out[0].view(-1, HEAD_DIM), out[1].view(-1, HEAD_DIM), self._error_flag)
        return out[0], out[1]

    def to_offloaded(self, request: int, cache) -> None:
        """Hands a request's tokens to an offloaded cache as its prompt (its slab rows,
        page metadata and INT4 codes): layer i to entries i*kv_heads .. of `cache`."""
        G = self.num_kv_heads
        for layer in range(self.num_layers):
            k, v = self.request_kv(layer, request)
            cache.prefill_layer(key_states=k, value_states=v,
                                entries=list(range(layer * G, (layer + 1) * G)))

    def synchronize(self) -> None:
        """Waits for the device and raises what its checks found."""
        flag = int(self._error_flag.item())
        if flag:
            self._error_flag.zero_()
            _lib.check(flag, "device-side check")
