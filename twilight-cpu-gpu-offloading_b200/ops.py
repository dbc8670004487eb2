"""Tensor-level wrappers of the C ABI (device memory from torch, work on the
current CUDA stream).  Every op runs the sm_100a kernels of
libtwilight_b200.so; a CPU tensor is rejected, never computed on the host.
"""

from __future__ import annotations

import ctypes
import functools
import math
import struct

import torch

from . import _lib

HEAD_DIM = 128
DTYPE_CODES = {torch.float16: _lib.TW_F16, torch.bfloat16: _lib.TW_BF16, torch.float32: _lib.TW_F32}
_SCALE = 1.0 / math.sqrt(HEAD_DIM)
SCALE_RECIPROCAL = 0   # "/ 15" as torch on CUDA: x * fp32(1/15)
SCALE_DIVIDE = 1       # "/ 15" as torch on CPU: IEEE division


def _stream(device: torch.device | None = None) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("twilight ops require CUDA tensors (no CPU fallback)")
        if not t.is_contiguous():
            raise ValueError("twilight ops require contiguous tensors")


def _kv_code(dtype: torch.dtype) -> int:
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"K/V dtype must be float16 or bfloat16, got {dtype}")
    return DTYPE_CODES[dtype]


def lib():
    return _lib.load()


# ---------------------------------------------------------------- metadata --

def quest_page_metadata(keys: torch.Tensor, *, sink: int, block_size: int,
                        page_min: torch.Tensor, page_max: torch.Tensor, first_page: int = 0,
                        n_pages: int | None = None) -> int:
    """keys [E, S, D] -> page_min/page_max [E, page_cap, D] pages [first_page, +n_pages).
    hi/quest_offload_cache.py:276-289.  Returns the number of pages written."""
    _cuda(keys, page_min, page_max)
    E, S, D = keys.shape
    if D != HEAD_DIM or page_min.shape[0] != E or page_min.shape != page_max.shape:
        raise ValueError("unexpected metadata shapes")
    complete = max(0, S - sink) // block_size if S > sink else 0
    if n_pages is None:
        n_pages = complete - first_page
    if n_pages < 0 or first_page + n_pages > page_min.shape[1] or first_page + n_pages > complete:
        raise ValueError("page range outside the keys or the metadata capacity")
    _lib.check(lib().tw_quest_page_metadata(
        _ptr(keys), S * D, E, sink, block_size, D, _kv_code(keys.dtype), first_page, n_pages,
        _ptr(page_min), _ptr(page_max), page_min.shape[1] * D, _stream(keys.device)),
        "quest_page_metadata")
    return n_pages


def int4_pack(keys: torch.Tensor, *, group_size: int, packed: torch.Tensor, scale: torch.Tensor,
              minimum: torch.Tensor, out_row_offset: int = 0,
              scale_div: int = SCALE_RECIPROCAL) -> None:
    """keys [E, S, D] -> packed [E, cap, D/2] u8, scale/minimum [E, cap, D/gs] at rows
    out_row_offset.. (hi/twilight_offload_cache.py:25-37 over keys.view(-1, gs))."""
    _cuda(keys, packed, scale, minimum)
    E, S, D = keys.shape
    if packed.dtype != torch.uint8 or packed.shape[0] != E or packed.shape[-1] != D // 2:
        raise ValueError("packed must be uint8 [E, cap, D/2]")
    if scale.dtype != keys.dtype or minimum.dtype != keys.dtype:
        raise ValueError("scale/minimum must have the K dtype")
    cap = packed.shape[1]
    if out_row_offset + S > cap or scale.shape != (E, cap, D // group_size) or minimum.shape != scale.shape:
        raise ValueError("INT4 output capacity or group layout mismatch")
    _lib.check(lib().tw_int4_pack_ex(
        _ptr(keys), S, E, S, D, group_size, _kv_code(keys.dtype), _ptr(packed), _ptr(scale),
        _ptr(minimum), cap, out_row_offset, scale_div, _stream(keys.device)), "int4_pack")


# --------------------------------------------------------------- selection --

def quest_score(q: torch.Tensor, page_min: torch.Tensor, page_max: torch.Tensor, n_pages: int,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """q [G,R,D] fp32, page_min/max [G, page_cap, D] -> scores [G,R,n_pages] fp32.
    hi/twilight_fused_quest.py:13-46."""
    _cuda(q, page_min, page_max)
    G, R, D = q.shape
    if q.dtype != torch.float32 or page_min.shape[0] != G or n_pages > page_min.shape[1]:
        raise ValueError("quest_score expects fp32 q [G,R,D] and [G,cap,D] metadata")
    if out is None:
        out = torch.empty((G, R, n_pages), device=q.device, dtype=torch.float32)
    _lib.check(lib().tw_quest_score(_ptr(q), _ptr(page_min), _ptr(page_max), G, R, n_pages,
                                    page_min.shape[1] * D, D, _kv_code(page_min.dtype), _ptr(out),
                                    _stream(q.device)), "quest_score")
    return out


def topk_pages(scores: torch.Tensor, k: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """scores [..., n] fp32 -> ascending ids of the k largest [..., k] int32."""
    _cuda(scores)
    n = scores.shape[-1]
    rows = scores.numel() // max(n, 1)
    if out is None:
        out = torch.empty((*scores.shape[:-1], k), device=scores.device, dtype=torch.int32)
    _lib.check(lib().tw_topk_pages(_ptr(scores), rows, n, k, _ptr(out), _stream(scores.device)),
               "topk_pages")
    return out


def int4_qk(q: torch.Tensor, packed: torch.Tensor, scale: torch.Tensor, minimum: torch.Tensor,
            pages: torch.Tensor, *, block_size: int, sink: int,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """q [G,R,D]; packed [G, cap, D/2]; scale/minimum [G, cap, ng]; pages [G,R,b0] int32
    -> logits [G,R,b0*block] fp32 (hi/twilight_fused_qk.py:13-55, /sqrt(D) :1261)."""
    _cuda(q, packed, scale, minimum, pages)
    G, R, D = q.shape
    b0 = pages.shape[-1]
    group = D // scale.shape[-1]
    if out is None:
        out = torch.empty((G, R, b0 * block_size), device=q.device, dtype=torch.float32)
    _lib.check(lib().tw_int4_qk(_ptr(q), _ptr(packed), _ptr(scale), _ptr(minimum), packed.shape[1],
                                _ptr(pages), G, R, b0, block_size, sink, D, group,
                                _kv_code(scale.dtype), _ptr(out), _stream(q.device)), "int4_qk")
    return out


def top_p_union(logits: torch.Tensor, pages: torch.Tensor, *, block_size: int, sink: int,
                top_p: float, old_length: int, sink_end: int, recent_start: int,
                union_pos: torch.Tensor, union_count: torch.Tensor, head_count: torch.Tensor,
                head_pos: torch.Tensor | None = None,
                error_flag: torch.Tensor | None = None) -> None:
    """Top-p counts per row and the sorted GQA union per group (device outputs)."""
    _cuda(logits, pages, union_pos, union_count, head_count, head_pos, error_flag)
    G, R, n = logits.shape
    b0 = pages.shape[-1]
    _lib.check(lib().tw_top_p_union(
        _ptr(logits), _ptr(pages), G, R, b0, block_size, sink, float(top_p), old_length, sink_end,
        recent_start, _ptr(union_pos), union_pos.shape[-1], _ptr(union_count), _ptr(head_count),
        _ptr(head_pos), _ptr(error_flag), _stream(logits.device)), "top_p_union")


def select_layer(q: torch.Tensor, page_min: torch.Tensor, page_max: torch.Tensor, n_pages: int,
                 packed: torch.Tensor, scale: torch.Tensor, minimum: torch.Tensor, *, b0_pages: int,
                 block_size: int, sink: int, top_p: float, old_length: int, sink_end: int,
                 recent_start: int, union_pos: torch.Tensor, union_count: torch.Tensor,
                 head_count: torch.Tensor, head_pos: torch.Tensor | None = None,
                 error_flag: torch.Tensor | None = None,
                 pages: torch.Tensor | None = None) -> torch.Tensor:
    """Both Twilight selection stages of one layer (tw_select_layer: Quest score,
    top-k pages, INT4 estimate, top-p + GQA union; one fused launch where the
    shape allows).  q [G,R,D] fp32, metadata / codes as quest_score / int4_qk.
    Returns the B0 pages [G,R,b0] int32; the union and counts go to the outputs."""
    _cuda(q, page_min, page_max, packed, scale, minimum, union_pos, union_count, head_count,
          head_pos, error_flag, pages)
    G, R, D = q.shape
    if q.dtype != torch.float32:
        raise ValueError("select_layer expects fp32 q [G,R,D]")
    if pages is None:
        pages = torch.empty((G, R, b0_pages), device=q.device, dtype=torch.int32)
    ws_bytes = select_layer_workspace_bytes(G, R, n_pages, b0_pages, block_size)
    ws = torch.zeros(max(ws_bytes, 256), dtype=torch.uint8, device=q.device)  # merge region zero
    _lib.check(lib().tw_select_layer(
        _ptr(q), _ptr(page_min), _ptr(page_max), page_min.shape[1] * D, n_pages, _ptr(packed),
        _ptr(scale), _ptr(minimum), packed.shape[1], G, R, b0_pages, block_size, sink, D,
        D // scale.shape[-1], _kv_code(scale.dtype), float(top_p), old_length, sink_end,
        recent_start, _ptr(pages), _ptr(union_pos), union_pos.shape[-1], _ptr(union_count),
        _ptr(head_count), _ptr(head_pos), _ptr(error_flag), _ptr(ws), ws.numel(),
        _stream(q.device)), "select_layer")
    return pages


def select_layer_workspace_bytes(groups: int, heads: int, n_pages: int, b0_pages: int,
                                 block_size: int) -> int:
    return int(lib().tw_select_layer_workspace_size(groups, heads, n_pages, b0_pages, block_size))


# ------------------------------------------------------------------ gather --

def gather_kv(k: torch.Tensor, v: torch.Tensor, rows: torch.Tensor, out_k: torch.Tensor,
              out_v: torch.Tensor, error_flag: torch.Tensor) -> None:
    """out[i] = src[rows[i]] (hi/cpu_kv_gather.cpp:3-16 contract) on the GPU.  k/v may be
    CUDA tensors or mapped-host views given as (tensor, device_pointer) pairs."""
    kp, k_rows, row_bytes = _source(k)
    vp, v_rows, _ = _source(v)
    _cuda(rows, out_k, out_v, error_flag)
    if rows.dtype != torch.int64:
        raise ValueError("int64 row indices required")
    _lib.check(lib().tw_gather_kv(kp, vp, _ptr(out_k), _ptr(out_v), _ptr(rows), rows.numel(),
                                  k_rows, row_bytes, _ptr(error_flag), _stream(rows.device)),
               "gather_kv")


def _source(x):
    if isinstance(x, tuple):
        t, dev = x
        return dev, t.shape[0], t.shape[-1] * t.element_size()
    _cuda(x)
    return x.data_ptr(), x.shape[0], x.shape[-1] * x.element_size()


def decode_attention_workspace_bytes(segments: int, heads: int, max_seqlen_k: int) -> int:
    return int(lib().tw_decode_attention_workspace_size(segments, heads, max_seqlen_k, HEAD_DIM))


def decode_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_k: torch.Tensor,
                     max_seqlen_k: int, *, workspace: torch.Tensor, out: torch.Tensor | None = None,
                     out_dtype: torch.dtype | None = None, lse: torch.Tensor | None = None,
                     softmax_scale: float | None = None) -> torch.Tensor:
    """q [S,R,D]; k/v [rows,(1,)D]; cu_seqlens_k [S+1] int32 -> out [S,R,D].
    Replaces flash_attn_varlen_func at hi/mp.py:258-279."""
    _cuda(q, k, v, cu_seqlens_k, workspace, out, lse)
    S, R, D = q.shape
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must share a dtype")
    if cu_seqlens_k.dtype != torch.int32 or cu_seqlens_k.numel() != S + 1:
        raise ValueError("cu_seqlens_k must be int32 [segments + 1]")
    out_dtype = out_dtype or q.dtype
    if out is None:
        out = torch.empty((S, R, D), device=q.device, dtype=out_dtype)
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D)
    _lib.check(lib().tw_decode_attention(
        _ptr(q), _ptr(k), _ptr(v), _ptr(cu_seqlens_k), S, R, int(max_seqlen_k), D,
        _kv_code(q.dtype), ctypes.c_float(scale), _ptr(out), DTYPE_CODES[out.dtype], _ptr(lse),
        _ptr(workspace), workspace.numel() * workspace.element_size(), _stream(q.device)),
        "decode_attention")
    return out


def attend_union(slab, first_entry: int, old_length: int, union_pos: torch.Tensor,
                 union_count: torch.Tensor, cur_k: torch.Tensor, cur_v: torch.Tensor,
                 q: torch.Tensor, max_rows_per_group: int, *, workspace: torch.Tensor,
                 error_flag: torch.Tensor, out: torch.Tensor | None = None,
                 out_dtype: torch.dtype | None = None, lse: torch.Tensor | None = None,
                 softmax_scale: float | None = None,
                 entry_dirs: torch.Tensor | None = None,
                 reuse: "_lib.RowReuse | None" = None) -> torch.Tensor:
    """Fused union gather + decode attention straight from the mapped slab (or,
    with entry_dirs [2, E] int64 row-0 addresses, from each entry's placement).
    q [G,R,D] (K/V dtype), cur_k/cur_v [G,D], union_pos [G, stride] int32,
    union_count [G] int32 -> out [G,R,D].  reuse (row_reuse()): read rows of
    the previous step from device memory and keep this step's rows."""
    _cuda(union_pos, union_count, cur_k, cur_v, q, workspace, error_flag, out, lse)
    G, R, D = q.shape
    out_dtype = out_dtype or q.dtype
    if out is None:
        out = torch.empty((G, R, D), device=q.device, dtype=out_dtype)
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(D)
    _lib.check(lib().tw_attend_union(
        slab.key_device_ptr, slab.value_device_ptr, _ptr(entry_dirs),
        entry_dirs.shape[-1] if entry_dirs is not None else 0, slab.geometry.max_cache_len, first_entry, G,
        old_length, _ptr(union_pos), union_pos.shape[-1], _ptr(union_count), _ptr(cur_k),
        _ptr(cur_v), _ptr(q), R, int(max_rows_per_group), D, _kv_code(q.dtype),
        ctypes.c_float(scale), _ptr(out), DTYPE_CODES[out.dtype], _ptr(lse), _ptr(error_flag),
        _ptr(workspace), workspace.numel() * workspace.element_size(),
        ctypes.byref(reuse) if reuse is not None else None, _stream(q.device)),
        "attend_union")
    return out


def row_reuse(row_map: torch.Tensor, next_tag: int, *, next_k: torch.Tensor | None = None,
              next_v: torch.Tensor | None = None, prev_tag: int = 0,
              prev_k: torch.Tensor | None = None, prev_v: torch.Tensor | None = None,
              row_counts: torch.Tensor | None = None) -> "_lib.RowReuse":
    """tw_row_reuse for attend_union / decode_layer (next_k / next_v
    [G, S, D] receive this step's rows) or tw_gather_union (no next rows: its
    output is kept).  row_map [G, stride] int64 (zeroed before first use) maps
    positions to (tag << 32) | row of the kept rows; prev_k / prev_v [rows, D]
    (any leading shape) are the rows kept under prev_tag (0: none).
    row_counts [G, 2] int32 accumulates (hit rows, miss rows)."""
    _cuda(row_map, next_k, next_v, prev_k, prev_v, row_counts)
    if row_map.dtype != torch.int64 or row_map.dim() != 2:
        raise ValueError("row_map must be int64 [G, stride]")
    r = _lib.RowReuse()
    r.row_map, r.map_stride = row_map.data_ptr(), row_map.shape[1]
    r.next_tag, r.prev_tag = int(next_tag), int(prev_tag)
    if next_k is not None or next_v is not None:
        if next_k is None or next_v is None or next_k.dim() != 3 or next_k.shape != next_v.shape:
            raise ValueError("next_k / next_v must be [G, S, D]")
        r.next_k, r.next_v = next_k.data_ptr(), next_v.data_ptr()
        r.rows_stride = next_k.shape[1]
    if prev_tag:
        if prev_k is None or prev_v is None or prev_k.shape != prev_v.shape:
            raise ValueError("prev_tag needs prev_k and prev_v of one shape")
        r.prev_k, r.prev_v = prev_k.data_ptr(), prev_v.data_ptr()
        r.prev_rows = prev_k.numel() // prev_k.shape[-1]
    if row_counts is not None:
        if row_counts.dtype != torch.int32 or row_counts.shape != (row_map.shape[0], 2):
            raise ValueError("row_counts must be int32 [G, 2]")
        r.row_counts = row_counts.data_ptr()
    return r


def qkv_rope(hidden: torch.Tensor, w_q: torch.Tensor, w_k: torch.Tensor, w_v: torch.Tensor,
             cos: torch.Tensor, sin: torch.Tensor, *, q_out: torch.Tensor | None = None,
             k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None):
    """Decode-layer front end (tw_qkv_rope): hidden [H] and the nn.Linear weights
    w_q [n_q*128, H], w_k / w_v [n_kv*128, H] -> q [n_q, 128] (rotated), k
    [n_kv, 128] (rotated), v [n_kv, 128]; cos / sin [128] of the token's position."""
    _cuda(hidden, w_q, w_k, w_v, cos, sin, q_out, k_out, v_out)
    dt = hidden.dtype
    if any(t.dtype != dt for t in (w_q, w_k, w_v, cos, sin)):
        raise ValueError("hidden, weights and cos / sin must share one dtype")
    H = hidden.numel()
    if w_q.shape[1] != H or w_k.shape != w_v.shape or w_k.shape[1] != H or \
            w_q.shape[0] % HEAD_DIM or w_k.shape[0] % HEAD_DIM or cos.numel() != HEAD_DIM or \
            sin.numel() != HEAD_DIM:
        raise ValueError("weights must be [heads*128, hidden], cos / sin [128]")
    n_q, n_kv = w_q.shape[0] // HEAD_DIM, w_k.shape[0] // HEAD_DIM
    q_out = q_out if q_out is not None else torch.empty((n_q, HEAD_DIM), dtype=dt, device=hidden.device)
    k_out = k_out if k_out is not None else torch.empty((n_kv, HEAD_DIM), dtype=dt, device=hidden.device)
    v_out = v_out if v_out is not None else torch.empty((n_kv, HEAD_DIM), dtype=dt, device=hidden.device)
    _lib.check(lib().tw_qkv_rope(
        _ptr(hidden), _ptr(w_q), _ptr(w_k), _ptr(w_v), H, n_q, n_kv, HEAD_DIM, _ptr(cos), _ptr(sin),
        _kv_code(dt), _ptr(q_out), _ptr(k_out), _ptr(v_out), _stream(hidden.device)), "qkv_rope")
    return q_out, k_out, v_out


# ------------------------------------------------------------- paged cache --
# These calls are made for every step and layer, and a short one's kernel takes a
# few microseconds.  So each has one expression of all checks (the message is
# worked out only when it fails) and packs its arguments in one go.

_PACK_POOL = struct.Struct(_lib.PAGED_POOL_FORMAT).pack
_PACK_STEP = struct.Struct(_lib.PAGED_STEP_FORMAT).pack
_PACK_ATTENTION = struct.Struct(_lib.PAGED_ATTENTION_FORMAT).pack
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice

# Workspaces of paged_attention calls that brought none, per (device, stream): calls on
# one stream follow one another, and a larger one takes the place of a smaller.
_paged_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def _paged_workspace(dev: int, stream: int, need: int) -> torch.Tensor:
    if torch.cuda.is_current_stream_capturing():  # a graph keeps its own
        return torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", dev))
    kept = _paged_workspaces.get((dev, stream))
    if kept is None or kept.numel() < need:
        kept = torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", dev))
        _paged_workspaces[dev, stream] = kept
    return kept


def _device_index(t: torch.Tensor) -> int:
    """The current device's index, which has to be t's."""
    dev = t.get_device()
    if dev < 0:
        raise ValueError("twilight ops require CUDA tensors (no CPU fallback)")
    if dev != _current_device():
        raise ValueError(f"the tensors are on cuda:{dev}: make it the current device")
    return dev


def _explain(dev: int, *wanted) -> None:
    """Raises for the first tensor that is not as wanted: (name, tensor, dtype, shape);
    a tensor of None is optional, an extent of None is any."""
    for name, t, dtype, shape in wanted:
        if t is None:
            continue
        if t.get_device() < 0:
            raise ValueError("twilight ops require CUDA tensors (no CPU fallback)")
        if t.get_device() != dev:
            raise ValueError(f"{name} must be on the device of the other tensors, cuda:{dev}")
        if t.dtype != dtype or t.dim() != len(shape) or \
                any(n is not None and n != m for n, m in zip(shape, t.shape)) or \
                not (t[0] if t.dim() > 1 and t.shape[0] else t).is_contiguous():
            want = ", ".join("*" if n is None else str(n) for n in shape)
            raise ValueError(f"{name} must be {dtype} [{want}] with contiguous rows, got "
                             f"{t.dtype} {list(t.shape)}")
    raise ValueError("unexpected tensors")


def _rows_strides(name: str, t: torch.Tensor) -> tuple[int, int]:
    """(token, head) strides of [tokens, heads, 128] rows; an extent of 1 has none of its own."""
    token, head, inner = t.stride()
    tokens, heads, _ = t.shape
    if inner != 1:
        raise ValueError(f"{name} needs contiguous rows of {HEAD_DIM} elements")
    if heads <= 1:
        head = HEAD_DIM
    if tokens <= 1:
        token = head * (heads or 1)
    if token <= 0 or head <= 0 or (token | head) & 7 or t.data_ptr() & 15:
        raise ValueError(f"{name} needs 16-byte aligned rows (positive strides in multiples of 8)")
    return token, head


def _paged_pool(dev: int, k_pages: torch.Tensor, v_pages: torch.Tensor) -> tuple:
    """The fields of tw_paged_pool for [pages, kv_heads, page_size, 128] tensors (any
    order of strides)."""
    shape, strides = k_pages.shape, k_pages.stride()
    if len(shape) != 4 or shape != v_pages.shape or k_pages.dtype != v_pages.dtype \
            or shape[3] != HEAD_DIM or 0 in shape:
        raise ValueError(f"k_pages and v_pages must be [pages, kv_heads, page_size, {HEAD_DIM}] "
                         "of one dtype")
    if k_pages.get_device() != dev or v_pages.get_device() != dev:
        _explain(dev, ("k_pages", k_pages, k_pages.dtype, shape),
                 ("v_pages", v_pages, v_pages.dtype, shape))
    if 1 in shape:  # an extent of 1 has no stride of its own
        other = tuple(HEAD_DIM if n == 1 else s for n, s in zip(shape, v_pages.stride()))
        strides = tuple(HEAD_DIM if n == 1 else s for n, s in zip(shape, strides))
    else:
        other = v_pages.stride()
    if strides != other:
        raise ValueError("k_pages and v_pages must have the same strides")
    page, head, token, inner = strides
    k, v = k_pages.data_ptr(), v_pages.data_ptr()
    if inner != 1 or page <= 0 or head <= 0 or token <= 0 or (page | head | token) & 7 or \
            (k | v) & 15:
        raise ValueError("pages need contiguous 16-byte aligned rows (strides in multiples of 8)")
    return k, v, page, head, token, shape[0], shape[2], shape[1], HEAD_DIM, _kv_code(k_pages.dtype)


def paged_step(lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
               free_pages: torch.Tensor, free_count: torch.Tensor, *, page_size: int,
               kv_lens: torch.Tensor, cu_q: torch.Tensor, slots: torch.Tensor,
               positions: torch.Tensor, free_count_out: torch.Tensor,
               error_flag: torch.Tensor | None = None) -> None:
    """Block tables and slot map of one serving step, in one launch (tw_paged_step).

    lens / new_lens [B] int32 (tokens held, tokens to add; new < 0: the request
    has ended and its pages go back), block_table [B, W] and the page stack
    free_pages [num_pages] with free_count [1] entries are updated; outputs
    kv_lens [B], cu_q [B+1], free_count_out [1] and, per new token, slots
    (int64, -1: none) and positions [tokens_cap].  A refused request or a full
    output sets error_flag to TW_ERR_CAPACITY."""
    dev = _device_index(lens)
    i32 = torch.int32
    B = lens.shape[0] if lens.dim() == 1 else -1
    each, cap = (B,), slots.shape
    if not (lens.dtype is new_lens.dtype is block_table.dtype is free_pages.dtype is
            free_count.dtype is kv_lens.dtype is cu_q.dtype is positions.dtype is
            free_count_out.dtype is i32 and slots.dtype is torch.int64
            and new_lens.shape == each and kv_lens.shape == each and cu_q.shape == (B + 1,)
            and free_pages.dim() == 1 and free_count.shape == (1,)
            and free_count_out.shape == (1,) and len(cap) == 1 and positions.shape == cap
            and block_table.dim() == 2 and block_table.shape[0] == B
            and (block_table.stride(1) == 1 or block_table.shape[1] == 1)
            and lens.is_contiguous() and new_lens.is_contiguous() and free_pages.is_contiguous()
            and kv_lens.is_contiguous() and cu_q.is_contiguous() and slots.is_contiguous()
            and positions.is_contiguous()
            and dev == new_lens.get_device() == block_table.get_device() ==
            free_pages.get_device() == free_count.get_device() == kv_lens.get_device() ==
            cu_q.get_device() == slots.get_device() == positions.get_device() ==
            free_count_out.get_device()
            and (error_flag is None
                 or (error_flag.get_device() == dev and error_flag.dtype is i32))):
        _explain(dev, ("lens", lens, i32, (None,)), ("new_lens", new_lens, i32, each),
                 ("block_table", block_table, i32, (B, None)),
                 ("free_pages", free_pages, i32, (None,)), ("free_count", free_count, i32, (1,)),
                 ("kv_lens", kv_lens, i32, each), ("cu_q", cu_q, i32, (B + 1,)),
                 ("slots", slots, torch.int64, (None,)),
                 ("positions", positions, i32, cap[:1]),
                 ("free_count_out", free_count_out, i32, (1,)),
                 ("error_flag", error_flag, i32, (1,)))
    W = block_table.shape[1]
    args = _PACK_STEP(
        lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(),
        block_table.stride(0) if B > 1 else W, W, B, page_size, cap[0], free_pages.data_ptr(),
        free_pages.shape[0], free_count.data_ptr(), kv_lens.data_ptr(), cu_q.data_ptr(),
        slots.data_ptr(), positions.data_ptr(), free_count_out.data_ptr(),
        0 if error_flag is None else error_flag.data_ptr())
    status = lib().tw_paged_step(args, _raw_stream(dev))
    if status:
        _lib.check(status, "paged_step")


def paged_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor,
                v_pages: torch.Tensor, *, error_flag: torch.Tensor | None = None) -> None:
    """New rows k / v [T, kv_heads, 128] (strided views of a projection are fine) to
    slots [T] int64 of the pool [pages, kv_heads, page_size, 128] (tw_paged_write);
    slot -1 is skipped."""
    dev = _device_index(k)
    pool = _paged_pool(dev, k_pages, v_pages)
    shape, dtype = k.shape, k_pages.dtype
    if not (len(shape) == 3 and shape == v.shape and shape[1] == pool[7] and shape[2] == HEAD_DIM
            and k.dtype is v.dtype is dtype and slots.dtype is torch.int64
            and slots.shape == shape[:1] and slots.is_contiguous()
            and dev == v.get_device() == slots.get_device()
            and (error_flag is None
                 or (error_flag.get_device() == dev and error_flag.dtype is torch.int32))):
        rows = (None, pool[7], HEAD_DIM)
        _explain(dev, ("k", k[:0], dtype, rows), ("v", v[:0], dtype, rows),
                 ("slots", slots, torch.int64, shape[:1]),
                 ("error_flag", error_flag, torch.int32, (1,)))
    k_token, k_head = _rows_strides("k", k)
    v_token, v_head = _rows_strides("v", v)
    status = lib().tw_paged_write(
        _PACK_POOL(*pool), k.data_ptr(), k_token, k_head, v.data_ptr(), v_token, v_head,
        slots.data_ptr(), shape[0], None if error_flag is None else error_flag.data_ptr(),
        _raw_stream(dev))
    if status:
        _lib.check(status, "paged_write")


@functools.lru_cache(maxsize=1024)
def paged_attention_workspace_bytes(requests: int, tokens: int, q_heads: int, kv_heads: int,
                                    max_q_len: int, max_kv_len: int, window: int = 0) -> int:
    """Bytes of the workspace of a paged_attention call of these sizes (0: none needed)."""
    return int(lib().tw_paged_attention_workspace_size(requests, tokens, q_heads, kv_heads,
                                                       max_q_len, max_kv_len, window, HEAD_DIM))


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    block_table: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor, *,
                    max_q_len: int, max_kv_len: int, window: int = 0,
                    softmax_scale: float | None = None, out: torch.Tensor | None = None,
                    out_dtype: torch.dtype | None = None, lse: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None,
                    error_flag: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of each request's new tokens over its paged tokens, the
    new ones included (tw_paged_attention): one token each, chunks of prompts,
    or both in one call.

    q [T, q_heads, 128] (token and head strides free), pool [pages, kv_heads,
    page_size, 128], block_table [B, W] int32, cu_q [B+1] and kv_lens [B] int32
    on the device; max_q_len bounds the requests' new tokens, max_kv_len is their
    longest kv_lens (it sizes the launch).  window > 0: each token sees the last
    `window` positions only.  Returns out [T, q_heads, 128] (q's dtype or
    float32); lse [T, q_heads] fp32 receives the log-sum-exp.  Without a
    workspace one is taken that is kept for the current stream."""
    dev = _device_index(q)
    pool = _paged_pool(dev, k_pages, v_pages)
    shape, dtype, i32 = q.shape, q.dtype, torch.int32
    if len(shape) != 3 or shape[2] != HEAD_DIM or dtype is not k_pages.dtype or \
            shape[1] == 0 or shape[1] % pool[7]:
        raise ValueError("q must be [T, q_heads, 128] in the pool's dtype, q_heads a multiple of "
                         "kv_heads")
    T, Hq, _ = shape
    if kv_lens.dim() != 1:
        raise ValueError("kv_lens must be [requests]")
    B = kv_lens.shape[0]
    if not (kv_lens.dtype is cu_q.dtype is block_table.dtype is i32 and cu_q.shape == (B + 1,)
            and block_table.dim() == 2 and block_table.shape[0] == B
            and (block_table.stride(1) == 1 or block_table.shape[1] == 1)
            and kv_lens.is_contiguous() and cu_q.is_contiguous()
            and dev == kv_lens.get_device() == cu_q.get_device() == block_table.get_device()
            and (lse is None or (lse.dtype is torch.float32 and lse.shape == (T, Hq)
                                 and lse.is_contiguous() and lse.get_device() == dev))
            and (error_flag is None
                 or (error_flag.get_device() == dev and error_flag.dtype is i32))):
        _explain(dev, ("kv_lens", kv_lens, i32, (None,)), ("cu_q", cu_q, i32, (B + 1,)),
                 ("block_table", block_table, i32, (B, None)),
                 ("lse", lse, torch.float32, (T, Hq)), ("error_flag", error_flag, i32, (1,)))
    if out is None:
        if (out_dtype is None or out_dtype is dtype) and q.is_contiguous():
            out = torch.empty_like(q)  # half the time of torch.empty
        else:
            out = torch.empty(shape, dtype=out_dtype or dtype, device=q.device)
        out_token, out_head = Hq * HEAD_DIM, HEAD_DIM
    else:
        if out.shape != shape or out.get_device() != dev or \
                (out_dtype is not None and out.dtype is not out_dtype):
            raise ValueError("out must have q's shape and device (and out_dtype)")
        out_token, out_head = _rows_strides("out", out)
    if out.dtype is not dtype and out.dtype is not torch.float32:
        raise ValueError("out must have q's dtype or float32")
    stream = _raw_stream(dev)
    if workspace is None:
        need = paged_attention_workspace_bytes(B, T, Hq, pool[7], max_q_len, max_kv_len, window)
        if need:
            workspace = _paged_workspace(dev, stream, need)
    else:
        need = workspace.numel() * workspace.element_size()
        if workspace.get_device() != dev or not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous, on q's device")
    W = block_table.shape[1]
    q_token, q_head = _rows_strides("q", q)
    args = _PACK_ATTENTION(
        *pool, q.data_ptr(), q_token, q_head, block_table.data_ptr(),
        block_table.stride(0) if B > 1 else W, W, B, cu_q.data_ptr(), kv_lens.data_ptr(), T, Hq,
        max_q_len, max_kv_len, window,
        _SCALE if softmax_scale is None else softmax_scale, out.data_ptr(), out_token, out_head,
        DTYPE_CODES[out.dtype], 0, 0 if lse is None else lse.data_ptr(),
        0 if error_flag is None else error_flag.data_ptr(),
        0 if workspace is None else workspace.data_ptr(), need)
    status = lib().tw_paged_attention(args, stream)
    if status:
        _lib.check(status, "paged_attention")
    return out
