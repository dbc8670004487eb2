"""ctypes binding of the C ABI (include/twilight_b200.h).

The library is the only compute path: there is no CPU fallback.  Loading
fails loudly when libtwilight_b200.so is absent.  Status codes map to the
exception types the reference raises: ValueError for bad shapes/arguments and
invalid row indices (hi/cpu_kv_gather.py:35-36), RuntimeError for CUDA and
capacity errors (hi/quest_offload_cache.py:104-106).
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libtwilight_b200.so"
BINDING_PATH = LIB_PATH.with_name("_binding.so")

TW_OK = 0
TW_ERR_INVALID_INDEX = 1
TW_ERR_BAD_ARG = 2
TW_ERR_CAPACITY = 3
TW_ERR_ORDER = 4
TW_ERR_CUDA = 5
TW_ERR_TIMEOUT = 6
TW_ERR_UNSUPPORTED = 7

TW_F16 = 0
TW_BF16 = 1
TW_F32 = 2

P = ctypes.c_void_p
I32 = ctypes.c_int
I64 = ctypes.c_int64
SZ = ctypes.c_size_t
DBL = ctypes.c_double
FLT = ctypes.c_float

I32T = ctypes.c_int32


class DecodeLayerArgs(ctypes.Structure):
    """tw_decode_layer_args of include/twilight_b200.h (same field order and types)."""

    _fields_ = [
        ("slab_k", P), ("slab_v", P), ("entry_dirs", P), ("n_entries", I64), ("max_len", I64), ("first_entry", I32T), ("groups", I32T),
        ("heads_per_group", I32T), ("dtype", I32T), ("page_min", P), ("page_max", P),
        ("page_capacity", I64), ("n_pages", I32T), ("packed", P), ("scale", P), ("minimum", P),
        ("int4_group_size", I32T), ("sink", I32T), ("block_size", I32T), ("b0_pages", I32T),
        ("top_p", DBL), ("old_length", I64), ("sink_end", I64), ("recent_start", I64), ("q", P),
        ("k_new", P), ("v_new", P), ("out", P), ("out_dtype", I32T), ("append", I32T),
        ("pages", P), ("union_pos", P), ("pos_stride", I64), ("union_count", P),
        ("head_count", P), ("head_pos", P), ("error_flag", P), ("select_workspace", P),
        ("select_workspace_bytes", SZ), ("attn_workspace", P), ("attn_workspace_bytes", SZ),
        ("max_rows_per_group", I32T), ("reuse", P), ("stage_k", P), ("stage_v", P),
        ("stage_rows", I64),
    ]


class RowReuse(ctypes.Structure):
    """tw_row_reuse of include/twilight_b200.h (previous-token row reuse)."""

    _fields_ = [
        ("row_map", P), ("map_stride", I64), ("prev_tag", ctypes.c_uint32),
        ("next_tag", ctypes.c_uint32), ("prev_k", P), ("prev_v", P), ("prev_rows", I64),
        ("next_k", P), ("next_v", P), ("rows_stride", I64), ("row_counts", P),
    ]


class PagedPool(ctypes.Structure):
    """tw_paged_pool of include/twilight_b200.h."""

    _fields_ = [
        ("k_pages", P), ("v_pages", P), ("page_stride", I64), ("head_stride", I64),
        ("token_stride", I64), ("num_pages", I64), ("page_size", I32T), ("kv_heads", I32T),
        ("head_dim", I32T), ("dtype", I32T),
    ]


class PagedStepArgs(ctypes.Structure):
    """tw_paged_step_args of include/twilight_b200.h."""

    _fields_ = [
        ("lens", P), ("new_lens", P), ("block_table", P), ("table_stride", I64),
        ("table_width", I32T), ("requests", I32T), ("page_size", I32T), ("tokens_cap", I32T),
        ("free_pages", P), ("num_pages", I64), ("free_count", P), ("kv_lens", P), ("cu_q", P),
        ("slots", P), ("positions", P), ("free_count_out", P), ("error_flag", P),
    ]


class PagedAttentionArgs(ctypes.Structure):
    """tw_paged_attention_args of include/twilight_b200.h."""

    _fields_ = [
        ("pool", PagedPool), ("q", P), ("q_token_stride", I64), ("q_head_stride", I64),
        ("block_table", P), ("table_stride", I64), ("table_width", I32T), ("requests", I32T),
        ("cu_q", P), ("kv_lens", P), ("tokens", I32T), ("q_heads", I32T), ("max_q_len", I32T),
        ("max_kv_len", I32T), ("window", I32T), ("softmax_scale", FLT), ("out", P),
        ("out_token_stride", I64), ("out_head_stride", I64), ("out_dtype", I32T),
        ("reserved", I32T), ("lse", P), ("error_flag", P), ("workspace", P),
        ("workspace_bytes", SZ),
    ]


class Rope(ctypes.Structure):
    """tw_rope of include/twilight_b200.h."""

    _fields_ = [("frequencies", P), ("pairs", I32T), ("interleaved", I32T), ("inverse", I32T),
                ("scale", FLT)]


class PagedRopeWriteArgs(ctypes.Structure):
    """tw_paged_rope_write_args of include/twilight_b200.h."""

    _fields_ = [
        ("pool", PagedPool), ("rope", Rope), ("q", P), ("q_token_stride", I64),
        ("q_head_stride", I64), ("k", P), ("k_token_stride", I64), ("k_head_stride", I64),
        ("v", P), ("v_token_stride", I64), ("v_head_stride", I64), ("q_out", P),
        ("q_out_token_stride", I64), ("q_out_head_stride", I64), ("positions", P), ("slots", P),
        ("tokens", I64), ("q_heads", I32T), ("reserved", I32T), ("row_weights", P),
        ("row_positions", P), ("error_flag", P),
    ]


class PagedWeightsArgs(ctypes.Structure):
    """tw_paged_weights_args of include/twilight_b200.h."""

    _fields_ = [
        ("pool", PagedPool), ("q", P), ("q_token_stride", I64), ("q_head_stride", I64),
        ("block_table", P), ("table_stride", I64), ("table_width", I32T), ("requests", I32T),
        ("cu_q", P), ("kv_lens", P), ("tokens", I32T), ("q_heads", I32T), ("max_q_len", I32T),
        ("max_kv_len", I32T), ("window", I32T), ("last", I32T), ("softmax_scale", FLT),
        ("reserved", I32T), ("lse", P), ("row_weights", P), ("error_flag", P),
    ]


class PagedEvictArgs(ctypes.Structure):
    """tw_paged_evict_args of include/twilight_b200.h."""

    _fields_ = [
        ("pool", PagedPool), ("layer_stride", I64), ("record_layer_stride", I64),
        ("row_weights", P), ("row_positions", P), ("block_table", P), ("table_stride", I64),
        ("table_width", I32T), ("requests", I32T), ("layers", I32T), ("max_len", I32T),
        ("sink", I32T), ("recent", I32T), ("lens", P), ("keep", P), ("offsets", P),
        ("lens_out", P), ("offsets_out", P), ("free_pages", P), ("free_count", P),
        ("free_count_out", P), ("error_flag", P),
    ]


# name -> (restype, argtypes); mirrors include/twilight_b200.h
SIGNATURES = {
    "tw_status_string": (ctypes.c_char_p, [I32]),
    "tw_last_cuda_error": (I32, []),
    "tw_abi_version": (I32, []),
    "tw_host_alloc_mapped": (I32, [SZ, ctypes.POINTER(P), ctypes.POINTER(P)]),
    "tw_host_alloc_mapped_numa": (I32, [SZ, I32, ctypes.POINTER(P), ctypes.POINTER(P),
                                        ctypes.POINTER(I32T)]),
    "tw_host_numa_node": (I32, [P, ctypes.POINTER(I32T)]),
    "tw_host_free": (I32, [P]),
    "tw_slab_write_rows": (I32, [P, I64, P, I64, I32, I64, I64, P]),
    "tw_host_device_pointer": (I32, [P, ctypes.POINTER(P)]),
    "tw_quest_page_metadata": (I32, [P, I64, I32, I32, I32, I32, I32, I32, I32, P, P, I64, P]),
    "tw_int4_pack": (I32, [P, I64, I32, I64, I32, I32, I32, P, P, P, I64, I64, P]),
    "tw_int4_pack_ex": (I32, [P, I64, I32, I64, I32, I32, I32, P, P, P, I64, I64, I32, P]),
    "tw_quest_score": (I32, [P, P, P, I32, I32, I32, I64, I32, I32, P, P]),
    "tw_topk_pages": (I32, [P, I32, I32, I32, P, P]),
    "tw_int4_qk": (I32, [P, P, P, P, I64, P, I32, I32, I32, I32, I32, I32, I32, I32, P, P]),
    "tw_top_p_union": (I32, [P, P, I32, I32, I32, I32, I32, DBL, I64, I64, I64, P, I64, P, P, P,
                             P, P]),
    "tw_select_layer_workspace_size": (SZ, [I32, I32, I32, I32, I32]),
    "tw_select_layer": (I32, [P, P, P, I64, I32, P, P, P, I64, I32, I32, I32, I32, I32, I32, I32,
                              I32, DBL, I64, I64, I64, P, P, I64, P, P, P, P, P, SZ, P]),
    "tw_gather_kv": (I32, [P, P, P, P, P, I64, I64, I64, P, P]),
    "tw_gather_union": (I32, [P, P, P, I64, I64, I32, I32, I64, P, I64, P, P, P, I32, I32, P, P, I64, P,
                              P, ctypes.POINTER(RowReuse), P]),
    "tw_gather_quest_heads": (I32, [P, P, P, I64, I64, I32, I32, I32, I64, I64, I64, I32, I32, P, I32, P,
                                    P, I32, I32, P, P, P, P]),
    "tw_append_token": (I32, [P, P, P, I64, I64, I32, I32, I64, P, P, I32, I32, I32, I32, P, P, I64, P, P,
                              P, I32, P]),
    "tw_decode_attention_workspace_size": (SZ, [I32, I32, I32, I32]),
    "tw_decode_attention": (I32, [P, P, P, P, I32, I32, I32, I32, I32, FLT, P, I32, P, P, SZ, P]),
    "tw_attend_union": (I32, [P, P, P, I64, I64, I32, I32, I64, P, I64, P, P, P, P, I32, I32, I32, I32, FLT,
                              P, I32, P, P, P, SZ, ctypes.POINTER(RowReuse), P]),
    "tw_twilight_decode_layer": (I32, [ctypes.POINTER(DecodeLayerArgs), P]),
    "tw_decode_layer_args_size": (SZ, []),
    "tw_row_reuse_size": (SZ, []),
    "tw_qkv_rope": (I32, [P, P, P, P, I32, I32, I32, I32, P, P, I32, P, P, P, P]),
    "tw_decode_attention_noalloc": (I32, [P, P, P, P, I32, I32, I32, I32, I32, FLT, P, I32, P, P]),
    "tw_paged_pool_size": (SZ, []),
    "tw_paged_step": (I32, [ctypes.POINTER(PagedStepArgs), P]),
    "tw_paged_step_args_size": (SZ, []),
    "tw_paged_write": (I32, [ctypes.POINTER(PagedPool), P, I64, I64, P, I64, I64, P, I64, P, P]),
    "tw_paged_attention_workspace_size": (SZ, [I32, I32, I32, I32, I32, I32, I32, I32]),
    "tw_paged_attention": (I32, [ctypes.POINTER(PagedAttentionArgs), P]),
    "tw_paged_attention_args_size": (SZ, []),
    "tw_rope_size": (SZ, []),
    "tw_rope_rows": (I32, [ctypes.POINTER(Rope), P, I64, I64, P, I64, I32, I32, I32, P, I64, I64,
                           P]),
    "tw_paged_rope_write": (I32, [ctypes.POINTER(PagedRopeWriteArgs), P]),
    "tw_paged_rope_write_args_size": (SZ, []),
    "tw_paged_step_at": (I32, [ctypes.POINTER(PagedStepArgs), P, P]),
    "tw_paged_weights": (I32, [ctypes.POINTER(PagedWeightsArgs), P]),
    "tw_paged_weights_args_size": (SZ, []),
    "tw_paged_evict": (I32, [ctypes.POINTER(PagedEvictArgs), P]),
    "tw_paged_evict_args_size": (SZ, []),
}

_lib = None
_binding = None


class TwilightError(RuntimeError):
    pass


def load():
    """Load the extension or raise (no fallback)."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise ImportError(
            f"{LIB_PATH.name} is missing: build it with "
            "`python twilight-cpu-gpu-offloading_b200/build.py` (there is no CPU fallback)")
    lib = ctypes.CDLL(str(LIB_PATH))
    for name, (restype, argtypes) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    _lib = lib
    return lib


def binding():
    """The compiled binding of the paged-cache calls (no fallback)."""
    global _binding
    if _binding is None:
        import torch  # noqa: F401  (its libraries first)

        load()
        if not BINDING_PATH.exists():
            raise ImportError(
                f"{BINDING_PATH.name} is missing: build it with "
                "`python twilight-cpu-gpu-offloading_b200/build.py` (there is no CPU fallback)")
        loader = importlib.machinery.ExtensionFileLoader("_binding", str(BINDING_PATH))
        spec = importlib.util.spec_from_file_location("_binding", BINDING_PATH, loader=loader)
        module = importlib.util.module_from_spec(spec)
        loader.exec_module(module)
        _binding = module
    return _binding


def status_string(status: int) -> str:
    return load().tw_status_string(status).decode()


def check(status: int, what: str = "") -> None:
    if status == TW_OK:
        return
    msg = f"{what}: {status_string(status)}" if what else status_string(status)
    if status == TW_ERR_CUDA:
        msg += f" (cudaError {load().tw_last_cuda_error()})"
        raise TwilightError(msg)
    if status in (TW_ERR_INVALID_INDEX, TW_ERR_BAD_ARG, TW_ERR_ORDER, TW_ERR_UNSUPPORTED):
        raise ValueError(msg)
    if status == TW_ERR_TIMEOUT:
        raise TimeoutError(msg)
    raise RuntimeError(msg)


def exported_symbols() -> list[str]:
    return list(SIGNATURES)
