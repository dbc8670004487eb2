"""Paged cache entry points: struct layouts and the argument checks that run on the
host (no kernel is launched)."""

from __future__ import annotations

import ctypes

import pytest


def test_struct_sizes(tw):
    lib, L = tw.load_library(), tw._lib
    assert ctypes.sizeof(L.PagedPool) == lib.tw_paged_pool_size()
    assert ctypes.sizeof(L.PagedStepArgs) == lib.tw_paged_step_args_size()
    assert ctypes.sizeof(L.PagedAttentionArgs) == lib.tw_paged_attention_args_size()


def pool(L, **change):
    fields = dict(k_pages=1 << 20, v_pages=1 << 21, page_stride=4096, head_stride=2048,
                  token_stride=128, num_pages=10, page_size=16, kv_heads=2, head_dim=128,
                  dtype=L.TW_F16)
    return L.PagedPool(**{**fields, **change})


def attention(L, **change):
    fields = dict(pool=pool(L), q=1 << 20, q_token_stride=1024, q_head_stride=128,
                  block_table=1 << 20, table_stride=4, table_width=4, requests=2, cu_q=1 << 20,
                  kv_lens=1 << 20, tokens=0, q_heads=8, max_q_len=1, max_kv_len=64, window=0,
                  softmax_scale=0.1, out=1 << 20, out_token_stride=1024, out_head_stride=128,
                  out_dtype=L.TW_F16)
    return L.PagedAttentionArgs(**{**fields, **change})


@pytest.mark.parametrize("change,status", [
    (dict(head_dim=64), "TW_ERR_UNSUPPORTED"), (dict(dtype=2), "TW_ERR_UNSUPPORTED"),
    (dict(k_pages=None), "TW_ERR_BAD_ARG"), (dict(k_pages=(1 << 20) + 8), "TW_ERR_BAD_ARG"),
    (dict(num_pages=0), "TW_ERR_BAD_ARG"), (dict(page_size=0), "TW_ERR_BAD_ARG"),
    (dict(token_stride=132), "TW_ERR_BAD_ARG"), (dict(head_stride=0), "TW_ERR_BAD_ARG"),
    (dict(page_stride=-8), "TW_ERR_BAD_ARG"), (dict(num_pages=1 << 31), "TW_ERR_BAD_ARG")])
def test_pool_checks(tw, change, status):
    lib, L = tw.load_library(), tw._lib
    p = pool(L, **change)
    want = getattr(L, status)
    assert lib.tw_paged_write(ctypes.byref(p), 16, 128, 128, 16, 128, 128, 16, 1, None, None) == want
    args = attention(L, pool=p, tokens=1)
    assert lib.tw_paged_attention(ctypes.byref(args), None) == want


@pytest.mark.parametrize("change,status", [
    (dict(q=None), "TW_ERR_BAD_ARG"), (dict(q=(1 << 20) + 2), "TW_ERR_BAD_ARG"),
    (dict(cu_q=None), "TW_ERR_BAD_ARG"), (dict(out=None), "TW_ERR_BAD_ARG"),
    (dict(requests=0), "TW_ERR_BAD_ARG"), (dict(q_heads=7), "TW_ERR_BAD_ARG"),
    (dict(q_heads=0), "TW_ERR_BAD_ARG"), (dict(q_heads=130), "TW_ERR_UNSUPPORTED"),
    (dict(table_stride=3), "TW_ERR_BAD_ARG"), (dict(table_width=0), "TW_ERR_BAD_ARG"),
    (dict(window=-1), "TW_ERR_BAD_ARG"), (dict(softmax_scale=0.0), "TW_ERR_BAD_ARG"),
    (dict(softmax_scale=float("nan")), "TW_ERR_BAD_ARG"),
    (dict(out_dtype=1), "TW_ERR_BAD_ARG"), (dict(q_token_stride=4), "TW_ERR_BAD_ARG"),
    (dict(out_head_stride=0), "TW_ERR_BAD_ARG"), (dict(tokens=-1), "TW_ERR_BAD_ARG"),
    (dict(reserved=1), "TW_ERR_BAD_ARG")])
def test_attention_checks(tw, change, status):
    lib, L = tw.load_library(), tw._lib
    args = attention(L, **{"tokens": 3, **change})
    assert lib.tw_paged_attention(ctypes.byref(args), None) == getattr(L, status)


def test_null_and_empty_calls(tw):
    lib, L = tw.load_library(), tw._lib
    assert lib.tw_paged_attention(None, None) == L.TW_ERR_BAD_ARG
    assert lib.tw_paged_step(None, None) == L.TW_ERR_BAD_ARG
    assert lib.tw_paged_write(None, 16, 128, 128, 16, 128, 128, 16, 1, None, None) == L.TW_ERR_BAD_ARG
    p, a = pool(L), attention(L)
    assert lib.tw_paged_write(ctypes.byref(p), None, 128, 128, None, 128, 128, None, 0, None,
                              None) == L.TW_OK
    assert lib.tw_paged_attention(ctypes.byref(a), None) == L.TW_OK
    assert lib.tw_paged_step(ctypes.byref(L.PagedStepArgs()), None) == L.TW_ERR_BAD_ARG


def test_binding_checks_its_arguments(tw):
    b = tw._lib.binding()
    for call, n in ((b.paged_step, 12), (b.paged_write, 6), (b.paged_attention, 15)):
        with pytest.raises(TypeError):
            call()
        args = [1 if n == 12 and i == 5 or n == 15 and i in (6, 7, 8) else None for i in range(n)]
        assert call(*args) == -1  # no tensors
    with pytest.raises(ValueError):
        b.paged_step(*[1 << 40 if i == 5 else None for i in range(12)])
    with pytest.raises(TypeError):
        b.paged_attention(*[None] * 15)


def test_cpu_tensors_are_refused(tw):
    import torch

    pages = torch.zeros(2, 1, 8, 128, dtype=torch.float16)
    rows = torch.zeros(1, 1, 128, dtype=torch.float16)
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        tw.ops.paged_write(rows, rows, torch.zeros(1, dtype=torch.int64), pages, pages)
    with pytest.raises(ValueError, match="CUDA"):
        tw.ops.paged_attention(rows, pages, pages, one[None], torch.zeros(2, dtype=torch.int32),
                               one, max_q_len=1, max_kv_len=1)
    with pytest.raises(ValueError, match="CUDA"):
        tw.ops.paged_step(one, one, one[None], one, one, page_size=16, kv_lens=one, cu_q=one,
                          slots=one.long(), positions=one, free_count_out=one)


@pytest.mark.parametrize("q_heads,kv_heads", [(32, 8), (8, 8), (64, 8), (8, 1), (128, 128)])
@pytest.mark.parametrize("max_kv", [1, 4097, 131072, 1 << 20, 2 ** 31 - 1])
def test_workspace_has_a_bound(tw, q_heads, kv_heads, max_kv):
    """Whatever the requests and their longest: 256 MiB of partial results of requests with
    few tokens (split only as far as that allows), and of the others at most one of 256 rows
    for each of two CTAs per SM, 132 numbers a row."""
    lib = tw.load_library()
    most = (256 << 20) + 2 * 148 * 256 * 132 * 4
    for requests in (1, 2, 16, 256, 700, 8192):
        for tokens in (requests, requests + 3000, 16384):
            for max_q in (1, 2, 4, 16, 3000):
                need = lib.tw_paged_attention_workspace_size(requests, tokens, q_heads, kv_heads,
                                                             max_q, max_kv, 0, 128)
                assert need <= most, (requests, tokens, max_q, need)
