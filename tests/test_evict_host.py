"""Rotary positions, attention weights and eviction: struct layouts, the argument checks
that run on the host (no kernel is launched), and the frequencies' formulas."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch


def test_struct_sizes(tw):
    lib, L = tw.load_library(), tw._lib
    assert ctypes.sizeof(L.Rope) == lib.tw_rope_size()
    assert ctypes.sizeof(L.PagedRopeWriteArgs) == lib.tw_paged_rope_write_args_size()
    assert ctypes.sizeof(L.PagedWeightsArgs) == lib.tw_paged_weights_args_size()
    assert ctypes.sizeof(L.PagedEvictArgs) == lib.tw_paged_evict_args_size()


A = 1 << 20  # an aligned address that nothing reads


def pool(L, **change):
    fields = dict(k_pages=A, v_pages=2 * A, page_stride=4096, head_stride=2048, token_stride=128,
                  num_pages=10, page_size=16, kv_heads=2, head_dim=128, dtype=L.TW_F16)
    return L.PagedPool(**{**fields, **change})


def rope(L, **change):
    return L.Rope(**{**dict(frequencies=A, pairs=64, interleaved=0, inverse=0, scale=1.0),
                     **change})


@pytest.mark.parametrize("change", [dict(pairs=65), dict(pairs=-1), dict(frequencies=None),
                                    dict(interleaved=2), dict(inverse=-1),
                                    dict(scale=float("inf")), dict(scale=float("nan"))])
def test_rope_checks(tw, change):
    lib, L = tw.load_library(), tw._lib
    bad = rope(L, **change)
    call = lambda r, **k: lib.tw_rope_rows(  # noqa: E731
        ctypes.byref(r), k.get("x", A), k.get("token", 512), k.get("head", 128),
        k.get("positions", A), k.get("tokens", 1), k.get("heads", 4), k.get("dim", 128),
        k.get("dtype", 0), k.get("out", A), 512, 128, None)
    assert call(bad) == L.TW_ERR_BAD_ARG
    args = L.PagedRopeWriteArgs(pool=pool(L), rope=bad, tokens=1)
    assert lib.tw_paged_rope_write(ctypes.byref(args), None) == L.TW_ERR_BAD_ARG
    good = rope(L)
    assert call(good, tokens=0) == L.TW_OK
    assert call(good, heads=0) == L.TW_OK
    assert call(good, tokens=-1) == L.TW_ERR_BAD_ARG
    assert call(good, x=None) == L.TW_ERR_BAD_ARG
    assert call(good, x=A + 8) == L.TW_ERR_BAD_ARG
    assert call(good, token=510) == L.TW_ERR_BAD_ARG
    assert call(good, head=-128) == L.TW_ERR_BAD_ARG
    assert call(good, positions=None) == L.TW_ERR_BAD_ARG
    assert call(good, out=None) == L.TW_ERR_BAD_ARG
    assert call(good, dim=64) == L.TW_ERR_UNSUPPORTED
    assert call(good, dtype=2) == L.TW_ERR_UNSUPPORTED


@pytest.mark.parametrize("change,status", [
    (dict(tokens=0), "TW_OK"), (dict(tokens=-1), "TW_ERR_BAD_ARG"),
    (dict(q=None), "TW_ERR_BAD_ARG"), (dict(q_out=None), "TW_ERR_BAD_ARG"),
    (dict(k=None), "TW_ERR_BAD_ARG"), (dict(v=A + 2), "TW_ERR_BAD_ARG"),
    (dict(k_head_stride=100), "TW_ERR_BAD_ARG"), (dict(slots=None), "TW_ERR_BAD_ARG"),
    (dict(positions=None), "TW_ERR_BAD_ARG"), (dict(q_heads=-1), "TW_ERR_BAD_ARG"),
    (dict(reserved=1), "TW_ERR_BAD_ARG")])
def test_rope_write_checks(tw, change, status):
    lib, L = tw.load_library(), tw._lib
    fields = dict(pool=pool(L), rope=rope(L), q=A, q_token_stride=1024, q_head_stride=128, k=A,
                  k_token_stride=256, k_head_stride=128, v=A, v_token_stride=256,
                  v_head_stride=128, q_out=A, q_out_token_stride=1024, q_out_head_stride=128,
                  positions=A, slots=A, tokens=1, q_heads=8)
    args = L.PagedRopeWriteArgs(**{**fields, **change})
    assert lib.tw_paged_rope_write(ctypes.byref(args), None) == getattr(L, status)


@pytest.mark.parametrize("change,status", [
    (dict(tokens=0), "TW_OK"), (dict(tokens=-1), "TW_ERR_BAD_ARG"),
    (dict(q=None), "TW_ERR_BAD_ARG"), (dict(q=A + 8), "TW_ERR_BAD_ARG"),
    (dict(lse=None), "TW_ERR_BAD_ARG"), (dict(row_weights=None), "TW_ERR_BAD_ARG"),
    (dict(cu_q=None), "TW_ERR_BAD_ARG"), (dict(kv_lens=None), "TW_ERR_BAD_ARG"),
    (dict(requests=0), "TW_ERR_BAD_ARG"), (dict(q_heads=7), "TW_ERR_BAD_ARG"),
    (dict(q_heads=130), "TW_ERR_UNSUPPORTED"), (dict(table_stride=3), "TW_ERR_BAD_ARG"),
    (dict(window=-1), "TW_ERR_BAD_ARG"), (dict(last=-1), "TW_ERR_BAD_ARG"),
    (dict(max_q_len=-1), "TW_ERR_BAD_ARG"), (dict(max_kv_len=-1), "TW_ERR_BAD_ARG"),
    (dict(softmax_scale=0.0), "TW_ERR_BAD_ARG"),
    (dict(softmax_scale=float("inf")), "TW_ERR_BAD_ARG"),
    (dict(q_token_stride=12), "TW_ERR_BAD_ARG"), (dict(reserved=1), "TW_ERR_BAD_ARG")])
def test_weights_checks(tw, change, status):
    lib, L = tw.load_library(), tw._lib
    fields = dict(pool=pool(L), q=A, q_token_stride=1024, q_head_stride=128, block_table=A,
                  table_stride=4, table_width=4, requests=2, cu_q=A, kv_lens=A, tokens=1,
                  q_heads=8, max_q_len=1, max_kv_len=64, softmax_scale=0.1, lse=A, row_weights=A)
    args = L.PagedWeightsArgs(**{**fields, **change})
    assert lib.tw_paged_weights(ctypes.byref(args), None) == getattr(L, status)
    if status != "TW_OK":
        bad = L.PagedWeightsArgs(**{**fields, "pool": pool(L, page_size=12)})
        assert lib.tw_paged_weights(ctypes.byref(bad), None) == L.TW_ERR_UNSUPPORTED


@pytest.mark.parametrize("change,status", [
    (dict(requests=0), "TW_OK"), (dict(requests=-1), "TW_ERR_BAD_ARG"),
    (dict(requests=8193), "TW_ERR_UNSUPPORTED"),
    (dict(max_len=(1 << 21) + 1), "TW_ERR_UNSUPPORTED"),
    (dict(max_len=-1), "TW_ERR_BAD_ARG"), (dict(sink=-1), "TW_ERR_BAD_ARG"),
    (dict(recent=-1), "TW_ERR_BAD_ARG"), (dict(layers=0), "TW_ERR_BAD_ARG"),
    (dict(layers=2), "TW_ERR_BAD_ARG"), (dict(layers=2, layer_stride=12, record_layer_stride=320),
                                         "TW_ERR_BAD_ARG"),
    (dict(row_weights=None), "TW_ERR_BAD_ARG"), (dict(row_positions=None), "TW_ERR_BAD_ARG"),
    (dict(lens=None), "TW_ERR_BAD_ARG"), (dict(keep=None), "TW_ERR_BAD_ARG"),
    (dict(offsets=None), "TW_ERR_BAD_ARG"), (dict(lens_out=None), "TW_ERR_BAD_ARG"),
    (dict(offsets_out=None), "TW_ERR_BAD_ARG"), (dict(table_width=0), "TW_ERR_BAD_ARG"),
    (dict(free_count=None), "TW_ERR_BAD_ARG"), (dict(free_pages=None), "TW_ERR_BAD_ARG"),
    (dict(free_count_out=None), "TW_ERR_BAD_ARG"),
    # outputs over inputs, or over each other
    (dict(lens_out=3 * A + 4), "TW_ERR_BAD_ARG"), (dict(offsets_out=3 * A), "TW_ERR_BAD_ARG"),
    (dict(lens_out=5 * A + 4), "TW_ERR_BAD_ARG"), (dict(free_count_out=9 * A), "TW_ERR_BAD_ARG"),
    (dict(free_pages=3 * A - 36), "TW_ERR_BAD_ARG"), (dict(lens_out=7 * A), "TW_ERR_BAD_ARG")])
def test_evict_checks(tw, change, status):
    lib, L = tw.load_library(), tw._lib
    fields = dict(pool=pool(L), row_weights=A, row_positions=A, block_table=A, table_stride=4,
                  table_width=4, requests=2, layers=1, max_len=64, sink=1, recent=2, lens=3 * A,
                  keep=4 * A, offsets=5 * A, lens_out=6 * A, offsets_out=7 * A, free_pages=8 * A,
                  free_count=9 * A, free_count_out=10 * A)
    args = L.PagedEvictArgs(**{**fields, **change})
    assert lib.tw_paged_evict(ctypes.byref(args), None) == getattr(L, status)


def test_step_offsets_apart(tw):
    lib, L = tw.load_library(), tw._lib
    args = L.PagedStepArgs(lens=A, new_lens=2 * A, block_table=3 * A, table_stride=4, table_width=4,
                           requests=2, page_size=16, tokens_cap=0, free_pages=4 * A, num_pages=8,
                           free_count=5 * A, kv_lens=6 * A, cu_q=7 * A, free_count_out=8 * A)
    for offsets in (A, 2 * A, 6 * A):
        assert lib.tw_paged_step_at(ctypes.byref(args), offsets, None) == L.TW_ERR_BAD_ARG


def test_cpu_tensors_are_rejected(tw):
    ops = tw.ops
    f, _ = ops.rope_frequencies(128)
    x = torch.zeros(2, 4, 128, dtype=torch.float16)
    pos = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope(x, pos, f)
    with pytest.raises(ValueError, match="layout"):
        ops.rope(x, pos, f, layout="quarter")
    pages = torch.zeros(3, 2, 16, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_rope_write(x, x[:, :2], x[:, :2], pos, pos.long(), f, pages, pages)
    i = torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_weights(x, pages, table, pos, i, x[..., 0].float(), pages[..., 0].float(),
                          max_q_len=1, max_kv_len=1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_evict(pages, pages, pages[..., 0].float(), pages[..., 0].int(), table, i, i, i,
                        max_len=4, sink=0, recent=0, lens_out=i, offsets_out=i)


def test_frequencies(tw):
    """Each scaling against its formula, written pair by pair."""
    f = tw.ops.rope_frequencies
    base, dims, factor, original = 500000.0, 96, 8.0, 8192
    plain = [base ** (-2 * n / dims) for n in range(dims // 2)]
    got, scale = f(dims, base=base)
    assert got.dtype == torch.float64 and scale == 1.0
    assert got.tolist() == pytest.approx(plain, rel=1e-12)
    got, _ = f(dims, base=base, scaling={"type": "linear", "factor": factor})
    assert got.tolist() == pytest.approx([x / factor for x in plain], rel=1e-12)
    got, _ = f(dims, base=base, scaling={"type": "ntk", "factor": factor})
    assert got[0] == 1.0 and got[-1].item() == pytest.approx(plain[-1] / factor, rel=1e-12)
    got, _ = f(dims, base=base, scaling={"type": "bands", "factor": factor, "original": original,
                                         "low": 1.0, "high": 4.0})
    for x, y in zip(plain, got.tolist()):
        turns = original * x / (2 * math.pi)
        if turns >= 4:
            want = x
        elif turns <= 1:
            want = x / factor
        else:
            smooth = (turns - 1) / 3
            want = (1 - smooth) * x / factor + smooth * x
        assert y == pytest.approx(want, rel=1e-12)
    got, scale = f(dims, base=base, scaling={"type": "yarn", "factor": factor,
                                             "original": original})
    assert scale == pytest.approx(0.1 * math.log(factor) + 1)

    def at(turns):
        return dims * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = math.floor(at(32)), math.ceil(at(1))
    for n, (x, y) in enumerate(zip(plain, got.tolist())):
        slowed = min(1.0, max(0.0, (n - low) / (high - low)))
        assert y == pytest.approx(x / factor * slowed + x * (1 - slowed), rel=1e-12)
    assert f(0)[0].numel() == 0 and f(2)[0].tolist() == [1.0]
    assert f(2, scaling={"type": "ntk", "factor": 2.0})[0].tolist() == [1.0]
    assert f(64, scaling={"type": "yarn", "factor": 2.0, "original": 4096, "scale": 1.5})[1] == 1.5
    for bad in (dict(dims=3), dict(dims=130), dict(base=1.0), dict(scaling={"type": "dynamic"}),
                dict(scaling={"type": "linear"}), dict(scaling={"type": "linear", "factor": 0.5}),
                dict(scaling={"type": "bands", "factor": 2.0}),
                dict(scaling={"type": "linear", "factor": 2.0, "low": 1}),
                dict(scaling={"type": "yarn", "factor": 2.0, "original": 8, "fast": 1, "slow": 2})):
        with pytest.raises(ValueError):
            f(**bad)
