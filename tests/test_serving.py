"""Refusals of the serving calls: shapes, types and layouts that the checks turn away before any device call
(no GPU needed), and the rotary table."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


def _plan(pkg, **kw):
    d = pkg.AttnCachePlan()
    d.page_size, d.B, d.W, d.num_pages, d.tokens, d.table_stride = 16, 4, 8, 64, 10, 8
    for f in ("lengths", "targets", "block_table", "free_pages", "free_count", "lengths_out", "free_count_out", "starts",
              "positions", "slots"):
        setattr(d, f, 0x10000)
    for k, v in kw.items():
        setattr(d, k, v)
    return pkg.lib().attn_cache_plan(ctypes.byref(d), None)


def _append(pkg, **kw):
    d = pkg.AttnCacheAppend()
    d.dtype = d.cache_dtype = pkg.ATTN_BF16
    d.page_size, d.N, d.T, d.Hkv, d.D, d.num_pages = 16, 4, 4, 2, 64, 8
    d.k_stride[:] = d.v_stride[:] = [128, 64]
    d.k_cache_stride[:] = d.v_cache_stride[:] = [2048, 1024, 64]
    for f in ("k", "v", "k_cache", "v_cache", "slots"):
        setattr(d, f, 0x10000)
    d.k_descale = d.v_descale = 1.0
    for k, v in kw.items():
        if isinstance(v, list):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    return pkg.lib().attn_cache_append(ctypes.byref(d), None)


def _rotary(pkg, **kw):
    d = pkg.AttnRotary()
    d.dtype, d.num_axes, d.B, d.N, d.Hq, d.Hk, d.D, d.R = pkg.ATTN_BF16, 1, 1, 4, 2, 1, 64, 64
    for f in ("q", "k", "qo", "ko", "positions", "freqs"):
        setattr(d, f, 0x10000)
    for k, v in kw.items():
        setattr(d, k, v)
    return pkg.lib().attn_rotary(ctypes.byref(d), None)


def _tree(pkg, **kw):
    d = pkg.AttnTree()
    d.dtype = d.cache_dtype = pkg.ATTN_BF16
    d.page_size, d.B, d.T, d.Hq, d.Hkv, d.D, d.W, d.num_pages, d.max_new = 16, 2, 6, 8, 2, 128, 4, 8, 3
    d.q_stride[:] = d.o_stride[:] = [1024, 128]
    d.k_stride[:] = d.v_stride[:] = [256, 128]
    d.k_cache_stride[:] = d.v_cache_stride[:] = [4096, 2048, 128]
    d.table_stride = 4
    for f in ("q", "k_new", "v_new", "k_cache", "v_cache", "o", "block_table", "lengths", "starts"):
        setattr(d, f, 0x10000)
    d.scale, d.k_descale, d.v_descale = 0.1, 1.0, 1.0
    for k, v in kw.items():
        if isinstance(v, list):
            getattr(d, k)[:] = v
        else:
            setattr(d, k, v)
    return pkg.lib().attn_tree_fwd(ctypes.byref(d), None)


@pytest.mark.parametrize("kw,code", [
    ({"flags": 2}, -1), ({"B": -1}, -2), ({"page_size": 24}, -8), ({"page_size": 8}, -8), ({"page_size": 2048}, -8),
    ({"B": 8193}, -8), ({"W": 1 << 28}, -2), ({"tokens": 1 << 31}, -2), ({"table_stride": 7}, -3), ({"slots": None}, -1),
    ({"free_count": None}, -1), ({"lengths": None}, -1),
])
def test_plan_refuses(pkg, kw, code):
    assert _plan(pkg, **kw) == code and pkg.last_error()


@pytest.mark.parametrize("kw,code", [
    ({"flags": 4}, -1), ({"N": -1}, -2), ({"dtype": 0}, -4), ({"cache_dtype": 3}, -4), ({"page_size": 17}, -8),
    ({"D": 72}, -8), ({"N": 5}, -2), ({"slots": None}, -1), ({"k": None}, -1), ({"k": 0x10008}, -5),
    ({"v_cache": 0x10004}, -5), ({"k_stride": [132, 64]}, -5), ({"k_cache_stride": [2048, 1024, 68]}, -5),
    ({"k_descale": 2.0}, -4), ({"cache_dtype": 2, "k_descale": 0.0}, -1),
    ({"cache_dtype": 2, "v_descale": float("inf")}, -1), ({"cache_dtype": 2, "v_cache_stride": [2048, 1024, 72]}, -5),
])
def test_append_refuses(pkg, kw, code):
    assert _append(pkg, **kw) == code and pkg.last_error()


@pytest.mark.parametrize("kw,code", [
    ({"flags": 8}, -1), ({"N": -1}, -2), ({"dtype": 2}, -4), ({"R": 63}, -2), ({"R": 66}, -2), ({"D": 2000}, -8),
    ({"num_axes": 0}, -2), ({"q": None}, -1), ({"freqs": None}, -1), ({"k": 0x10001}, -5),
])
def test_rotary_refuses(pkg, kw, code):
    assert _rotary(pkg, **kw) == code and pkg.last_error()


@pytest.mark.parametrize("kw,code", [
    ({"flags": 2}, -1), ({"T": -1}, -2), ({"dtype": 0}, -4), ({"cache_dtype": 3}, -4), ({"page_size": 20}, -8),
    ({"D": 96}, -8), ({"D": 64, "cache_dtype": 2}, -8), ({"Hkv": 3}, -2), ({"Hq": 130, "Hkv": 2}, -8),
    ({"q": None}, -1), ({"starts": None}, -1), ({"block_table": None}, -1), ({"table_stride": 3}, -3),
    ({"mask": 0x10000, "mask_stride": 2}, -3), ({"scale": float("nan")}, -1), ({"q": 0x10002}, -5),
    ({"q_stride": [1024, 129]}, -5), ({"v_cache_stride": [4096, 2048, 130]}, -5), ({"k_descale": 0.5}, -4),
    ({"cache_dtype": 2, "k_descale": -1.0}, -1), ({"W": 1 << 28}, -2),
])
def test_tree_refuses(pkg, kw, code):
    assert _tree(pkg, **kw) == code and pkg.last_error()


def test_null_descriptors(pkg):
    L = pkg.lib()
    for name in ("attn_cache_plan", "attn_cache_append", "attn_rotary", "attn_tree_fwd"):
        assert getattr(L, name)(None, None) == -1


def test_empty_calls_do_nothing(pkg):
    """No rows: nothing is launched, so no device is needed and pointers are not looked at."""
    assert _append(pkg, N=0, k=None) == 0
    assert _rotary(pkg, N=0) == 0
    assert _tree(pkg, T=0, q=None) == 0 and _tree(pkg, B=0) == 0 and _tree(pkg, max_new=0) == 0


def test_host_tensors_are_refused(pkg):
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cache = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    table = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(pkg.VerifyError, match="CUDA"):
        pkg.cache_plan(i, i, table, i, i[:1], 16, 4)
    with pytest.raises(pkg.VerifyError, match="CUDA"):
        pkg.cache_append(x, x, cache, cache, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(pkg.VerifyError, match="CUDA"):
        pkg.rotary(x, x, torch.zeros(4, dtype=torch.int32), pkg.rotary_table(64, device="cpu"))
    with pytest.raises(pkg.VerifyError, match="CUDA"):
        pkg.fused_tree(x, x, x, cache, cache, table, i, torch.zeros(3, dtype=torch.int32), 0.1)


def test_shapes_are_checked_first(pkg):
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(pkg.VerifyError, match="tokens, heads, head_dim"):
        pkg.fused_tree(x[0], x, x, x, x, x, x, x, 0.1)
    with pytest.raises(pkg.VerifyError, match="K seq_len must equal Q seq_len"):
        pkg.fused_tree(x, x[:3], x[:3], x, x, x, x, x, 0.1)
    with pytest.raises(pkg.VerifyError, match="K head_dim must equal Q head_dim"):
        pkg.fused_tree(x, x[..., :32], x[..., :32], x, x, x, x, x, 0.1)
    with pytest.raises(pkg.VerifyError, match="go together"):
        pkg.fused(x[0], x[0], x[0], 0.1, positions=torch.zeros(2))
    with pytest.raises(pkg.VerifyError, match="Q or K"):
        pkg.rotary(None, None, None, None)


def test_rotary_table(pkg):
    t = pkg.rotary_table(16, [3, 3, 2], 100.0, device="cpu")
    assert t.axes.tolist() == [0, 0, 0, 1, 1, 1, 2, 2]
    assert torch.equal(t.freqs, 100.0 ** (-torch.arange(8, dtype=torch.float64) / 8))
    assert pkg.rotary_table(16, [3, 3, 2], interleaved=True, device="cpu").axes.tolist() == [0, 1, 2, 0, 1, 2, 0, 1]
    assert pkg.rotary_table(8, device="cpu").axes.tolist() == [0] * 4
    for dim, sections in ((15, None), (16, [4, 3]), (16, [9, -1]), (0, None)):
        with pytest.raises(pkg.VerifyError):
            pkg.rotary_table(dim, sections, device="cpu")
