"""The 8-bit cache's calls without a GPU: every refusal is a return code that comes before the device is touched, and the
workspace's size is plain arithmetic."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import kv_plain
from autorust_b200 import _abi

POOL = dict(k=0x1000, v=0x2000, k_scale=0x3000, v_scale=0x4000, k_mean=None, pages=10, Hkv=2, D=128, page=16, format=0)
BATCH = dict(page_table=0x5000, lengths=0x6000, starts=0x7000, table_stride=4, table_pages=4, B=3, T=9)


def pool(**kw):
    return _abi.KvPool(**{**POOL, **kw})


def batch(**kw):
    return _abi.KvBatch(**{**BATCH, **kw})


def strides(a, b):
    return (ctypes.c_int64 * 2)(a, b)


def calls(L, pl, bt, dtype=_abi.DTYPE_BF16, x=0x8000, y=0x9000, sx=(256, 128), sy=(256, 128)):
    """append, read and attention (eight query heads) with the same arguments."""
    sx, sy = (None if s is None else strides(*s) for s in (sx, sy))
    return [L.ar_kv_cache_append(pl, bt, dtype, x, sx, y, sy, None), L.ar_kv_cache_read(pl, bt, dtype, x, sx, y, sy, None),
            L.ar_kv_cache_attention(pl, bt, dtype, x, sx, y, sy, 8, 64, 1, None, 0, None)]


@pytest.mark.parametrize("pl,bt,kw,rc", [
    (dict(k=None), {}, {}, _abi.AR_ERR_NULL), (dict(v_scale=None), {}, {}, _abi.AR_ERR_NULL),
    (dict(pages=0), {}, {}, _abi.AR_ERR_SHAPE), (dict(Hkv=-1), {}, {}, _abi.AR_ERR_SHAPE),
    (dict(D=96), {}, {}, _abi.AR_ERR_UNSUPPORTED), (dict(page=8), {}, {}, _abi.AR_ERR_UNSUPPORTED),
    (dict(page=48), {}, {}, _abi.AR_ERR_UNSUPPORTED), (dict(page=256), {}, {}, _abi.AR_ERR_UNSUPPORTED),
    (dict(page=0), {}, {}, _abi.AR_ERR_UNSUPPORTED), (dict(format=2), {}, {}, _abi.AR_ERR_UNSUPPORTED),
    (dict(pages=2 ** 31), {}, {}, _abi.AR_ERR_UNSUPPORTED),
    (dict(k=0x1008), {}, {}, _abi.AR_ERR_ALIGNMENT), (dict(k_scale=0x3002), {}, {}, _abi.AR_ERR_ALIGNMENT),
    (dict(k_mean=0x3001), {}, {}, _abi.AR_ERR_ALIGNMENT),
    ({}, dict(page_table=None), {}, _abi.AR_ERR_NULL), ({}, dict(lengths=None), {}, _abi.AR_ERR_NULL),
    ({}, dict(B=0), {}, _abi.AR_ERR_SHAPE), ({}, dict(T=-1), {}, _abi.AR_ERR_SHAPE), ({}, dict(table_pages=0), {}, _abi.AR_ERR_SHAPE),
    ({}, dict(table_stride=3), {}, _abi.AR_ERR_SHAPE), ({}, dict(starts=None), {}, _abi.AR_ERR_SHAPE),  # 9 rows, 3 sequences
    ({}, dict(table_pages=2 ** 28, table_stride=2 ** 28), {}, _abi.AR_ERR_UNSUPPORTED), ({}, dict(T=2 ** 29), {}, _abi.AR_ERR_UNSUPPORTED),
    ({}, dict(lengths=0x6002), {}, _abi.AR_ERR_ALIGNMENT),
    ({}, {}, dict(dtype=7), _abi.AR_ERR_UNSUPPORTED), ({}, {}, dict(x=None), _abi.AR_ERR_NULL), ({}, {}, dict(sy=None), _abi.AR_ERR_NULL),
    ({}, {}, dict(x=0x8004), _abi.AR_ERR_ALIGNMENT), ({}, {}, dict(sx=(260, 128)), _abi.AR_ERR_ALIGNMENT),
    ({}, {}, dict(sx=(-256, 128)), _abi.AR_ERR_SHAPE),
])
def test_refusals(attn_lib, pl, bt, kw, rc):
    assert calls(attn_lib, pool(**pl), batch(**bt), **kw) == [rc] * 3


def test_refusals_of_single_calls(attn_lib):
    L = attn_lib
    assert L.ar_kv_cache_append(None, batch(), 1, 0x8000, strides(256, 128), 0x9000, strides(256, 128), None) == _abi.AR_ERR_NULL
    assert L.ar_kv_cache_append(pool(), None, 1, 0x8000, strides(256, 128), 0x9000, strides(256, 128), None) == _abi.AR_ERR_NULL
    # what is read may be broadcast, what is written may not
    assert L.ar_kv_cache_read(pool(), batch(), 1, 0x8000, strides(0, 128), 0x9000, strides(256, 128), None) == _abi.AR_ERR_SHAPE
    attend = lambda Hq=8, length=64, ws=None, n=0, bt=None, so=(1024, 128): L.ar_kv_cache_attention(
        pool(), bt or batch(), 1, 0x8000, strides(1024, 128), 0x9000, strides(*so), Hq, length, 1, ws, n, None)
    assert attend(Hq=7) == _abi.AR_ERR_SHAPE and attend(Hq=0) == _abi.AR_ERR_SHAPE and attend(length=0) == _abi.AR_ERR_SHAPE
    assert attend(so=(0, 128)) == _abi.AR_ERR_SHAPE
    assert attend(length=2 ** 31 - 1) == _abi.AR_ERR_UNSUPPORTED
    long = batch(table_pages=10000, table_stride=10000)
    need = L.ar_kv_cache_attention_workspace_bytes(pool(), long, 1, 8, 160000, 1)
    assert need > 0
    assert attend(length=160000, bt=long) == _abi.AR_ERR_WORKSPACE
    assert attend(length=160000, bt=long, ws=0x10000, n=need - 1) == _abi.AR_ERR_WORKSPACE
    assert attend(length=160000, bt=long, ws=0x10004, n=need) == _abi.AR_ERR_ALIGNMENT
    assert L.ar_kv_cache_attention_workspace_bytes(pool(D=96), long, 1, 8, 160000, 1) == 0


def test_no_rows_is_no_work(attn_lib):
    assert calls(attn_lib, pool(), batch(T=0)) == [_abi.AR_OK] * 3
    assert calls(attn_lib, pool(), batch(T=0), x=None, y=None) == [_abi.AR_OK] * 3  # (an empty tensor has no address)
    assert calls(attn_lib, pool(), batch(T=0), dtype=7) == [_abi.AR_ERR_UNSUPPORTED] * 3


def test_the_stride_of_a_single_row_or_head_is_not_looked_at(attn_lib):
    import torch
    ok = _abi.AR_ERR_NO_DEVICE if not torch.cuda.is_available() else None
    one = batch(B=1, T=1, starts=None)
    for sx in ((3, 128), (0, 128), (-7, 128)):
        if ok is not None:
            assert calls(attn_lib, pool(), one, sx=sx, sy=sx) == [ok] * 3
    assert calls(attn_lib, pool(), one, sx=(256, 3)) == [_abi.AR_ERR_ALIGNMENT] * 3


def test_no_device_is_an_error(attn_lib):
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert calls(attn_lib, pool(), batch()) == [_abi.AR_ERR_NO_DEVICE] * 3
    from autorust_b200 import ops
    with pytest.raises(ValueError, match="no CPU path"):
        ops.kv_cache(4, 2, 16, 64, device="cpu")
    with pytest.raises(ValueError, match="codes"):
        ops.KvCache(*(torch.zeros(4, 2, 16, 64) for _ in range(4)))


def test_page_errors_have_a_text():
    assert "page" in _abi.strerror(_abi.AR_ERR_PAGE)


def test_the_plain_cache_against_another_restatement():
    """kv_plain's own arithmetic: E4M3 codes against torch's conversion, a page rounded twice against direct arithmetic."""
    torch = pytest.importorskip("torch")
    x = np.clip(np.random.default_rng(0).standard_normal(20000).astype(np.float32) * 60, -448, 448)
    x = np.concatenate([x, x * 1e-3, x * 1e-5])
    assert np.array_equal(kv_plain.to_e4m3(x), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    c = kv_plain.PlainCache(1, 1, 16, 64, False)
    a, b = np.full((1, 1, 64), 1.0, np.float32), np.full((1, 1, 64), 2.0, np.float32)
    c.append(a, a, [[0]], [1], [0, 1])
    c.append(b, a, [[0]], [2], [0, 1])
    assert (c.codes[0][0, 0, 0] == 64).all() and (c.codes[0][0, 0, 1] == 127).all()  # 127 / 2 rounds to the even 64
    assert (c.codes[1][0, 0, :2] == 127).all()
