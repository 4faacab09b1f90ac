"""How cache attention calls are divided (ar_kv_cache_attention_plan; no GPU needed): the plan is what the workspace is sized for, and
refuses what the call refuses."""
from __future__ import annotations

import pytest

from autorust_b200 import _abi


@pytest.fixture(scope="module", autouse=True)
def _lib(attn_lib):
    return attn_lib


def pool(**kw):
    return _abi.KvPool(**{**dict(k=0x1000, v=0x2000, k_scale=0x3000, v_scale=0x4000, k_mean=None, pages=10, Hkv=2, D=128, page=16,
                                 format=0), **kw})


def batch(B, T, width, starts=0x7000):
    return _abi.KvBatch(0x5000, 0x6000, starts, width, width, B, T)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [_abi.DTYPE_F32, _abi.DTYPE_BF16])
@pytest.mark.parametrize("B,T,Hq,length", [(1, 1, 8, 100), (8, 8, 8, 8192), (1, 1, 64, 131072), (16, 80, 32, 3001), (2, 2048, 8, 16384),
                                           (4, 512, 8, 16384), (40, 3000, 4, 700), (1, 4096, 2, 4096)])
def test_plans_are_what_the_workspace_is_for(D, dtype, B, T, Hq, length):
    width = -(-length // 16)
    at = (pool(D=D), batch(B, T, width), dtype, Hq, length)
    rows, ctas, parts = _abi.kv_plan(*at, True)
    need = _abi.load().ar_kv_cache_attention_workspace_bytes(*at, 1)
    if rows == 256:
        assert dtype == _abi.DTYPE_BF16 and ctas == 0 and 1 <= parts <= 16
        assert need == (parts * T * Hq * (D + 4) * 4 if parts > 1 else 0)
    else:
        assert rows in (8, 16) and parts == 1
        assert need == ctas * (16 + 2 * 4 * rows * (D + 4))


def test_every_form_is_taken():
    forms = {tuple(f(x) for f, x in zip((int, bool, lambda p: p > 1), _abi.kv_plan(pool(), batch(B, T, 8192), 1, 8, length, True)))
             for B, T, length in ((1, 1, 100), (1, 1, 100000), (2, 6, 300), (2, 6, 100000), (8, 8192, 1024), (1, 256, 100000))}
    assert forms == {(8, False, False), (8, True, False), (16, False, False), (16, True, False), (256, False, False), (256, False, True)}


def test_refusals_and_empty_calls():
    L = _abi.load()
    plan = lambda p, b, out, Hq=8, dtype=1: L.ar_kv_cache_attention_plan(p, b, dtype, Hq, 64, 1, out)
    import ctypes
    out = (ctypes.c_int32 * 3)(7, 7, 7)
    assert plan(pool(), batch(3, 9, 4), None) == _abi.AR_ERR_NULL
    assert plan(pool(D=96), batch(3, 9, 4), out) == _abi.AR_ERR_UNSUPPORTED
    assert plan(pool(), batch(3, 9, 4), out, Hq=7) == _abi.AR_ERR_SHAPE
    assert plan(pool(), batch(3, 9, 4), out, dtype=5) == _abi.AR_ERR_UNSUPPORTED
    assert list(out) == [7, 7, 7]
    assert plan(pool(), batch(3, 0, 4), out) == _abi.AR_OK and list(out) == [0, 0, 0]
