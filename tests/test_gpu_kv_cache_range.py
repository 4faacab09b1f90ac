"""The cache attention over the range of f32: logits of any finite size in every form of the kernels."""
from __future__ import annotations

import numpy as np
import pytest

from kv_forms import BF16_ONLY, FORMS, assert_close, assert_form, expect
from test_gpu_kv_cache import Setup

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(attn_lib):
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device: there is no fallback path to test")
    from autorust_b200 import ops as _ops
    return _ops


CASES = [(form, f32) for form in FORMS for f32 in (False, True) if not (f32 and form in BF16_ONLY)]


def fill(s, lengths, k, scale_v=None):
    """k [T, Hkv, D] f32 of all tokens, values whose size differs from page to page, into the pool and its plain twin."""
    torch = s.torch
    T, kind = sum(lengths), torch.float32 if s.f32 else torch.bfloat16
    v = s.rng.standard_normal((T, s.Hkv, s.D)).astype(np.float32)
    v *= (np.resize([1.0, 0.3, 2.5, 0.9] if scale_v is None else scale_v, -(-T // s.page)).repeat(s.page)[:T, None, None]).astype(np.float32)
    kt, vt = (torch.from_numpy(x).cuda().to(kind) for x in (k, v))
    starts = np.concatenate([[0], np.cumsum(lengths)])
    s.ops.kv_cache_append(s.cache, kt, vt, s.dtable, s.ints(lengths), s.ints(starts))
    s.plain.append(kt.float().cpu().numpy(), vt.float().cpu().numpy(), s.table, lengths, starts)
    s.check_pool()


def call(s, form, q, lengths, new, Hq, causal=True):
    """q [T, Hq, D] f32.  The result and what the tensor held."""
    torch = s.torch
    T = sum(new)
    assert_form(form, s.cache, T, Hq, len(lengths), max(lengths), s.f32, causal)
    qt = torch.from_numpy(np.ascontiguousarray(q, dtype=np.float32)).cuda().to(torch.float32 if s.f32 else torch.bfloat16)
    starts = np.concatenate([[0], np.cumsum(new)])
    got = s.ops.kv_cache_attention(s.cache, qt, s.dtable, s.ints(lengths), s.ints(starts), causal=causal, max_length=max(lengths))
    assert s.ops.last_status(None) == 0
    return got.double().cpu().numpy(), qt.float().cpu().numpy(), starts


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q_exp,k_exp", [(12, 12), (55, 55), (-20, 80), (80, -20)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("form,f32", CASES)
def test_equal_logits_of_any_size(ops, form, f32, sign, q_exp, k_exp, fp8):
    """Every key of a row has the same logit, up to +-1e34: the result is the mean of the values it sees, whatever the scales of
    their pages; a logit's rounding must not decide what is added up."""
    lengths, new, Hkv, Hq = FORMS[form]
    s = Setup(ops, 3, lengths, Hkv=Hkv, D=128 if fp8 else 64, page=32, fp8=fp8, f32=f32)
    fill(s, lengths, np.full((sum(lengths), Hkv, s.D), sign * 2.0 ** k_exp, np.float32))
    q = np.full((sum(new), Hq, s.D), 2.0 ** q_exp, np.float32)
    q[1::3] *= 0.5  # (rows of one tile that differ)
    got, qf, starts = call(s, form, q, lengths, new, Hq)
    assert_close(got, *expect(s, qf, lengths, starts), f32, max(lengths), exact_logits=True)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("form,f32", CASES)
def test_large_logits_that_differ_by_page(ops, form, f32, sign, fp8):
    """Pages whose keys are 2^20, 2^21 and 2^22 against queries of 2^15, and the largest logit's page scales beside one another: the
    keys with the largest logit share the weight."""
    lengths, new, Hkv, Hq = FORMS[form]
    s = Setup(ops, 4, lengths, Hkv=Hkv, D=64 if fp8 else 128, page=16, fp8=fp8, f32=f32)
    k = np.concatenate([sign * 2.0 ** (20 + np.arange(n) // s.page * 7 % 3) for n in lengths]).astype(np.float32)
    fill(s, lengths, np.broadcast_to(k[:, None, None], (sum(lengths), Hkv, s.D)).copy())
    q = np.full((sum(new), Hq, s.D), 2.0 ** 15, np.float32)
    got, qf, starts = call(s, form, q, lengths, new, Hq)
    assert_close(got, *expect(s, qf, lengths, starts), f32, max(lengths), exact_logits=True)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("form,f32", CASES)
def test_pages_of_large_keys_among_ordinary_ones(ops, form, f32, fp8):
    """One page of keys of 3e4 inside ordinary ones, queries of 10: the kernels change over in the middle of a sequence."""
    lengths, new, Hkv, Hq = FORMS[form]
    s = Setup(ops, 5, lengths, Hkv=Hkv, D=64, page=32, fp8=fp8, f32=f32)
    k = s.rng.standard_normal((sum(lengths), Hkv, s.D)).astype(np.float32)
    k[lengths[0] // 2:lengths[0] // 2 + 40] *= 3e4
    k[sum(lengths) - 20:] *= 3e4
    fill(s, lengths, k)
    q = (s.rng.standard_normal((sum(new), Hq, s.D)) * 10).astype(np.float32)
    q[:, 1::2] *= 1e-4  # (heads of ordinary logits)
    got, qf, starts = call(s, form, q, lengths, new, Hq)
    assert_close(got, *expect(s, qf, lengths, starts), f32, max(lengths))
