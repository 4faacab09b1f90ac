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


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("form,f32", CASES)
def test_a_query_that_is_not_finite_makes_its_row_nan(ops, form, f32, bad, fp8):
    """Whichever channel it stands in, in every form: that row of that head, if it sees a key, and nothing else."""
    lengths, new, Hkv, Hq = FORMS[form]
    s = Setup(ops, 6, lengths, Hkv=Hkv, D=128 if fp8 else 64, page=32, fp8=fp8, f32=f32)
    fill(s, lengths, s.rng.standard_normal((sum(lengths), Hkv, s.D)).astype(np.float32))
    q = s.rng.standard_normal((sum(new), Hq, s.D)).astype(np.float32)
    nan = np.zeros((sum(new), Hq), bool)
    for i, (row, head, channel) in enumerate(zip(range(0, sum(new), max(1, sum(new) // 23)), s.rng.permutation(1000), s.rng.permutation(1000))):
        q[row, head % Hq, channel % s.D] = bad
        nan[row, head % Hq] = True
    got, qf, starts = call(s, form, q, lengths, new, Hq)
    assert np.array_equal(np.isnan(got).all(axis=2), nan) and np.array_equal(np.isnan(got).any(axis=2), nan)
    want = expect(s, np.where(np.isfinite(qf), qf, 0), lengths, starts)
    assert_close(got[~nan], *[w[~nan] for w in want], f32, max(lengths))
    # every row of a call, in batches of which some rows see nothing: an idle slot, padding, a page that does not exist
    idle = [0] * len(lengths)
    got, _, _ = call(s, form, np.full((sum(new), Hq, s.D), bad), lengths, new, Hq)
    assert np.isnan(got).all()
    qt = s.torch.full((sum(new), Hq, s.D), bad, device="cuda", dtype=s.torch.float32 if f32 else s.torch.bfloat16)
    where = (s.ints(idle), s.ints(starts))
    assert (s.ops.kv_cache_attention(s.cache, qt, s.dtable, *where, max_length=max(lengths)) == 0).all()
    table = s.dtable.clone()
    table[0, :] = -1
    o = s.ops.kv_cache_attention(s.cache, qt, table, s.ints(lengths), s.ints(starts), max_length=max(lengths))
    assert (o[:new[0]] == 0).all() and s.torch.isnan(o[new[0]:]).all() and s.ops.last_status(None) != 0


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("form,f32", CASES)
def test_logits_beyond_f32_make_the_row_nan(ops, form, f32, fp8):
    """A page of keys of 1e30 in the middle: heads with queries of 1e12 are NaN from there on, in front of it and in the other heads nothing changes."""
    lengths, new, Hkv, Hq = FORMS[form]
    s = Setup(ops, 8, lengths, Hkv=Hkv, D=64 if fp8 else 128, page=16, fp8=fp8, f32=f32)
    k = s.rng.standard_normal((sum(lengths), Hkv, s.D)).astype(np.float32)
    at = lengths[0] - max(new[0] // 2, 1)  # rows in front of and behind it where there are any
    k[at // 16 * 16:at // 16 * 16 + 16] = 1e30
    fill(s, lengths, k)
    q = s.rng.standard_normal((sum(new), Hq, s.D)).astype(np.float32)
    q[:, 0] = np.sign(q[:, 0]) * 1e12
    q[:, 1] = 1e12
    got, qf, starts = call(s, form, q, lengths, new, Hq)
    nan = np.zeros((sum(new), Hq), bool)
    for b, n in enumerate(new):  # (a page's keys share its scale: a row sees it from the page's first token on)
        huge = np.abs(k[sum(lengths[:b]):sum(lengths[:b + 1])]).max(axis=(1, 2)) > 1e29
        if huge.any():
            nan[starts[b]:starts[b + 1], :2] = (lengths[b] - n + np.arange(n) >= np.argmax(huge) // 16 * 16)[:, None]
    assert nan.any() and np.array_equal(np.isnan(got).all(axis=2), nan) and np.array_equal(np.isnan(got).any(axis=2), nan)
    with np.errstate(over="ignore"):
        want = expect(s, qf, lengths, starts)
    assert_close(got[~nan], *[w[~nan] for w in want], f32, max(lengths))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("k_exp", [-50, -30])
@pytest.mark.parametrize("form,f32", CASES)
def test_queries_at_the_upper_end(ops, form, f32, k_exp, fp8):
    """|q| of 3e38, beyond 2^127: keys of either sign, of which those with the sign of q share the weight."""
    lengths, new, Hkv, Hq = FORMS[form]
    s = Setup(ops, 10, lengths, Hkv=Hkv, D=64 if fp8 else 128, page=32, fp8=fp8, f32=f32)
    k = np.concatenate([2.0 ** k_exp * (-1.0) ** (np.arange(n) % 3) for n in lengths]).astype(np.float32)
    fill(s, lengths, np.broadcast_to(k[:, None, None], (sum(lengths), Hkv, s.D)).copy())
    q = np.full((sum(new), Hq, s.D), 3e38, np.float32)
    q[:, 1::2] *= -1.0
    got, qf, starts = call(s, form, q, lengths, new, Hq)
    assert_close(got, *expect(s, qf, lengths, starts), f32, max(lengths), exact_logits=True)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("q_exp", [-125, -118, -104])
@pytest.mark.parametrize("form,f32", CASES)
def test_queries_at_the_lower_end(ops, form, f32, q_exp, fp8):
    """Queries down to the subnormal numbers against keys up to 2^126: ordinary logits."""
    lengths, new, Hkv, Hq = FORMS[form]
    s = Setup(ops, 12, lengths, Hkv=Hkv, D=128 if fp8 else 64, page=16, fp8=fp8, f32=f32)
    k = np.clip(s.rng.standard_normal((sum(lengths), Hkv, s.D)), -3.9, 3.9) * 2.0 ** (-q_exp - 1)
    fill(s, lengths, k.astype(np.float32))
    q = s.rng.standard_normal((sum(new), Hq, s.D)) * 2.0 ** q_exp
    got, qf, starts = call(s, form, q, lengths, new, Hq)
    assert_close(got, *expect(s, qf, lengths, starts), f32, max(lengths))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D,new,Hq", [(128, 4, 12), (128, 1, 12), (64, 4, 12), (64, 1, 4)])
def test_long_sums_of_f32_tensors_have_no_bias(ops, D, new, Hq, fp8):
    """Every token of a head has the same positive values, so that they are the result whatever the weights.  Roundings to f32 are as often up as down:
    each output is off by a few 2^-24 sqrt(additions), the mean of tens of thousands by less than 2^-24; the constant parts -- two products cut at
    2^-23 of 16 keys' sum, the weights' second term, the division, 2^-23 each -- stay below 2^-21.  (Cut at every one of 400 products the mean would be off
    by 2^-18.)"""
    import torch
    L, B, Hkv = 12219, 74, 4
    s = Setup(ops, 14, [L], Hkv=Hkv, D=D, page=64, fp8=fp8, f32=True)
    k = torch.from_numpy(s.rng.standard_normal((L, Hkv, D)).astype(np.float32)).cuda()
    v = torch.from_numpy(s.rng.uniform(1, 2, (1, Hkv, D)).astype(np.float32)).cuda().expand(L, Hkv, D).contiguous()
    ops.kv_cache_append(s.cache, k, v, s.dtable, s.ints([L]), s.ints([0, L]))
    _, held = ops.kv_cache_read(s.cache, s.dtable, s.ints([L]), s.ints([0, 1]), 1, dtype=torch.float32)
    table = s.dtable.expand(B, -1).contiguous()  # (sequences may share pages that they only read)
    q = torch.from_numpy(s.rng.standard_normal((B * new, Hq, D)).astype(np.float32)).cuda()
    o = ops.kv_cache_attention(s.cache, q, table, s.ints([L] * B), s.ints(range(0, B * new + 1, new)), max_length=L)
    want = held[0].double().repeat_interleave(Hq // Hkv, dim=0)
    off = o.double() / want - 1
    assert off.abs().max() < 400 * 2.0 ** -24 and off.mean().abs() < 2.0 ** -21


def test_late_and_missing_tiles_with_large_logits(attn_lib):
    """The waits' test (its library, its late and missing tiles) on logits that take the kernels' other loop."""
    import subprocess
    import sys
    from test_gpu_kv_cache_waits import CHILD, ROOT
    ordinary = "q = rand(m + 49, 2 * heads, D)"
    assert CHILD.count(ordinary) == 1
    out = subprocess.run([sys.executable, "-c", CHILD.replace(ordinary, ordinary + " * 3000"), str(ROOT)], capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0 and "done" in out.stdout, out.stdout + out.stderr
