"""What the cache attention has to hold in each form of its kernels, which every test here makes sure of: stale and missing pages, pages that are NaN,
scales far apart, queries of any size, captured calls, offsets beyond 32 bits, and batches of many sequences."""
from __future__ import annotations

import numpy as np
import pytest

from kv_forms import BF16_ONLY, FORMS, assert_close, assert_form, expect, plan_of
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


class Form:
    """A filled cache and a call of the form."""

    def __init__(self, ops, form, seed, f32=False, fp8=False, D=128, page=32, q_scale=1.0, **kw):
        self.form, (self.lengths, self.new, Hkv, self.Hq) = form, FORMS[form]
        self.s = Setup(ops, seed, self.lengths, Hkv=Hkv, D=D, page=page, fp8=fp8, f32=f32, **kw)
        self.s.append(self.lengths, self.lengths)
        self.T, self.starts = sum(self.new), np.concatenate([[0], np.cumsum(self.new)])
        self.q, self.qf = self.s.rows(self.T, self.Hq, q_scale)
        self.where = (self.s.dtable, self.s.ints(self.lengths), self.s.ints(self.starts))
        self.positions = np.concatenate([n - m + np.arange(m) for n, m in zip(self.lengths, self.new)])

    def run(self, q=None, table=None, causal=True, cache=None, **kw):
        assert_form(self.form, self.s.cache, self.T, self.Hq, len(self.lengths), max(self.lengths), self.s.f32, causal)
        where = self.where if table is None else (table, *self.where[1:])
        return self.s.ops.kv_cache_attention(cache or self.s.cache, self.q if q is None else q, *where, causal=causal,
                                             max_length=max(self.lengths), **kw)

    def check(self, got, causal=True, keep=None, rows=None):
        want = expect(self.s, self.qf, self.lengths, self.starts, causal, keep)
        got = got.double().cpu().numpy()
        rows = np.ones(got.shape[:2], bool) if rows is None else rows
        assert_close(got[rows], *[w[rows] for w in want], self.s.f32, max(self.lengths))


@pytest.mark.parametrize("fp8,D,page,causal", [(False, 128, 64, True), (True, 64, 16, True), (False, 64, 128, False), (True, 128, 32, False)])
@pytest.mark.parametrize("form,f32", CASES)
def test_each_form(ops, form, f32, fp8, D, page, causal):
    f = Form(ops, form, 1, f32, fp8, D, page, mean=True)
    f.check(f.run(causal=causal), causal)
    assert ops.last_status(None) == 0


@pytest.mark.parametrize("scale", [300.0, 1e-30, 0.0])
@pytest.mark.parametrize("form,f32", CASES)
def test_large_tiny_and_zero_queries(ops, form, f32, scale):
    f = Form(ops, form, 2, f32, q_scale=scale)
    f.check(f.run())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("form,f32", CASES)
def test_stale_rows_and_pages_change_no_bit(ops, form, f32, fp8):
    """NaN patterns, or codes of -128, behind the last token and on pages that nobody has, whose scales are NaN."""
    import torch
    f = Form(ops, form, 3, f32, fp8, page=64)
    first, cache = f.run(), f.s.cache
    used = torch.zeros(cache.k.shape[0], f.s.page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(f.lengths):
        for t in range(0, n, f.s.page):
            used[int(f.s.table[b, t // f.s.page]), :min(f.s.page, n - t)] = True
    assert not used.all() and not used.any(dim=1).all()
    for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes.masked_fill_(~used[:, None, :, None], 0x7f if fp8 else -128)
        scales.masked_fill_(~used.any(dim=1)[:, None], float("nan"))
    assert torch.equal(first, f.run())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("form,f32", CASES)
def test_missing_pages_in_the_middle(ops, form, f32, fp8):
    """Pages inside the part of a sequence that all rows see, and the last one: their keys are left out, and it is reported."""
    from autorust_b200 import _abi
    f = Form(ops, form, 4, f32, fp8, D=64, page=32)
    n = f.lengths[0]
    for wrong, at in ((-1, n // 64), (f.s.cache.k.shape[0], n // 96), (2 ** 31 - 1, (n - 1) // 32)):
        table = f.s.dtable.clone()
        table[0, at] = wrong
        got = f.run(table=table)
        assert ops.last_status(None) == _abi.AR_ERR_PAGE and ops.last_status(None) == 0
        keep = np.ones(n, bool)
        keep[at * 32:(at + 1) * 32] = False
        f.check(got, keep={0: keep})


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("form,f32", CASES)
def test_a_page_that_is_nan(ops, form, f32, fp8, which):
    """One value of a token in the middle is NaN: rows that see its page are NaN in that kv head, rows in front of it and other heads are not."""
    f = Form(ops, form, 5, f32, fp8, D=128, page=32)
    n, s = f.lengths[0], f.s
    token = max(n - f.new[0] // 2 - 1, 0)
    k, v = (x.clone() for x in (s.rows(1, s.Hkv)[0], s.rows(1, s.Hkv)[0]))
    (k if which == "k" else v)[0, -1, 5] = float("nan")
    s.ops.kv_cache_append(s.cache, k, v, s.dtable[:1].contiguous(), s.ints([token + 1]), s.ints([0, 1]))
    kf, vf = k.float().cpu().numpy(), v.float().cpu().numpy()
    s.plain.append(kf, vf, s.table[:1], [token + 1], [0, 1])
    s.check_pool()
    nan = np.zeros((f.T, f.Hq), bool)
    nan[:f.new[0], -(f.Hq // s.Hkv):] = (f.positions[:f.new[0]] >= token // 32 * 32)[:, None]
    assert nan.any()
    got = f.run()
    bad = np.isnan(got.double().cpu().numpy())
    assert np.array_equal(bad.all(axis=2), nan) and np.array_equal(bad.any(axis=2), nan)
    with np.errstate(invalid="ignore"):
        f.check(got, rows=~nan)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("order", ["zeros first", "largest first", "mixed"])
@pytest.mark.parametrize("form,f32", CASES)
def test_scales_of_hidden_pages_do_not_reach_a_row(ops, form, f32, fp8, order):
    """Pages of values of 0, 2^-40, 1 and 2^40 behind one another: what a row must not see is larger than what it sees by any factor, and the bound is
    made of what it sees.  Rows whose values are all zero are exactly zero."""
    lengths, new, Hkv, Hq = FORMS[form]
    s = Setup(ops, 6, lengths, Hkv=Hkv, D=64, page=16, fp8=fp8, f32=f32)
    torch, T = s.torch, sum(lengths)
    sizes = {"zeros first": [0.0, 1.0, 2.0 ** 40], "largest first": [2.0 ** 40, 1.0, 2.0 ** -40, 0.0], "mixed": [1.0, 0.0, 2.0 ** -20, 2.0 ** 20, 2.0 ** -40]}[order]
    v = np.clip(s.rng.standard_normal((T, Hkv, 64)), -4, 4)
    page = np.concatenate([np.arange(n) // 16 for n in lengths])
    # in the last pages of a sequence, where rows differ in what they see, the sizes follow one another; zeros before them where they come first
    last = np.concatenate([np.full(n, (n - min(m, n)) // 16) for n, m in zip(lengths, new)])
    if order == "zeros first":
        v *= np.where(page <= last + 1, 0.0, np.resize(sizes, 1000)[np.minimum(page - last, 999)])[:, None, None]
    else:
        v *= np.resize(sizes, 1000)[page][:, None, None]
    k = torch.from_numpy((s.rng.standard_normal((T, Hkv, 64)) * 0.3).astype(np.float32)).cuda()
    v = torch.from_numpy(v.astype(np.float32)).cuda()
    k, v = (x if f32 else x.to(torch.bfloat16) for x in (k, v))
    all_starts = np.concatenate([[0], np.cumsum(lengths)])
    s.ops.kv_cache_append(s.cache, k, v, s.dtable, s.ints(lengths), s.ints(all_starts))
    s.plain.append(k.float().cpu().numpy(), v.float().cpu().numpy(), s.table, lengths, all_starts)
    s.check_pool()
    q, qf = s.rows(sum(new), Hq, 2.0)
    starts = np.concatenate([[0], np.cumsum(new)])
    assert_form(form, s.cache, sum(new), Hq, len(lengths), max(lengths), f32)
    got = s.ops.kv_cache_attention(s.cache, q, s.dtable, s.ints(lengths), s.ints(starts), max_length=max(lengths)).double().cpu().numpy()
    o, size, reach, most = expect(s, qf, lengths, starts)
    assert_close(got, o, size, reach, most, f32, max(lengths))
    nothing = (size == 0).all(axis=2)
    assert (got[nothing] == 0).all() and (order != "zeros first" or nothing.any())


@pytest.mark.parametrize("form,f32", CASES)
def test_captured_and_replayed(ops, form, f32):
    """Between an append and a read, on other tokens than it was captured with; behind a join of two streams that brought the tokens."""
    import torch
    f = Form(ops, form, 7, f32, D=64)
    s = f.s
    k, v = (s.rows(f.T, s.Hkv)[0].clone() for _ in range(2))
    q = f.q.clone()
    news = [torch.empty_like(x) for x in (k, v, q)]
    need = ops._abi.load().ar_kv_cache_attention_workspace_bytes(s.cache._pool, ops._kv_batch(s.cache, *f.where, f.T), int(not f32), f.Hq,
                                                                 max(f.lengths), 1)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()

    def step():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            k.copy_(news[0])
        v.copy_(news[1])
        q.copy_(news[2])
        main.wait_stream(side)
        ops.kv_cache_append(s.cache, k, v, *f.where)
        o = f.run(q=q, workspace=ws)
        return o, *ops.kv_cache_read(s.cache, *f.where, f.T, dtype=k.dtype)

    def fresh():
        for x, H in zip(news, (s.Hkv, s.Hkv, f.Hq)):
            x.copy_(s.rows(f.T, H)[0])

    pool = (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale)
    saved = [x.clone() for x in pool]
    fresh()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        fresh()
        results = []
        for go in (graph.replay, step):
            for x, y in zip(pool, saved):
                x.copy_(y)
            r = go()
            results.append([x.clone() for x in (out if r is None else r)])
        assert all(torch.equal(x, y) for x, y in zip(*results))
    assert ops.last_status(None) == 0


@pytest.mark.parametrize("form", BF16_ONLY)
def test_many_rows_beyond_32_bit_offsets(ops, form):
    """Pages whose codes lie more than 2^32 bytes into the pool, rows of q and of the result that do so too: the bits of a small pool."""
    import torch
    f = Form(ops, form, 8, D=128, page=128)
    s, Hkv = f.s, f.s.Hkv
    pages = (5 << 30) // (Hkv * 128 * 128)
    far = ops.kv_cache(pages, Hkv, 128, 128)
    table = torch.where(f.s.dtable < 0, f.s.dtable, pages - 1 - f.s.dtable)
    for x, y in ((far.k, s.cache.k), (far.v, s.cache.v), (far.k_scale, s.cache.k_scale), (far.v_scale, s.cache.v_scale)):
        x[pages - y.shape[0]:] = y.flip(0)
    want = f.run()
    assert torch.equal(f.run(table=table.contiguous(), cache=far), want)
    wide = (2 ** 32 // 2 // f.T // 8 + 2 * f.Hq * 128) * 8  # elements between the rows
    big = torch.empty((f.T - 1) * wide + 2 * f.Hq * 128, dtype=torch.bfloat16, device="cuda")
    q, out = (torch.as_strided(big, (f.T, f.Hq, 128), (wide, 128, 1), i * f.Hq * 128) for i in range(2))
    q.copy_(f.q)
    f.run(q=q, out=out)
    assert torch.equal(out, want) and ops.last_status(None) == 0


# ---- batches of many sequences ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,fp8", [(33, False), (33, True), (70, False), (70, True), (1100, False)])
def test_writing_and_reading_many_sequences(ops, B, fp8):
    """More sequences than a warp looks at at once, and than it does twice; some without rows, idle, or with padding."""
    import torch
    rng = np.random.default_rng(B)
    lengths = [int(x) for x in rng.integers(0, 50, B)]
    s = Setup(ops, B, [50] * B, Hkv=1, D=64, page=16, fp8=fp8)
    for _ in range(2):
        new = [int(x) for x in rng.integers(0, 4, B)]
        new[B // 2] = 40
        starts = np.concatenate([[0], np.cumsum(new)])
        k, v = s.append(lengths, new)
        s.check_pool()
        got = ops.kv_cache_read(s.cache, s.dtable, s.ints(lengths), s.ints(starts), int(starts[-1]), dtype=torch.float32)
        for which, g in enumerate(got):
            rows = []
            for b, n in enumerate(new):
                x = s.plain.tokens(which, s.table[b], lengths[b], np.float32)
                rows.append(np.concatenate([np.zeros((max(n - lengths[b], 0), 1, 64), np.float32), x])[-n:] if n else x[:0])
            assert np.array_equal(g.cpu().numpy(), np.concatenate(rows))
        lengths = [min(n + m + 1, 50) for n, m in zip(lengths, new)]
    assert ops.last_status(None) == 0


@pytest.mark.parametrize("B,new,cut,kind", [(*x, kind) for kind in ((False, False), (True, True), (True, False)) for x in (
    (40, 1, True), (75, 1, True), (70, 5, True), (70, 1, False), (300, 3, False))] + [(1100, 1, False, (False, False))])
def test_attention_of_many_sequences(ops, B, new, cut, kind):
    """Shares of the keys over more than 32 and 64 sequences, and whole tiles found among them: lengths from nothing to long ones, sequences without rows."""
    fp8, f32 = kind
    rng = np.random.default_rng(B + new)
    lengths = [int(x) for x in rng.integers(0, 100, B)]
    if cut:
        lengths[3], lengths[B // 2], lengths[B - 1] = 3000, 1, 2000
    rows = [int(x) for x in rng.integers(0, new + 1, B)] if new > 1 else [int(x) for x in rng.integers(0, 2, B)]
    rows[3] = rows[B - 1] = new
    s = Setup(ops, B, lengths, Hkv=1, D=64, page=32, fp8=fp8, f32=f32)
    s.append(lengths, lengths)
    T, bound = sum(rows), 8192 if cut else 128
    starts = np.concatenate([[0], np.cumsum(rows)])
    plan = plan_of(s.cache, T, 4, B, bound, f32)
    assert plan[0] in (8, 16) and (plan[1] > 0) == cut, plan
    q, qf = s.rows(T, 4)
    s.dtable = s.torch.nn.functional.pad(s.dtable, (0, -(-bound // 32) - s.dtable.shape[1]), value=-1).contiguous()
    got = ops.kv_cache_attention(s.cache, q, s.dtable, s.ints(lengths), s.ints(starts), max_length=bound)
    assert_close(got.double().cpu().numpy(), *expect(s, qf, lengths, starts), f32, max(lengths))
    if new == 1 and not cut:
        one, onef = s.rows(B, 4)
        got = ops.kv_cache_attention(s.cache, one, s.dtable, s.ints(lengths), max_length=bound)
        assert_close(got.double().cpu().numpy(), *expect(s, onef, lengths, np.arange(B + 1)), f32, max(lengths))
    assert ops.last_status(None) == 0


@pytest.mark.parametrize("fp8", [False, True])
def test_many_rows_of_many_sequences(ops, fp8):
    rng = np.random.default_rng(9)
    B = 45
    lengths = [int(x) for x in rng.integers(1, 330, B)]
    rows = [int(min(n + 2, x)) for n, x in zip(lengths, rng.integers(0, 200, B))]
    s = Setup(ops, 9, lengths, Hkv=1, D=64, page=64, fp8=fp8)
    s.append(lengths, lengths)
    starts = np.concatenate([[0], np.cumsum(rows)])
    assert plan_of(s.cache, sum(rows), 3, B, 384, False) == [256, 0, 1]
    s.dtable = s.torch.nn.functional.pad(s.dtable, (0, 6 - s.dtable.shape[1]), value=-1).contiguous()
    q, qf = s.rows(sum(rows), 3)
    got = ops.kv_cache_attention(s.cache, q, s.dtable, s.ints(lengths), s.ints(starts), max_length=384)
    assert_close(got.double().cpu().numpy(), *expect(s, qf, lengths, starts), False, max(lengths))


@pytest.mark.parametrize("fp8,D", [(False, 128), (True, 64)])
def test_a_chunk_among_single_tokens(ops, fp8, D):
    """What `starts` is for: a chunk of one prompt packed with single tokens of other sequences and an idle slot."""
    lengths, rows = [1700, 33, 900, 0, 2048, 128, 1999, 1, 64], [1, 1, 1, 1, 500, 1, 1, 1, 1]
    s = Setup(ops, 10, lengths, Hkv=2, D=D, page=64, fp8=fp8)
    s.append(lengths, lengths)
    starts = np.concatenate([[0], np.cumsum(rows)])
    q, qf = s.rows(sum(rows), 8)
    assert plan_of(s.cache, sum(rows), 8, len(rows), 2048, False)[0] == 256
    got = ops.kv_cache_attention(s.cache, q, s.dtable, s.ints(lengths), s.ints(starts), max_length=2048)
    assert_close(got.double().cpu().numpy(), *expect(s, qf, lengths, starts), False, max(lengths))
    assert (got[3] == 0).all() and ops.last_status(None) == 0


# ---- reading one row of each sequence ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("B", [1, 5, 40])
def test_read_without_starts(ops, fp8, f32, B):
    import torch
    lengths = [int(x) for x in np.random.default_rng(B).integers(0, 70, B)]
    lengths[-1] = 33
    s = Setup(ops, 11, lengths, Hkv=3, D=64, page=32, fp8=fp8, f32=f32, mean=True)
    s.append(lengths, lengths)
    kind = torch.float32 if f32 else torch.bfloat16
    for got in (ops.kv_cache_read(s.cache, s.dtable, s.ints(lengths), None, B, dtype=kind),
                ops.kv_cache_read(s.cache, s.dtable, s.ints(lengths), None, B, out=tuple(torch.full((B, 3, 64), 7.0, dtype=kind, device="cuda") for _ in range(2)))):
        for which, g in enumerate(got):
            want = np.zeros((B, 3, 64), np.float32)
            for b, n in enumerate(lengths):
                if n:
                    want[b] = s.plain.tokens(which, s.table[b], n, np.float32)[-1] + (s.k_mean if which == 0 else 0)
            assert torch.equal(g.cpu(), torch.from_numpy(want).to(kind))
