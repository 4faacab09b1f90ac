"""The 8-bit key/value cache (ar_kv_cache_append / _read / _attention): codes and scales bit for bit against the plain
restatement, values read back, attention against 64 bits, and the calls around the edges -- ragged batches, padding, pages that end
inside a tile, stale and poisoned pages, bad page numbers, streams and captured graphs."""
from __future__ import annotations

import numpy as np
import pytest

import kv_plain
from kv_plain import PlainCache, assert_attention_close, attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(attn_lib):
    import torch
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device: there is no fallback path to test")
    from autorust_b200 import ops as _ops
    return _ops


class Setup:
    """A pool with shuffled pages, its plain twin, and the packed tensors of one call at a time."""

    def __init__(self, ops, seed, capacity, Hkv=2, D=128, page=16, fp8=False, f32=False, mean=False, spare=5, fill=0):
        import torch
        self.torch, self.ops, self.page, self.f32, self.D, self.Hkv = torch, ops, page, f32, D, Hkv
        self.rng = np.random.default_rng(seed)
        counts = [-(-c // page) for c in capacity]
        pages = sum(counts) + spare
        order = self.rng.permutation(pages)
        width = max(max(counts), 1)
        self.table = np.full((len(capacity), width), -1, np.int32)
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.k_mean = (self.rng.standard_normal((Hkv, D)) * 2).astype(np.float32) if mean else None
        self.plain = PlainCache(pages, Hkv, page, D, fp8, self.k_mean, fill)
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        self.cache = ops.kv_cache(pages, Hkv, page, D, fp8, None if self.k_mean is None else dev(self.k_mean))
        if fill:
            self.cache.k.fill_(fill)
            self.cache.v.fill_(fill)
        self.dtable = dev(self.table)

    def ints(self, x):
        return self.torch.tensor([int(i) for i in x], dtype=self.torch.int32, device="cuda")

    def rows(self, T, H, scale=1.0):
        """[T, H, D] rows as a strided view of a wider tensor on the GPU, and what they hold as f32."""
        x = (self.rng.standard_normal((T, H + 3, self.D)) * scale).astype(np.float32)
        t = self.torch.from_numpy(x).cuda()
        t = (t if self.f32 else t.to(self.torch.bfloat16))[:, 1:1 + H]
        return t, t.float().cpu().numpy()

    def batch(self, lengths, new):
        starts = np.concatenate([[0], np.cumsum(new)]).astype(int)
        one_each = all(n == 1 for n in new)
        return starts, (self.dtable, self.ints(lengths), None if one_each else self.ints(starts))

    def append(self, lengths, new, k_scale=1.0):
        starts, where = self.batch(lengths, new)
        T = int(starts[-1])
        k, kf = self.rows(T, self.Hkv, k_scale)
        v, vf = self.rows(T, self.Hkv)
        self.ops.kv_cache_append(self.cache, k, v, *where)
        self.plain.append(kf, vf, self.table, lengths, starts)
        return kf, vf

    def check_pool(self):
        for which, (codes, scales) in enumerate(((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale))):
            assert np.array_equal(scales.cpu().numpy(), self.plain.scales[which], equal_nan=True)
            assert np.array_equal(codes.cpu().numpy(), self.plain.codes[which])

    def attend(self, lengths, new, Hq, causal=True, max_length=None, q_scale=1.0, out=None):
        starts, where = self.batch(lengths, new)
        q, qf = self.rows(int(starts[-1]), Hq, q_scale)
        got = self.ops.kv_cache_attention(self.cache, q, *where, causal=causal, max_length=max_length, out=out)
        return got, qf, starts

    def expect(self, qf, lengths, starts, causal):
        parts = []
        for b, length in enumerate(lengths):
            n = int(starts[b + 1] - starts[b])
            k, v = (self.plain.tokens(which, self.table[b], int(length)) for which in (0, 1))
            parts.append(attention(qf[starts[b]:starts[b + 1]].astype(np.float64), k, v, int(length) - n + np.arange(n), causal))
        return [np.concatenate(p) for p in zip(*parts)]

    def check_attention(self, lengths, new, Hq, causal=True, **kw):
        got, qf, starts = self.attend(lengths, new, Hq, causal, **kw)
        assert_attention_close(got.double().cpu().numpy(), *self.expect(qf, lengths, starts, causal), self.f32)
        assert self.ops.last_status(None) == 0
        return got


# ---- writing ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("D,page", [(64, 16), (64, 32), (128, 16), (128, 64), (64, 128), (128, 128)])
def test_append_codes_and_scales(ops, fp8, f32, D, page):
    """Whole pages, parts of pages, tokens behind others in an open page, several sequences at once: every bit of the pool,
    the pages that no call names included."""
    s = Setup(ops, D + page, [300, 5, page, 2 * page + 1, 0, 129], D=D, page=page, fp8=fp8, f32=f32, mean=page != 32, fill=3)
    s.append([37, 1, page, page - 1, 0, 100], [37, 1, page, page - 1, 0, 100])
    s.check_pool()
    s.append([38, 2, page, page + 1, 0, 129], [1, 1, 0, 2, 0, 29], k_scale=3.0)  # larger keys: scales grow
    s.check_pool()
    s.append([300, 5, page, 2 * page + 1, 0, 129], [262, 3, 0, page, 0, 0], k_scale=0.1)
    s.check_pool()
    assert ops.last_status(None) == 0


@pytest.mark.parametrize("fp8", [False, True])
def test_append_token_by_token(ops, fp8):
    s = Setup(ops, 5, [70, 70, 70], Hkv=3, D=64, page=32, fp8=fp8)
    for t in range(1, 71):
        s.append([t, max(t - 3, 0), t], [1, 1, 1], k_scale=1.0 + 0.05 * t)  # (the second one's first rows are padding)
        if t in (1, 2, 31, 32, 33, 70):
            s.check_pool()
    # E4M3 scales are powers of two: what was written token by token is what one call would have written
    if fp8:
        import torch
        one = Setup(ops, 5, [70], Hkv=3, D=64, page=32, fp8=True)
        k, _ = one.rows(70, 3, 4.0)
        v, _ = one.rows(70, 3)
        one.ops.kv_cache_append(one.cache, k, v, one.dtable, one.ints([70]), one.ints([0, 70]))
        whole = [x.clone() for x in (one.cache.k, one.cache.v, one.cache.k_scale, one.cache.v_scale)]
        for t in range(70):
            one.ops.kv_cache_append(one.cache, k[t:t + 1], v[t:t + 1], one.dtable, one.ints([t + 1]))
        assert torch.equal(whole[2], one.cache.k_scale) and torch.equal(whole[3], one.cache.v_scale)
        for a, b in ((whole[0], one.cache.k), (whole[1], one.cache.v)):
            x, y = (torch.from_numpy(kv_plain.TABLE)[c.cpu().long()] for c in (a, b))
            # (subnormal codes may have been rounded at a smaller scale first: one step of 2^-9 at most)
            assert (x - y).abs().max() <= 2.0 ** -9


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("amax", [0.0, 1e-30, 2.0 ** -52, 1.0, 447.9, 448.0, 448.1, 1e30])
def test_append_scales_at_their_edges(ops, fp8, amax):
    import torch
    s = Setup(ops, 9, [16], Hkv=1, D=64, fp8=fp8, f32=True)
    k = torch.linspace(-1, 1, 16 * 64, device="cuda").view(16, 1, 64) * amax
    s.ops.kv_cache_append(s.cache, k, -k, s.dtable, s.ints([16]), s.ints([0, 16]))
    s.plain.append(k.cpu().numpy(), -k.cpu().numpy(), s.table, [16], [0, 16])
    s.check_pool()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("fp8", [False, True])
def test_a_value_that_is_not_finite_poisons_its_page_and_head_only(ops, fp8, bad):
    import torch
    s = Setup(ops, 11, [64], Hkv=2, D=64, page=16, fp8=fp8)
    k, _ = s.rows(64, 2)
    v, _ = s.rows(64, 2)
    k = k.clone()
    k[20, 1, 7] = bad
    where = (s.dtable, s.ints([64]), s.ints([0, 64]))
    s.ops.kv_cache_append(s.cache, k, v, *where)
    kb, vb = s.ops.kv_cache_read(s.cache, *where, 64)
    nan = torch.isnan(kb).all(dim=2)
    want = torch.zeros_like(nan)
    want[16:32, 1] = True
    assert torch.equal(nan, want) and torch.equal(torch.isnan(kb).any(dim=2), want) and not torch.isnan(vb).any()
    # rows that see the page are NaN in that head, rows in front of it are not; the next token on the page does not heal it
    q, _ = s.rows(64, 2)
    o = s.ops.kv_cache_attention(s.cache, q, *where)
    assert not torch.isnan(o[:16]).any() and not torch.isnan(o[:, 0]).any() and torch.isnan(o[16:, 1]).all()
    s.ops.kv_cache_append(s.cache, k[:4], v[:4], s.dtable, s.ints([30]), s.ints([0, 4]))
    assert torch.isnan(s.cache.k_scale[int(s.table[0, 1]), 1])


# ---- reading back -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("D,page,mean", [(64, 16, True), (128, 32, False), (128, 128, True), (64, 64, False)])
def test_read_gives_the_values(ops, fp8, f32, D, page, mean):
    import torch
    s = Setup(ops, 3 * D + page, [150, 1, 2, 0, 40], D=D, page=page, fp8=fp8, f32=f32, mean=mean)
    lengths = [150, 1, 2, 0, 40]
    s.append(lengths, lengths)
    kind = torch.float32 if f32 else torch.bfloat16
    for back in (lengths, [17, 1, 0, 0, 40], [1, 1, 1, 1, 1], [150, 4, 2, 3, 41]):  # (the last: rows in front of the tokens)
        starts, where = s.batch(lengths, back)
        T = int(starts[-1])
        wide = [torch.full((T + 2, 5, D), 7.0, dtype=kind, device="cuda") for _ in range(2)]
        out = tuple(w[:, 1:3] for w in wide)
        one_each = where[2] is None
        got = s.ops.kv_cache_read(s.cache, where[0], where[1], s.ints(starts) if one_each else where[2], T + 2, out=out)
        for which, (g, w) in enumerate(zip(got, wide)):
            rows = []
            for b, n in enumerate(back):
                x = s.plain.tokens(which, s.table[b], lengths[b], np.float32)
                if which == 0 and mean:
                    x = x + s.k_mean
                x = np.concatenate([np.zeros((max(n - lengths[b], 0), 2, D), np.float32), x])
                rows.append(x[len(x) - n:])
            want = torch.from_numpy(np.concatenate(rows)).to(kind)
            assert torch.equal(g[:T].cpu(), want)
            assert (w[T:] == 7).all() and (w[:, 0] == 7).all() and (w[:, 3:] == 7).all()  # what belongs to no row
    if T == 5:
        k, v = s.ops.kv_cache_read(s.cache, s.dtable, s.ints(lengths), None, 5, dtype=kind)
        assert torch.equal(k, got[0][:5])


# ---- attention ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (128, 16), (64, 128)])
def test_single_tokens(ops, fp8, f32, D, page):
    """Lengths around the tile edges, idle slots, one to sixteen query heads per kv head."""
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 0, 64, 65, 127, 128, 129, 300, 513]
    s = Setup(ops, D + page + fp8, lengths, Hkv=2, D=D, page=page, fp8=fp8, f32=f32, mean=True)
    s.append(lengths, lengths)
    for Hq in (2, 8, 32):
        got = s.check_attention(lengths, [1] * len(lengths), Hq)
        assert (got[8] == 0).all()  # the idle slot


@pytest.mark.parametrize("fp8,f32", [(False, False), (True, True), (False, True), (True, False)])
@pytest.mark.parametrize("D,page", [(64, 32), (128, 16), (128, 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_several_tokens(ops, fp8, f32, D, page, causal):
    """Chunks of a prompt behind what is there, whole prompts, padding in front, rows of no sequence at both ends of the packing."""
    lengths, new = [100, 5, 37, 3, 200, 64, 0], [17, 5, 1, 5, 100, 0, 2]
    s = Setup(ops, D * 3 + page, lengths, Hkv=3, D=D, page=page, fp8=fp8, f32=f32)
    s.append(lengths, lengths)
    for Hq in (3, 9, 21):
        s.check_attention(lengths, new, Hq, causal)


@pytest.mark.parametrize("fp8,f32,D,page,Hkv,Hq", [(False, False, 128, 16, 1, 4), (True, False, 128, 128, 2, 40), (False, True, 64, 64, 1, 1),
                                                   (True, True, 128, 32, 1, 16)])
def test_long_sequences_are_cut_and_joined(ops, fp8, f32, D, page, Hkv, Hq):
    lengths = [9001, 130, 4096]
    s = Setup(ops, D + Hq, lengths, Hkv=Hkv, D=D, page=page, fp8=fp8, f32=f32)
    s.append(lengths, lengths)
    assert ops.kv_cache_attention_workspace(s.cache, 3, Hq, 3, 9008) > 0
    s.check_attention(lengths, [1, 1, 1], Hq)
    s.check_attention(lengths, [3, 1, 7], Hq, max_length=9001)
    s.check_attention(lengths, [2, 2, 2], Hq, causal=False)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 32), (128, 128), (64, 64)])
@pytest.mark.parametrize("causal", [False, True])
def test_many_rows(ops, fp8, D, page, causal):
    """Calls that the tensor-core kernel takes: row tiles of 128 and 256 and their edges, key tiles of 128 and theirs, rows
    without keys, sequences of one row beside them, groups that do not divide a tile."""
    lengths, new = [300, 129, 256, 257, 5, 640, 90, 0], [300, 128, 255, 1, 5, 100, 130, 3]
    s = Setup(ops, D + page + 7, lengths, Hkv=2, D=D, page=page, fp8=fp8, mean=True)
    s.append(lengths, lengths)
    for Hq in (2, 6, 8):
        s.check_attention(lengths, new, Hq, causal)


@pytest.mark.parametrize("fp8,D,page", [(False, 128, 64), (True, 128, 16), (False, 64, 128), (True, 64, 32)])
def test_many_rows_on_long_sequences(ops, fp8, D, page):
    """Few row tiles: the keys are divided over CTAs and joined.  Sequences shorter than the parts are many, idle ones, a row
    that belongs to none."""
    lengths, new = [4000, 1000, 100, 0], [170, 133, 90, 2]
    s = Setup(ops, 17 + page, lengths, Hkv=1, D=D, page=page, fp8=fp8)
    s.append(lengths, lengths)
    parts, rest = divmod(ops.kv_cache_attention_workspace(s.cache, 395, 4, 4, 4000), 395 * 4 * (D + 4) * 4)
    assert parts > 1 and rest == 0  # (a row of results for each)
    for causal in (True, False):
        s.check_attention(lengths, new, 4, causal, max_length=4000)
    out = s.torch.full((397, 4, D), 7.0, dtype=s.torch.bfloat16, device="cuda")
    q, qf = s.rows(397, 4)
    s.ops.kv_cache_attention(s.cache, q, s.dtable, s.ints(lengths), s.ints([1, 171, 304, 394, 396]), out=out, max_length=4000)
    want = s.expect(qf[1:396], lengths, np.array([0, 170, 303, 393, 395]), True)
    assert_attention_close(out[1:396].double().cpu().numpy(), *want, False)
    assert (out[:1] == 7).all() and (out[396:] == 7).all()


def test_rows_of_no_sequence_are_left(ops):
    import torch
    s = Setup(ops, 21, [40, 9], Hkv=1, D=64)
    s.append([40, 9], [40, 9])
    q, qf = s.rows(12, 2)
    out = torch.full((12, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    s.ops.kv_cache_attention(s.cache, q, s.dtable, s.ints([40, 9]), s.ints([2, 5, 9]), out=out)
    want = s.expect(qf[2:9], [40, 9], np.array([0, 3, 7]), True)
    assert_attention_close(out[2:9].double().cpu().numpy(), *want, False)
    assert (out[:2] == 7).all() and (out[9:] == 7).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("f32", [False, True])
def test_unused_rows_and_pages_do_not_matter(ops, fp8, f32):
    """Stale codes (NaN patterns among them) behind the last token and on unused pages, NaN scales there: not a bit of the result changes."""
    import torch
    lengths = [33, 70, 1]
    s = Setup(ops, 31, lengths, Hkv=2, D=128, page=64, fp8=fp8, f32=f32)
    s.append(lengths, lengths)
    q, _ = s.rows(3, 8)
    many, _ = s.rows(90, 8)
    where = (s.dtable, s.ints(lengths))
    wide = (many, *where, s.ints([0, 20, 89, 90]))
    first = s.ops.kv_cache_attention(s.cache, q, *where)
    first_wide = s.ops.kv_cache_attention(s.cache, *wide)
    used = torch.zeros(s.cache.k.shape[0], s.page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        for t in range(n):
            used[int(s.table[b, t // s.page]), t % s.page] = True
    for codes, scales in ((s.cache.k, s.cache.k_scale), (s.cache.v, s.cache.v_scale)):
        codes.masked_fill_(~used[:, None, :, None], 0x7f if fp8 else -128)
        scales.masked_fill_(~used.any(dim=1)[:, None], float("nan"))
    assert torch.equal(first, s.ops.kv_cache_attention(s.cache, q, *where))
    assert torch.equal(first_wide, s.ops.kv_cache_attention(s.cache, *wide))


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
def test_scales_that_differ_by_orders_of_magnitude(ops, f32, fp8):
    """Pages whose values are 2^-40 to 2^40 of one another, all-zero pages: weights of the small ones must not vanish in f16."""
    import torch
    L, page, D = 160, 16, 64
    s = Setup(ops, 41, [L], Hkv=1, D=D, page=page, fp8=fp8, f32=f32)
    k, kf = s.rows(L, 1, 0.3)
    v = s.rng.standard_normal((L, 1, D)).astype(np.float32)
    for j, e in enumerate([0, -20, 20, 0, -40, 40, 3, 0, 1, -1]):
        v[j * page:(j + 1) * page] *= 2.0 ** e
    v[3 * page:4 * page] = 0.0
    v = torch.from_numpy(v).cuda().to(k.dtype)
    q, qf = s.rows(40, 4, 2.0)
    where = (s.dtable, s.ints([L]), s.ints([0, L]))
    s.ops.kv_cache_append(s.cache, k, v, *where)
    s.plain.append(kf, v.float().cpu().numpy(), s.table, [L], [0, L])
    s.check_pool()
    # causal rows up to the end of each page: what a row sees differs by 2^40 from what the next one does
    for last in (16, 32, 33, 48, 64, 80, 95, 96, 160):
        for n in (8, 40):
            got = s.ops.kv_cache_attention(s.cache, q[:n], s.dtable, s.ints([last]), s.ints([0, n]))
            want = s.expect(qf[:n], [last], np.array([0, n]), True)
            assert_attention_close(got.double().cpu().numpy(), *want, f32)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("order", ["zero first", "largest first"])
def test_scales_at_both_ends(ops, f32, fp8, order):
    """All-zero pages (the least scale) and pages of 1e37, either in front: whole tiles, cut ones, many rows, many rows in parts."""
    import torch
    L, page, D = 4096, 16, 64
    s = Setup(ops, 43, [L], Hkv=1, D=D, page=page, fp8=fp8, f32=f32)
    k, kf = s.rows(L, 1, 0.3)
    v = s.rng.standard_normal((L, 1, D)).astype(np.float32)
    size = np.tile([0.0, 1e37, 1e-16, 1.0] if order == "zero first" else [1e37, 1e-16, 0.0, 1.0], L // 64)
    v = np.clip(v, -4, 4) * np.repeat(size, page).astype(np.float32)[:, None, None]
    v = torch.from_numpy(v).cuda().to(k.dtype)
    q, qf = s.rows(40, 4, 2.0)
    where = (s.dtable, s.ints([L]), s.ints([0, L]))
    s.ops.kv_cache_append(s.cache, k, v, *where)
    s.plain.append(kf, v.float().cpu().numpy(), s.table, [L], [0, L])
    s.check_pool()
    # (rows that see the first page, the first two, and so on; then all of it)
    def check(q, qf, lengths, starts, table, bound):
        got = s.ops.kv_cache_attention(s.cache, q, table, s.ints(lengths), s.ints(starts), max_length=bound)
        assert_attention_close(got.double().cpu().numpy(), *s.expect(qf, lengths, np.array(starts), True), f32)
    for last in (16, 32, 48, 64, L):
        for n in (1, 8, 40):
            check(q[:n], qf[:n], [last], [0, n], s.dtable, max(last, 64))
    if f32:
        return
    q, qf = s.rows(1000, 4, 2.0)
    assert ops.kv_cache_attention_workspace(s.cache, 1000, 4, 1, L) == 8 * 1000 * 4 * (D + 4) * 4  # many rows, in eight parts
    check(q, qf, [L], [0, 1000], s.dtable, L)
    s.table = np.repeat(s.table, 6, axis=0)
    lengths = [600, 16, 450, 560, 599, 48]
    q, qf = s.rows(sum(lengths), 4, 2.0)
    assert ops.kv_cache_attention_workspace(s.cache, sum(lengths), 4, 6, 600) == 0  # many rows, not cut
    check(q, qf, lengths, [0, *np.cumsum(lengths)], s.dtable.expand(6, -1).contiguous(), 600)


@pytest.mark.parametrize("f32", [False, True])
def test_large_and_tiny_queries(ops, f32):
    """One key holds all the weight; logits of +-1e4; queries of 1e-30 (uniform weights) and zero."""
    lengths = [200]
    s = Setup(ops, 51, lengths, Hkv=1, D=128, page=32, f32=f32)
    s.append(lengths, lengths)
    for scale in (300.0, 1e-30, 0.0):
        for n in (5, 30):
            got, qf, starts = s.attend(lengths, [n], 4, q_scale=scale)
            want = s.expect(qf, lengths, starts, True)
            assert_attention_close(got.double().cpu().numpy(), *want, f32)


def test_pages_shared_by_sequences_that_only_read_them(ops):
    """A common prefix: two rows of the table name the same full pages."""
    s = Setup(ops, 61, [64, 10, 10], Hkv=2, D=128, page=32)
    s.append([64, 0, 0], [64, 0, 0])
    for b in (1, 2):
        own = s.table[b, 0]
        s.table[b, :2] = s.table[0, :2]
        s.table = np.concatenate([s.table, np.full((3, 1), -1, np.int32)], axis=1) if s.table.shape[1] < 3 else s.table
        s.table[b, 2] = own
    s.dtable = s.torch.from_numpy(s.table).cuda()
    s.append([64, 74, 74], [0, 10, 10])
    s.check_pool()
    s.check_attention([64, 74, 74], [1, 10, 3], 8)


# ---- what the device finds wrong ------------------------------------------------------------------------------------------
def test_bad_pages_are_skipped_and_reported(ops):
    import torch
    from autorust_b200 import _abi
    s = Setup(ops, 71, [64, 64], Hkv=2, D=64, page=16, fill=3)
    s.append([64, 64], [64, 64])
    s.check_pool()
    for wrong in (-1, -2 ** 31, s.cache.k.shape[0], 2 ** 31 - 1):
        table = s.dtable.clone()
        table[0, 1] = wrong
        where = (table, s.ints([64, 64]))
        # reading: zeros there, the rest as it is
        k, v = s.ops.kv_cache_read(s.cache, *where, s.ints([0, 64, 128]), 128)
        assert ops.last_status(None) == _abi.AR_ERR_PAGE and ops.last_status(None) == 0
        good = s.ops.kv_cache_read(s.cache, s.dtable, where[1], s.ints([0, 64, 128]), 128)
        for got, want in zip((k, v), good):
            want = want.clone()
            want[16:32] = 0
            assert torch.equal(got, want)
        # attention: those keys are left out
        q, qf = s.rows(2, 4)
        o = s.ops.kv_cache_attention(s.cache, q, *where)
        assert ops.last_status(None) == _abi.AR_ERR_PAGE and ops.last_status(None) == 0
        kk, vv = (s.plain.tokens(i, s.table[0], 64) for i in (0, 1))
        keep = np.r_[0:16, 32:64]
        want = attention(qf[:1].astype(np.float64), kk[keep], vv[keep], np.array([63]), True)
        assert_attention_close(o[:1].double().cpu().numpy(), *want, False)
        assert torch.equal(o[1:], s.ops.kv_cache_attention(s.cache, q, s.dtable, where[1])[1:])
        # the same in a call of many rows
        many, mf = s.rows(100, 4)
        o = s.ops.kv_cache_attention(s.cache, many, *where, s.ints([0, 60, 100]))
        assert ops.last_status(None) == _abi.AR_ERR_PAGE and ops.last_status(None) == 0
        pos = np.arange(4, 64)
        seen = np.where(pos < 16, pos, np.where(pos < 32, 15, pos - 16))
        want = attention(mf[:60].astype(np.float64), kk[keep], vv[keep], seen, True)
        assert_attention_close(o[:60].double().cpu().numpy(), *want, False)
        # writing: nothing of that page's tokens, the others are written
        before = [x.clone() for x in (s.cache.k, s.cache.v)]
        new, _ = s.rows(16, 2)
        s.ops.kv_cache_append(s.cache, new, new, table, s.ints([32, 64]), s.ints([0, 16, 16]))
        assert ops.last_status(None) == _abi.AR_ERR_PAGE
        assert torch.equal(before[0], s.cache.k) and torch.equal(before[1], s.cache.v)


def test_lengths_outside_the_table_are_reported(ops):
    import torch
    from autorust_b200 import _abi
    s = Setup(ops, 73, [64, 64], Hkv=1, D=64, page=16, fill=3)
    s.append([64, 64], [64, 64])
    q, qf = s.rows(2, 2)
    for length in (65, 2 ** 31 - 1):
        o = s.ops.kv_cache_attention(s.cache, q, s.dtable, s.ints([length, 64]))
        assert ops.last_status(None) == _abi.AR_ERR_PAGE
        assert torch.equal(o, s.ops.kv_cache_attention(s.cache, q, s.dtable, s.ints([64, 64])))  # the tokens that exist
        before = s.cache.k.clone()
        s.ops.kv_cache_append(s.cache, q[:, :1], q[:, :1], s.dtable, s.ints([length, 0]))
        assert ops.last_status(None) == _abi.AR_ERR_PAGE and torch.equal(before, s.cache.k)
        k, _ = s.ops.kv_cache_read(s.cache, s.dtable, s.ints([length, 64]), None, 2)
        assert ops.last_status(None) == _abi.AR_ERR_PAGE and (k[0] == 0).all()
    # a bound that is too small: the tokens in front of it
    o = s.ops.kv_cache_attention(s.cache, q, s.dtable, s.ints([64, 20]), max_length=32)
    assert ops.last_status(None) == _abi.AR_ERR_PAGE
    k, v = (s.plain.tokens(i, s.table[0], 32) for i in (0, 1))
    assert_attention_close(o[:1].double().cpu().numpy(), *attention(qf[:1].astype(np.float64), k, v, np.array([63]), True), False)
    # negative lengths are empty sequences; starts that lie outside the packing or run backwards touch nothing outside it
    o = s.ops.kv_cache_attention(s.cache, q, s.dtable, s.ints([-5, 64]))
    assert (o[0] == 0).all() and ops.last_status(None) == 0
    for starts in ([-3, 1, 900], [2, 1, 0], [0, 2 ** 31 - 1, 2 ** 31 - 1], [-2 ** 31, -1, 2]):
        out = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
        s.ops.kv_cache_attention(s.cache, q, s.dtable, s.ints([64, 64]), s.ints(starts), out=out[1:3])
        s.ops.kv_cache_read(s.cache, s.dtable, s.ints([64, 64]), s.ints(starts), 2, out=(out[1:3, :1], out[1:3, 1:]))
        s.ops.last_status(None)
        assert (out[0] == 0).all() and (out[3] == 0).all()


# ---- streams, graphs, runs --------------------------------------------------------------------------------------------------
def test_generation_loop(ops):
    """A prompt in chunks, then token by token, as a server runs it: every step's rows against 64 bits over the cache at that time."""
    s = Setup(ops, 81, [130, 90], Hkv=2, D=128, page=32, mean=True)
    done = [0, 0]
    for new in ([50, 7], [40, 50], [1, 1], [1, 1], [2, 1], [1, 1], [30, 1]):
        done = [d + n for d, n in zip(done, new)]
        s.append(done, new)
        s.check_attention(done, new, 8)
    s.check_pool()


def test_other_streams_and_graphs(ops):
    """Calls on two streams at once with workspaces of their own; a captured step replayed on new lengths and tokens gives the
    bits of the eager calls; two graphs that share one workspace, replayed after one another."""
    import torch
    lengths = [3000, 1500]
    s = Setup(ops, 91, [3050, 1550], Hkv=2, D=128, page=16)
    s.append(lengths, lengths)
    q = [s.rows(2, 8)[0] for _ in range(2)]
    where = (s.dtable, s.ints(lengths))
    want = [s.ops.kv_cache_attention(s.cache, x, *where) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    torch.cuda.synchronize()
    for i in (0, 1):
        got[i] = s.ops.kv_cache_attention(s.cache, q[i], *where, stream=streams[i])
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

    need = s.ops.kv_cache_attention_workspace(s.cache, 2, 8, 2, s.dtable.shape[1] * 16)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    k, v, qs = s.rows(2, 2)[0].clone(), s.rows(2, 2)[0].clone(), q[0].clone()
    at = s.ints(lengths)
    out = [torch.empty(2, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    graphs = []
    saved = [x.clone() for x in (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale)]
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            if i == 0:
                s.ops.kv_cache_append(s.cache, k, v, s.dtable, at)
            s.ops.kv_cache_attention(s.cache, qs, s.dtable, at, out=out[i], workspace=ws)
        graphs.append(graph)
    steps = [(s.rows(2, 2)[0], s.rows(2, 2)[0], s.rows(2, 8)[0]) for _ in range(3)]
    replayed = []
    for t, (kn, vn, qn) in enumerate(steps):
        k.copy_(kn); v.copy_(vn); qs.copy_(qn); at.copy_(s.ints([x + t + 1 for x in lengths]))
        graphs[0].replay()
        graphs[1].replay()
        replayed.append((out[0].clone(), out[1].clone()))
    pool = [x.clone() for x in (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale)]
    for x, y in zip((s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale), saved):
        x.copy_(y)
    for t, (kn, vn, qn) in enumerate(steps):
        now = s.ints([x + t + 1 for x in lengths])
        s.ops.kv_cache_append(s.cache, kn, vn, s.dtable, now)
        eager = s.ops.kv_cache_attention(s.cache, qn, s.dtable, now)
        assert torch.equal(eager, replayed[t][0]) and torch.equal(eager, replayed[t][1])
    for x, y in zip((s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale), pool):
        assert torch.equal(x, y)


def test_same_call_same_bits(ops):
    import torch
    s = Setup(ops, 95, [5000, 800, 33], Hkv=2, D=64, page=64, f32=True)
    s.append([5000, 800, 33], [5000, 800, 33])
    q, _ = s.rows(3, 12)
    where = (s.dtable, s.ints([5000, 800, 33]))
    first = s.ops.kv_cache_attention(s.cache, q, *where)
    for _ in range(5):
        assert torch.equal(first, s.ops.kv_cache_attention(s.cache, q, *where))


def test_many_rows_captured(ops):
    """The tensor-core kernel, whole and in parts, captured between an append and a read and replayed on other tokens."""
    import torch
    for lengths, new, heads in (([500, 300], [200, 130], 8), ([3000, 200], [300, 150], 4)):
        s = Setup(ops, 97, lengths, Hkv=2, D=64, page=32)
        s.append([x - n for x, n in zip(lengths, new)], [x - n for x, n in zip(lengths, new)])
        T = sum(new)
        starts, where = s.batch(lengths, new)
        k, v, q = s.rows(T, 2)[0].clone(), s.rows(T, 2)[0].clone(), s.rows(T, heads)[0].clone()
        need = s.ops.kv_cache_attention_workspace(s.cache, T, heads, 2, max(lengths))
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")

        def step():
            s.ops.kv_cache_append(s.cache, k, v, *where)
            o = s.ops.kv_cache_attention(s.cache, q, *where, max_length=max(lengths), workspace=ws)
            return o, s.ops.kv_cache_read(s.cache, *where, T)

        step()
        graph = torch.cuda.CUDAGraph()
        saved = [x.clone() for x in (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale)]
        with torch.cuda.graph(graph):
            o, (rk, rv) = step()
        for _ in range(3):
            for x, H in ((k, 2), (v, 2), (q, heads)):
                x.copy_(s.rows(T, H)[0])
            for x, y in zip((s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale), saved):
                x.copy_(y)
            graph.replay()
            got = [x.clone() for x in (o, rk, rv)]
            for x, y in zip((s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale), saved):
                x.copy_(y)
            eager, (ek, ev) = step()
            for x, y in zip(got, (eager, ek, ev)):
                assert torch.equal(x, y)
        assert ops.last_status(None) == 0


def test_a_pool_beyond_32_bit_offsets(ops):
    """Pages whose codes lie more than 2^32 bytes into the pool, and rows of packed tensors that do so too."""
    import torch
    Hkv, page, D = 8, 128, 128
    pages = (5 << 30) // (Hkv * page * D)
    cache = ops.kv_cache(pages, Hkv, page, D)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table = ints([[pages - 1, 0, pages - 2], [pages // 2, pages - 3, 1]])
    g = torch.Generator(device="cuda").manual_seed(5)
    n = [300, 129]
    T, wide = sum(n), 5_100_000  # elements between the rows: the last one lies 4.4 GB behind the first
    big = torch.empty((T - 1) * wide + 2 * Hkv * D, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.as_strided(big, (T, Hkv, D), (wide, D, 1), i * Hkv * D) for i in range(2))
    rows = torch.randn(2, T, Hkv, D, device="cuda", generator=g).to(torch.bfloat16)
    k.copy_(rows[0]); v.copy_(rows[1])
    where = (table, ints(n), ints([0, n[0], T]))
    ops.kv_cache_append(cache, k, v, *where)
    small = ops.kv_cache(8, Hkv, page, D)
    near = (ints([[5, 0, 2], [3, 7, 1]]), *where[1:])
    ops.kv_cache_append(small, rows[0], rows[1], *near)
    for far, close in zip(ops.kv_cache_read(cache, *where, T), ops.kv_cache_read(small, *near, T)):
        assert torch.equal(far, close)
    for m in (1, 40):
        q = torch.randn(2 * m, 16, D, device="cuda", generator=g).to(torch.bfloat16)
        out = torch.as_strided(big, (2 * m, 16, D), (wide * (T // (2 * m)) // 8 * 8 if m == 1 else wide, D, 1))
        few = ints([0, m, 2 * m])
        want = ops.kv_cache_attention(small, q, near[0], near[1], few)
        assert torch.equal(ops.kv_cache_attention(cache, q, table, near[1], few, out=out), want)
    assert ops.last_status(None) == 0


def test_copies_have_tensors_of_their_own(ops):
    import copy
    import io
    import torch
    s = Setup(ops, 61, [40, 9], Hkv=1, D=64, mean=True)
    s.append([40, 9], [40, 9])
    q, _ = s.rows(2, 2)
    where = (s.dtable, s.ints([40, 9]))
    want = ops.kv_cache_attention(s.cache, q, *where)
    file = io.BytesIO()
    torch.save(s.cache, file)
    file.seek(0)
    copies = [copy.deepcopy(s.cache), torch.load(file, weights_only=False)]
    s.cache.k.zero_()
    s.cache.v_scale.zero_()
    for c in copies:
        assert c.k.data_ptr() != s.cache.k.data_ptr() and not c.fp8
        assert torch.equal(ops.kv_cache_attention(c, q, *where), want)


def test_empty_calls(ops):
    import torch
    s = Setup(ops, 99, [10], Hkv=1, D=64)
    none = torch.empty(0, 1, 64, dtype=torch.bfloat16, device="cuda")
    where = (s.dtable, s.ints([10]), s.ints([0, 0]))
    s.ops.kv_cache_append(s.cache, none, none, *where)
    assert s.ops.kv_cache_read(s.cache, *where, 0)[0].shape == (0, 1, 64)
    assert s.ops.kv_cache_attention(s.cache, none, *where).shape == (0, 1, 64)
