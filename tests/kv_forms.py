"""Calls that take each form of the cache attention, for tests that have to reach all of them, and a bound on the results that looks only at
what a row sees."""
from __future__ import annotations

import numpy as np

from autorust_b200 import _abi

# name: lengths, rows of each sequence, kv heads, query heads
FORMS = {
    "8 rows whole": ([300, 45], [2, 1], 2, 8),
    "16 rows whole": ([300, 129], [5, 9], 2, 8),
    "8 rows cut": ([9000, 200], [2, 1], 1, 4),
    "16 rows cut": ([9000, 200], [9, 4], 1, 4),
    "many whole": ([640, 500, 77], [640, 260, 77], 2, 8),
    "many in parts": ([4000, 700], [300, 133], 1, 4),
}
BF16_ONLY = ("many whole", "many in parts")


def plan_of(cache, tokens, Hq, sequences, max_length, f32, causal=True):
    page = cache.k.shape[2]
    width = -(-max_length // page)
    batch = _abi.KvBatch(16, 16, 16, width, width, sequences, tokens)  # (placeholders: the sizes decide)
    return _abi.kv_plan(cache._pool, batch, _abi.DTYPE_F32 if f32 else _abi.DTYPE_BF16, Hq, max_length, causal)


def assert_form(name, cache, tokens, Hq, sequences, max_length, f32, causal=True):
    rows, ctas, parts = plan_of(cache, tokens, Hq, sequences, max_length, f32, causal)
    want = {"8": 8, "1": 16, "m": 256}[name[0]]
    assert (rows, ctas > 0, parts > 1) == (want, name.endswith("cut"), name.endswith("parts")), (name, rows, ctas, parts)


def attention(q, k, v, positions, causal, page, keep=None):
    """One sequence in 64 bits: q [n, Hq, D], k, v [L, Hkv, D].  The result; the weighted average of |v|; the largest sum |q k| / sqrt(D) over the
    keys a row sees; their number times the largest |v| of the pages they lie on (a later token of the last page may have set its scale).
    A row that sees no key has zeros everywhere.  keep [L]: keys that are not left out."""
    n, Hq, D = q.shape
    L, G, most_k = k.shape[0], Hq // k.shape[1], np.abs(k).max(initial=0.0)
    o, size, reach, most = np.zeros((n, Hq, D)), np.zeros((n, Hq, D)), np.zeros((n, Hq, 1)), np.zeros((n, Hq, 1))
    last = np.clip(np.asarray(positions) + 1 if causal else np.full(n, L), 0, L)
    seen = np.arange(L)[None, :] < last[:, None]
    if keep is not None:
        seen &= keep[None, :]
    rows = np.flatnonzero(seen.any(axis=1))
    if len(rows) == 0:
        return o, size, reach, most
    seen, held = seen[rows], np.minimum(L, -(-last[rows] // page) * page)
    for h in range(Hq):
        kk, vv, qq = k[:, h // G], v[:, h // G], q[rows, h]
        if most_k * np.abs(qq).max() < 1e9:
            s = qq @ kk.T
        else:  # (a matrix product may add equal rows in different orders, which decides between them where logits are huge)
            s = np.stack([(kk * x).sum(axis=1) for x in qq])
        s = np.where(seen, s / np.sqrt(D), -np.inf)
        p = np.exp(s - s.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        vv = np.nan_to_num(vv, nan=0.0)  # (a row that sees one has no result to compare)
        o[rows, h], size[rows, h] = p @ vv, p @ np.abs(vv)
        reach[rows, h, 0] = np.where(seen, np.abs(qq) @ np.abs(np.nan_to_num(kk, nan=0.0)).T, 0.0).max(axis=1) / np.sqrt(D)
        most[rows, h, 0] = seen.sum(axis=1) * np.maximum.accumulate(np.abs(vv).max(axis=1))[held - 1]
    return o, size, reach, most


def expect(s, qf, lengths, starts, causal=True, keep=None):
    """The rows of all sequences of a Setup's plain cache; keep: by sequence, the keys that are not left out."""
    parts = []
    for b, length in enumerate(lengths):
        n = int(starts[b + 1] - starts[b])
        k, v = (s.plain.tokens(which, s.table[b], int(length)) for which in (0, 1))
        parts.append(attention(qf[starts[b]:starts[b + 1]].astype(np.float64), k, v, int(length) - n + np.arange(n), causal, s.page, (keep or {}).get(b)))
    return [np.concatenate(p) for p in zip(*parts)]


def assert_close(got, o, size, reach, most, f32, keys, exact_logits=False):
    """As kv_plain.assert_attention_close derives it, with `most` of what a row sees.  A tensor-core sum of values is cut at 2^-24 of its largest
    partial sum for each of its products, so that `keys` of them, 16 at a time and in two terms for f32 tensors, add 2^-24 each of the weighted
    average of |v|.  exact_logits: the call's logits are all the same for a row, or so far apart that only the largest has a weight."""
    import torch
    half = torch.finfo(torch.float32 if f32 else torch.bfloat16).eps / 2
    weight = (2.0 ** -20 if f32 else 2.0 ** -11 + 1.1e-4 + 2.0 ** -20) + keys / 8 * 2.0 ** -24
    if not exact_logits:
        weight = weight + 2.0 * 2.0 ** -18 * reach
    assert np.all(np.isfinite(got))
    err, tol = np.abs(got - o), half * np.abs(o) + weight * size + 2.0 ** (-36 if f32 else -32) * most
    worst = np.unravel_index(np.argmax(err - tol), err.shape)
    assert np.all(err <= tol), (worst, got[worst], o[worst], err[worst], tol[worst])
