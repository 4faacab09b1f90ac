"""The 8-bit cache restated plainly for the tests: writing in the f32 steps of the definition (so that codes and scales are
compared bit for bit), attention in 64 bits over the values the codes stand for."""
from __future__ import annotations

import numpy as np

FLOOR = np.float32(2.0 ** -60)


def e4m3_table() -> np.ndarray:
    code = np.arange(256)
    e, m = (code >> 3) & 15, code & 7
    x = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e.astype(np.float64) - 10))
    x = np.where(code & 128, -x, x)
    x[(code & 127) == 127] = np.nan
    return x


TABLE = e4m3_table()


def to_e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest code, ties to the even one, of f32 values inside +-448."""
    mag = np.abs(x.astype(np.float64))
    pos = TABLE[:127]  # 0 .. 448, ascending
    hi = np.clip(np.searchsorted(pos, mag), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = pos[hi] - mag, mag - pos[lo]
    code = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 0, hi, lo)))
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


class PlainCache:
    def __init__(self, pages, Hkv, page, D, fp8, k_mean=None, fill=0):
        kind = np.uint8 if fp8 else np.int8
        self.codes = [np.full((pages, Hkv, page, D), fill, kind) for _ in range(2)]
        self.scales = [np.zeros((pages, Hkv), np.float32) for _ in range(2)]
        self.page, self.fp8, self.k_mean = page, fp8, k_mean

    def _scale(self, amax):
        if not np.isfinite(amax):
            return np.float32(np.nan)
        if not self.fp8:
            return max(np.float32(amax) / np.float32(127.0), FLOOR)
        k = -60
        while 448.0 * 2.0 ** k < float(amax):
            k += 1
        return np.float32(2.0 ** k)

    def _encode(self, x):
        if self.fp8:
            return to_e4m3(x)
        return np.clip(np.rint(x), -127, 127).astype(np.int8)

    def values(self, which):
        c = self.codes[which]
        return (TABLE[c] if self.fp8 else c).astype(np.float32)

    def append(self, k, v, table, lengths, starts):
        """k, v [T, Hkv, D] f32."""
        if self.k_mean is not None:
            k = k - self.k_mean
        for b in range(len(lengths)):
            n = starts[b + 1] - starts[b]
            first = int(lengths[b]) - n
            lo = max(first, 0)
            for j in range(lo // self.page, (int(lengths[b]) + self.page - 1) // self.page):
                t0, t1 = max(lo - j * self.page, 0), min(int(lengths[b]) - j * self.page, self.page)
                if t1 <= t0:
                    continue
                pg = table[b][j]
                rows = slice(starts[b] + j * self.page + t0 - first, starts[b] + j * self.page + t1 - first)
                for which, x in ((0, k), (1, v)):
                    for h in range(x.shape[1]):
                        self._write(which, pg, h, t0, t1, x[rows, h])

    def _write(self, which, pg, h, t0, t1, x):
        codes, scales = self.codes[which], self.scales[which]
        s = self._scale(np.max(np.abs(x)))
        s0 = scales[pg, h]
        if t0 > 0 and not np.isnan(s) and not s > s0:
            s = s0
        if np.isnan(s):
            codes[pg, h, t0:t1] = 0
        else:
            if t0 > 0 and s > s0:
                old = (TABLE[codes[pg, h, :t0]] if self.fp8 else codes[pg, h, :t0]).astype(np.float32)
                codes[pg, h, :t0] = self._encode(old * np.float32(s0 / s))
            codes[pg, h, t0:t1] = self._encode(x * np.float32(np.float32(1.0) / s))
        scales[pg, h] = s

    def tokens(self, which, row, length, dtype=np.float64):
        """[length, Hkv, D]: what the codes stand for, without the mean."""
        n = (length + self.page - 1) // self.page
        at = np.asarray(row[:n], dtype=np.int64)
        x = self.values(which)[at].astype(dtype) * self.scales[which][at][:, :, None, None].astype(dtype)
        return x.transpose(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])[:length]


def attention(q, k, v, n_rows_pos, causal):
    """One sequence in 64 bits.  q [n, Hq, D], k, v [L, Hkv, D], n_rows_pos [n] positions.  Returns (o, size, reach, most): the
    result, the weighted average of |v|, the largest sum |q k| / sqrt(D) over the keys a row sees, and their number times
    the largest |v| of the head."""
    n, Hq, D = q.shape
    L, Hkv = k.shape[0], k.shape[1]
    G = Hq // Hkv
    o, size, reach, most = np.zeros((n, Hq, D)), np.zeros((n, Hq, D)), np.zeros((n, Hq, 1)), np.zeros((n, Hq, 1))
    for i in range(n):
        last = min(L, n_rows_pos[i] + 1) if causal else L
        if last <= 0:
            continue
        for h in range(Hq):
            kk, vv = k[:last, h // G], v[:last, h // G]
            s = kk @ q[i, h] / np.sqrt(D)
            p = np.exp(s - s.max())
            p /= p.sum()
            o[i, h], size[i, h] = p @ vv, p @ np.abs(vv)
            reach[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() / np.sqrt(D)
            most[i, h] = last * np.abs(v[:, h // G]).max()
    return o, size, reach, most


def assert_attention_close(got, o, size, reach, most, f32):
    """What the kernel may be off by.  A logit: the products of 16 channels are added at once, cut at 2^-24 of the largest, and
    at most 16 such sums after one another (two passes for f32 tensors), each rounded to f32 -- under 2^-18 of sum |q k| / sqrt(D)
    in all, with the f32 factors around it.  That shifts a weight by at most that much relative to the sum, twice (weight and
    sum).  The weight itself is rounded to f16, half a step 2^-11 (f32 tensors: two f16 terms, 2^-22), its exponential
    is within 2^-21 -- in calls of many rows, a quarter of them within 1.1e-4 (the polynomial of the bf16 forward) --; sums and
    joins are f32, 2^-21 in all.  The result is rounded once to its type.
    Weights that are small against the row's largest meet the end of the f16 range: with the largest weight times page scale
    at 2^12 or more (many rows: 2^8), a weight is rounded to a multiple of 2^-24, so it is off by up to 2^-37 (2^-33) of
    the largest, whatever its own size.  A page's largest code times its scale is at most twice the largest value that
    set the scale (E4M3: the scale is the next power of two), so each key adds at most 2^-36 (2^-32) of the largest |v|."""
    import torch
    half = torch.finfo(torch.float32 if f32 else torch.bfloat16).eps / 2
    weight = (2.0 ** -20 if f32 else 2.0 ** -11 + 1.1e-4 + 2.0 ** -20) + 2.0 * 2.0 ** -18 * reach
    err, tol = np.abs(got - o), half * np.abs(o) + weight * size + 2.0 ** (-36 if f32 else -32) * most
    assert np.all(np.isfinite(got))
    worst = np.unravel_index(np.argmax(err - tol), err.shape)
    assert np.all(err <= tol), (worst, got[worst], o[worst], err[worst], tol[worst])
    if f32 and o.size >= 1024:
        # the errors of different weights are independent: far below the bound in the mean.  One f16 term instead of two
        # would leave 2^-12 of a logit or weight, about 1e-4
        assert np.sqrt(np.mean(err ** 2)) <= 2.0 ** -18 * np.sqrt(np.mean(size ** 2))
