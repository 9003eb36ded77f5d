"""Plain float64 forms of the serving operators (window attention, 8-bit paged
K/V cache) for the tests, written from their definitions with numpy."""
from __future__ import annotations

import math

import numpy as np


def e4m3_values() -> np.ndarray:
    """The value of each of the 256 codes: sign, 4 exponent bits (bias 7), 3 mantissa bits;
    0x7F and 0xFF are NaN."""
    out = np.empty(256)
    for c in range(256):
        sign, e, m = c >> 7, (c >> 3) & 15, c & 7
        v = (m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[c] = math.nan if (e == 15 and m == 7) else (-v if sign else v)
    return out


E4M3 = e4m3_values()


def to_e4m3(x: np.ndarray) -> np.ndarray:
    """Codes of the nearest values, ties to the even code; past 448 the largest; NaN stays NaN."""
    a = np.minimum(np.abs(x), 448.0)
    pos = E4M3[:127]
    hi = np.clip(np.searchsorted(pos, np.where(np.isnan(a), 0, a)), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - pos[lo], pos[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    code = np.where(np.isnan(x), 0x7F, code).astype(np.uint8)
    return np.where(np.signbit(x) & ~np.isnan(x), code | 0x80, code).astype(np.uint8)


def block_scale(x: np.ndarray) -> float:
    """2^e, the smallest with every finite |x| <= 448 * 2^e, e in [-100, 119]."""
    a = np.abs(x[np.isfinite(x)])
    top = a.max() if a.size else 0.0
    e = -100
    while e < 119 and top > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(codes, scales, new, table, start, counts, page_size):
    """codes [pages][H][P][d] uint8 and scales [pages][H] in place; new [T][H][d]."""
    t0 = 0
    for b, n in enumerate(counts):
        at, end = start[b], start[b] + n
        while at < end:
            stop = min(end, (at // page_size + 1) * page_size)
            x = new[t0 + at - start[b]:t0 + stop - start[b]]
            page, slot = table[b][at // page_size], at % page_size
            for h in range(new.shape[1]):
                s = block_scale(x[:, h])
                if slot:
                    old = float(scales[page, h])
                    s = max(s, old)
                    if s != old:
                        codes[page, h, :slot] = to_e4m3(E4M3[codes[page, h, :slot]] * old / s)
                scales[page, h] = s
                codes[page, h, slot:slot + len(x)] = to_e4m3(x[:, h] / s)
            at = stop
        t0 += n


def visible(pos, n, window, sinks):
    """Keys below n that the token at `pos` sees."""
    j = np.arange(max(0, min(n, pos + 1)))
    return j if window == 0 else j[(pos - j < window) | (j < sinks)]


def _row(q, k, v, scale_log2):
    """One softmax row in base 2 over the given keys."""
    if len(k) == 0:
        return np.zeros(q.shape[-1])
    s = (k @ q) * scale_log2
    p = np.exp2(s - s.max())
    return (p / p.sum()) @ v


def window_attn(q, k, v, lens, window, sinks, scale_log2, rows=None):
    """q [B][Hq][Nq][d], k, v [B][Hkv][Nk][d]: float64 rows (all, or those listed), None where a
    row is left as it was."""
    B, Hq, Nq, d = q.shape
    Hkv, Nk = k.shape[1], k.shape[2]
    out = {}
    for b in range(B):
        n = Nk if lens is None else min(max(int(lens[b]), 0), Nk)
        for h in range(Hq):
            for i in range(Nq) if rows is None else rows:
                t = i + Nk - Nq
                if lens is not None and t >= n:
                    out[b, h, i] = None
                    continue
                j = visible(t, n, window, sinks)
                out[b, h, i] = _row(q[b, h, i], k[b, h // (Hq // Hkv), j], v[b, h // (Hq // Hkv), j],
                                    scale_log2)
    return out


def cache_attn(q, kc, ks, vc, vs, table, lens, window, sinks, scale_log2, page_size):
    """q [B][Hq][d] against codes [pages][H][P][d] and scales [pages][H]."""
    B, Hq, d = q.shape
    H = kc.shape[1]
    out = np.zeros((B, Hq, d))
    for b in range(B):
        j = visible(int(lens[b]) - 1, int(lens[b]), window, sinks)
        page = np.asarray(table[b])[j // page_size]
        for h in range(H):
            k = E4M3[kc[page, h, j % page_size]] * ks[page, h].astype(np.float64)[:, None]
            v = E4M3[vc[page, h, j % page_size]] * vs[page, h].astype(np.float64)[:, None]
            for g in range(h * (Hq // H), (h + 1) * (Hq // H)):
                out[b, g] = _row(q[b, g], k, v, scale_log2)
    return out
