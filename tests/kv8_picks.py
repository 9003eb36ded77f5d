"""Data on which a lost tile shows: each query head has one key whose score is 40 log2 units above all
others (its weight is 1 - n 2^-40), with a value of its own, so that the output is that value, wherever
the key lies and however the work was split. Shared by the GPU tests and the CPU test that wrong
results are told from right ones."""
from __future__ import annotations

import numpy as np

SCALE_LOG2 = 5.0  # times 1.0 in the query and 8.0 in the key: 40
KEY = 8.0


def queries(heads, d):
    """Head h asks for dimension h % d."""
    q = np.zeros((heads, d))
    q[np.arange(heads), np.arange(heads) % d] = 1.0
    return q


def keys(n, d, positions):
    """Zero but for the key at each position, which has the dimension of its head."""
    k = np.zeros((n, d))
    k[positions, np.arange(len(positions)) % d] = KEY
    return k


class Picked:
    """What the heads should give over values v [n][d], and how far off they may be."""

    def __init__(self, v, visible, u_out, u_weight):
        self.v, self.visible, self.u_out, self.u_weight = v, np.asarray(visible), u_out, u_weight
        rows = v[self.visible]
        self.mean, self.size, self.most = rows.mean(0), np.abs(rows).mean(0), np.abs(rows).max()

    def want(self, positions):
        """The values of the heads' keys, the mean of what they see where that is hidden."""
        return np.stack([self.v[p] if self.visible[p] else self.mean for p in positions])

    def bound(self, positions):
        """The output's rounding, that of one weight that is not in the sum, fp32 sums of up to 64
        terms in a row, the n keys of weight 2^-40 in product and sum; where the key is hidden, every
        weight's rounding, in product and sum."""
        some = np.stack([np.zeros_like(self.mean) if self.visible[p] else self.size for p in positions])
        return (np.abs(self.want(positions)) * (self.u_out + self.u_weight + 2.0 ** -17) +
                some * 2 * self.u_weight + 2 * len(self.v) * 2.0 ** -40 * self.most + 2.0 ** -24)


def tiles_of(visible, tile=128):
    """The tiles that hold a visible key."""
    v = np.append(np.asarray(visible), np.zeros(-len(visible) % tile, bool)).reshape(-1, tile)
    return np.flatnonzero(v.any(1))


def one_of_each_tile(rng, visible, tile=128):
    """A visible key of every tile, the first or the last one in the tiles at the ends."""
    out = []
    tiles = tiles_of(visible, tile)
    for i, t in enumerate(tiles):
        own = np.flatnonzero(visible[t * tile:(t + 1) * tile]) + t * tile
        out.append(own[0] if i % 3 == 0 else own[-1] if i % 3 == 1 or t == tiles[-1] else rng.choice(own))
    return np.array(out)


def mixed(q, k, v, v_scale, scale_log2, u_out):
    """Attention rows q [h][d] over k, v [n][d] (v with its pages' scales v_scale [n] in it), and a bound
    from the weights as they are: the output's rounding; each weight times scale to fp16, 2^-11 of it
    or 2^-25 of the largest; the scores' fp32 error (d + 8) 2^-24 of the sum of |q k|, in numerator and
    sum; fp32 sums of up to 64 terms in a row and exponentials, 2^-17."""
    out, tol = [], []
    d = q.shape[1]
    for x in q:
        s = (k @ x) * scale_log2
        p = np.exp2(s - s.max())
        p /= p.sum()
        w = p * v_scale
        code = np.abs(v) / np.where(v_scale > 0, v_scale, 1.0)[:, None]
        o = p @ v
        ds = (d + 8) * 2.0 ** -24 * (np.abs(k) @ np.abs(x)).max() * scale_log2
        out.append(o)
        tol.append(u_out * np.abs(o) + np.maximum(w * 2.0 ** -11, w.max() * 2.0 ** -25) @ code +
                   (2 * np.log(2) * ds + 2.0 ** -17) * (p @ np.abs(v)) + 2.0 ** -24)
    return np.stack(out), np.stack(tol)
