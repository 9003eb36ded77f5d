"""The comparison that the GPU tests of long splits make tells wrong results from right ones, on the
CPU: zeros, a result without one tile, one from the first quarter of the tiles, one in which a part was
added twice."""
from __future__ import annotations

import numpy as np
import pytest

import kv8_picks as picks
import kv8_plain as plain


@pytest.mark.parametrize("u_out,u_weight", [(2.0 ** -11, 2.0 ** -11), (2.0 ** -8, 2.0 ** -11), (2.0 ** -8, 2.0 ** -8)])
@pytest.mark.parametrize("n,window,sinks", [(20000, 0, 0), (20000, 9000, 130), (3001, 0, 0)])
def test_wrong_results_are_rejected(n, window, sinks, u_out, u_weight):
    rng, d = np.random.default_rng(n + window), 64
    v = rng.standard_normal((n, d))
    visible = np.ones(n, bool)
    if window:
        visible[sinks:n - window] = False
    each = picks.one_of_each_tile(rng, visible)
    assert sorted(each // 128) == picks.tiles_of(visible).tolist() and visible[each].all()
    pos = each[rng.permutation(len(each))[:16]]
    q = picks.queries(len(pos), d)
    k = picks.keys(n, d, pos)
    expect = picks.Picked(v, visible, u_out, u_weight)
    want, tol = expect.want(pos), expect.bound(pos)

    def result(keep):
        return np.stack([plain._row(x, k[keep], v[keep], picks.SCALE_LOG2) for x in q])

    def passes(got):
        return (np.abs(got - want) <= tol).all(1)

    assert passes(result(visible)).all()
    assert not passes(np.zeros_like(want)).any()
    for i, p in enumerate(pos):  # without the tile of that key
        keep = visible.copy()
        keep[p // 128 * 128:(p // 128 + 1) * 128] = False
        assert not passes(result(keep))[i]
    tiles = picks.tiles_of(visible)
    keep = visible.copy()
    keep[tiles[len(tiles) // 4] * 128:] = False
    assert not passes(result(keep))[pos >= tiles[len(tiles) // 4] * 128].any()
    assert not passes(result(visible) * 2).any()


@pytest.mark.parametrize("n,u_out", [(20000, 2.0 ** -11), (300000, 2.0 ** -8)])
def test_mixed_results_without_a_part_are_rejected(n, u_out):
    """Random data, whose outputs shrink with the root of the keys: the bound from the actual weights
    still tells zeros, half of the keys and a lost eighth from the result."""
    rng, d = np.random.default_rng(n), 64
    q, k, v = rng.standard_normal((3, d)), rng.standard_normal((n, d)), rng.standard_normal((n, d))
    scale = 1.4426950408889634 / 8
    want, tol = picks.mixed(q, k, v, np.ones(n), scale, u_out)
    assert all(np.abs(plain._row(x, k, v, scale) - w).max() < 1e-12 for x, w in zip(q, want))
    for lost in (slice(0, n), slice(n // 2, n), slice(n // 4, n // 4 + n // 8)):
        keep = np.ones(n, bool)
        keep[lost] = False
        for x, w, t in zip(q, want, tol):
            got = plain._row(x, k[keep], v[keep], scale)
            assert not (np.abs(got - w) <= t).all(), lost
