"""Long splits of the serving attentions on the GPU, a key of every tile picked in turn (kv8_picks.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv8_picks as picks
import kv8_plain as plain
from test_gpu_serving import TYPES, Cache, _done, _dt, _f64, _ints

pytestmark = pytest.mark.gpu


def _code(x):
    return int(plain.to_e4m3(np.array([float(x)]))[0])


def _pick_every_tile(gpu, t, n, H, G, d, P, window, sinks, ws=None, lens=None, most=None):
    """Sequence 0 of n tokens (and others of `lens` beside it), every tile's keys in rounds of G heads."""
    rng = np.random.default_rng(n + G + window)
    lens = [n] + list(lens or [])
    B, need = len(lens), [-(-x // P) for x in lens]
    c = Cache(gpu, sum(need), H, P, d)
    order = rng.permutation(sum(need)).astype(np.int32)
    table = np.full((B, max(need)), -1, np.int32)
    for b in range(B):
        table[b, :need[b]] = order[sum(need[:b]):sum(need[:b + 1])]
    c.k.fill_(0)
    c.ks.fill_(1.0)
    c.v.copy_(torch.randint(0, 256, c.v.shape, dtype=torch.uint8, device="cuda") & 0xF7)  # no NaN code
    c.vs.copy_(torch.from_numpy(rng.uniform(0.5, 2.0, tuple(c.vs.shape)).astype(np.float32)) * 2.0 ** -8)
    row, slot = table[0][np.arange(n) // P], np.arange(n) % P
    v = plain.E4M3[c.v.cpu().numpy()[row, :, slot]] * c.vs.cpu().double().numpy()[row][:, :, None]  # [n][H][d]
    visible = np.ones(n, bool)
    if window:
        visible[sinks:max(n - window, sinks)] = False
    each = picks.one_of_each_tile(rng, visible)
    if most:  # the tiles at the ends and some between
        each = np.concatenate([each[:most // 4], rng.permutation(each[most // 4:-(most // 4)])[:most // 2], each[-(most // 4):]])
    each = rng.permutation(np.append(each, np.flatnonzero(~visible)[:1]))  # and a hidden one
    ws = ws if ws is not None else torch.zeros(gpu.kv8_attn_workspace(c.handle, B, H * G)[1], dtype=torch.uint8,
                                               device="cuda")
    tab, ln = _ints(table), _ints(lens)
    q = torch.from_numpy(np.tile(picks.queries(G, d), (B, H, 1)).reshape(B, H * G, d)).to("cuda", t)
    outs, chosen = [], []
    for at in range(0, len(each), G):
        pos = np.resize(each[at:at + G], G)
        where = (torch.from_numpy(row[pos]).long().cuda(), slice(None), torch.from_numpy(slot[pos]).cuda(),
                 torch.arange(G, device="cuda") % d)
        c.k[where] = _code(picks.KEY)
        o = torch.full_like(q, 7.0)
        assert gpu.kv8_attn(c.handle, q, o, tab, table.shape[1], ln, B, H * G, picks.SCALE_LOG2, _dt(gpu, t), ws,
                            ws.numel(), window=window, sinks=sinks) == 0
        c.k[where] = 0
        outs.append(o[0])
        chosen.append(pos)
    _done(gpu)
    u = torch.finfo(t).eps / 2
    expect = [picks.Picked(v[:, h], visible, u, 2.0 ** -11) for h in range(H)]
    for o, pos in zip(outs, chosen):
        got = _f64(o).reshape(H, G, d)
        for h in range(H):
            off = np.abs(got[h] - expect[h].want(pos)) - expect[h].bound(pos)
            assert (off <= 0).all(), (pos[(off > 0).any(1)], off.max())


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("n,H,G,d,P,window,sinks", [
    (3000, 2, 4, 128, 32, 0, 0), (7000, 4, 2, 64, 32, 0, 0), (20011, 1, 8, 64, 128, 0, 0),
    (20011, 1, 8, 64, 128, 9000, 128), (1000, 1, 20, 128, 16, 300, 17), (4097, 3, 16, 128, 64, 0, 0)])
def test_attn_every_tile_counts(gpu, n, H, G, d, P, window, sinks, t):
    _pick_every_tile(gpu, t, n, H, G, d, P, window, sinks)


def test_attn_every_tile_counts_beside_others(gpu):
    """A long sequence among short ones, and one workspace for all shapes."""
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    _pick_every_tile(gpu, torch.float16, 5000, 2, 8, 128, 16, 0, 0, ws=ws, lens=[17, 3333, 0, 900])
    _pick_every_tile(gpu, torch.bfloat16, 900, 1, 16, 64, 32, 0, 0, ws=ws, lens=[100] * 40)
    _pick_every_tile(gpu, torch.float16, 3000, 2, 4, 128, 32, 1000, 4, ws=ws, lens=[5])


@pytest.mark.parametrize("G,t,window,sinks", [(2, torch.float16, 0, 0), (16, torch.float16, 0, 0),
                                              (16, torch.bfloat16, 0, 0), (16, torch.bfloat16, 200000, 4)])
def test_attn_every_part_counts_of_the_longest(gpu, G, t, window, sinks):
    """300001 tokens: a part for every block of the GPU, joined in two steps. With 16 heads every tile."""
    _pick_every_tile(gpu, t, 300001, 1, G, 64, 128, window, sinks, most=400 if G == 2 else None)


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("Nq,Nk,Hq,d,window,sinks", [
    (4, 300000, 2, 64, 1000, 130), (2, 200001, 4, 128, 0, 0), (3, 20000, 4, 64, 0, 0), (130, 3000, 1, 128, 700, 200)])
def test_window_every_tile_counts(gpu, Nq, Nk, Hq, d, window, sinks, t):
    """Late rows of long sequences: each row and head of a call picks a key of a tile in turn, what the
    row does not see among them."""
    rng = np.random.default_rng(Nk + d)
    rows = sorted({0, 1, Nq - 1})
    v = torch.randn(1, 1, Nk, d, device="cuda").to(t)
    k = torch.zeros(1, 1, Nk, d, device="cuda").to(t)
    vn = _f64(v)[0, 0]
    ask = [(h, i) for h in range(Hq) for i in rows]
    q = torch.zeros(1, Hq, Nq, d, device="cuda").to(t)
    for x, (h, i) in enumerate(ask):
        q[0, h, i, x] = 1.0
    seen = {i: np.isin(np.arange(Nk), plain.visible(i + Nk - Nq, Nk, window, sinks)) for i in rows}
    each = picks.one_of_each_tile(rng, seen[rows[-1]])
    if len(each) > 300:
        each = np.concatenate([each[:20], rng.permutation(each[20:-20])[:200], each[-20:]])
    extra = [p for i in rows for p in (i + Nk - Nq, i + Nk - Nq + 1) if p < Nk]  # its own, and the next one
    if window:
        extra += [p for i in rows for p in (i + Nk - Nq - window, i + Nk - Nq - window + 1)] + [sinks - 1, sinks]
    each = rng.permutation(np.append(each, extra))
    u = torch.finfo(t).eps / 2
    expect = {i: picks.Picked(vn, seen[i], u, u) for i in rows}
    for at in range(0, len(each), len(ask)):
        pos = np.resize(each[at:at + len(ask)], len(ask))
        where = (0, 0, torch.from_numpy(pos).cuda(), torch.arange(len(ask), device="cuda"))
        k[where] = picks.KEY
        o = torch.full_like(q, 7.0)
        assert gpu.flash_window_fwd(q, k, v, o, 1, Hq, 1, Nq, Nk, d, picks.SCALE_LOG2, _dt(gpu, t), window=window,
                                    sinks=sinks) == 0
        k[where] = 0
        _done(gpu)
        got = _f64(o[0])
        for x, (h, i) in enumerate(ask):
            off = np.abs(got[h, i] - expect[i].want(pos[x:x + 1])) - expect[i].bound(pos[x:x + 1])
            assert (off <= 0).all(), (h, i, pos[x], off.max())


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("n,G,d,window", [(3000, 4, 128, 0), (20011, 8, 64, 0), (300001, 16, 64, 0),
                                          (300001, 4, 64, 200000)])
def test_attn_mixed_values_of_long_sequences(gpu, n, G, d, window, t):
    """Random keys and values, compared within a bound from the actual weights."""
    P = 64
    rng = np.random.default_rng(n + G)
    pages = -(-n // P)
    c = Cache(gpu, pages, 1, P, d)
    for codes, scales in ((c.k, c.ks), (c.v, c.vs)):
        codes.copy_((torch.randn(codes.shape, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
        scales.copy_(torch.from_numpy(rng.uniform(0.5, 2, (pages, 1)).astype(np.float32)) * 2.0 ** -7)
    table = rng.permutation(pages).astype(np.int32)[None]
    q = torch.randn(1, G, d, device="cuda").to(t)
    o = torch.full_like(q, 7.0)
    ws = torch.zeros(gpu.kv8_attn_workspace(c.handle, 1, G)[1], dtype=torch.uint8, device="cuda")
    scale = 1.4426950408889634 / d ** 0.5
    assert gpu.kv8_attn(c.handle, q, o, _ints(table), pages, _ints([n]), 1, G, scale, _dt(gpu, t), ws, ws.numel(),
                        window=window, sinks=4) == 0
    _done(gpu)
    seen = plain.visible(n - 1, n, window, 4)
    page, slot = table[0][seen // P], seen % P
    kc, ks, vc, vs = c.host()
    k = plain.E4M3[kc[page, 0, slot]] * ks[page, 0].astype(np.float64)[:, None]
    v = plain.E4M3[vc[page, 0, slot]] * vs[page, 0].astype(np.float64)[:, None]
    want, tol = picks.mixed(_f64(q)[0], k, v, vs[page, 0].astype(np.float64), scale, torch.finfo(t).eps / 2)
    off = np.abs(_f64(o)[0] - want) - tol
    assert (off <= 0).all(), (off.max(), tol.min(), np.abs(want).max())
