"""The serving entries on the GPU against their plain float64 forms
(kv8_plain.py): prompt attention through a window with sinks, the 8-bit paged
cache's append, single-token attention and page copy, and a run of them
together.

Tolerances. Codes, scales and copies are exact. An attention output o over
values of magnitude at most V differs from float64 by at most
  u_out |o|            the output's rounding (u = eps / 2 of its type),
  2 u_P V              the weights' rounding to 16 bits, numerator and sum,
  2 ln2 ds V           the scores' fp32 error ds = (d + 8) 2^-24 S in log2
                       units, S = the largest sum |q k| * scale_log2,
  2^-20 V              exponentials, fp32 sums, the division,
  n 2^-25 V            fp16 weights below 2^-14 (n keys),
  2^-24                an fp16 output below its normal range."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import kv8_plain as plain

pytestmark = pytest.mark.gpu
LOG2E = 1.4426950408889634
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _dt(gpu, t):
    return gpu.Dtype.F16 if t is torch.float16 else gpu.Dtype.BF16


def _tol(want, t, u_p, vmax, smax, d, n):
    u = torch.finfo(t).eps / 2
    return (u * np.abs(want) + vmax * (2 * u_p + 2 * math.log(2) * (d + 8) * 2.0 ** -24 * smax +
                                       2.0 ** -20 + n * 2.0 ** -25) + 2.0 ** -24)


def _f64(x):
    return x.detach().cpu().double().numpy()


def _done(gpu):
    torch.cuda.synchronize()
    assert gpu.kernel_error(True) == 0


# ------------------------------------------------------------------ window
def _window_case(gpu, t, B, Hq, Hkv, Nq, Nk, d, window, sinks, lens=None, tokens_first=False,
                 q_scale=1.0, seed=0, rows=None):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def make(H, N, scale=1.0):
        shape = (B, N, H, d) if tokens_first else (B, H, N, d)
        x = (torch.randn(*shape, device="cuda", generator=g) * scale).to(t)
        return x.transpose(1, 2) if tokens_first else x

    q, k, v = make(Hq, Nq, q_scale), make(Hkv, Nk), make(Hkv, Nk)
    o = torch.full((B, Nq, Hq, d) if tokens_first else (B, Hq, Nq, d), 7.0, dtype=t, device="cuda")
    o = o.transpose(1, 2) if tokens_first else o
    dev_lens = None
    if lens is not None:
        dev_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for b, n in enumerate(lens):  # the padding holds what an earlier batch left
            for x in (k, v):
                x[b, :, max(n, 0):] = float("nan")
                x[b, :, max(n, 0) + 1::2] = float("inf")
    scale = LOG2E / math.sqrt(d)
    st = [x.stride()[:3] for x in (q, k, v, o)] if tokens_first else [None] * 4
    assert gpu.flash_window_fwd(q, k, v, o, B, Hq, Hkv, Nq, Nk, d, scale, _dt(gpu, t), window=window,
                                sinks=sinks, lens=dev_lens, q_strides=st[0], k_strides=st[1],
                                v_strides=st[2], o_strides=st[3]) == 0
    _done(gpu)
    got = _f64(o)
    qn, kn, vn = _f64(q), _f64(k), _f64(v)
    want = plain.window_attn(qn, kn, vn, lens, window, sinks, scale, rows)
    finite = np.where(np.isfinite(kn), kn, 0.0)
    smax = np.abs(qn).sum(-1).max() * np.abs(finite).max() * scale
    vmax = np.abs(vn[np.isfinite(vn)]).max() if np.isfinite(vn).any() else 0.0
    u_p = torch.finfo(t).eps / 2
    for (b, h, i), w in want.items():
        if w is None:
            assert (got[b, h, i] == 7.0).all(), (b, h, i)
            continue
        tol = _tol(w, t, u_p, vmax, smax, d, Nk)
        assert (np.abs(got[b, h, i] - w) <= tol).all(), (b, h, i, np.abs(got[b, h, i] - w).max(), tol.min())
    return q, k, v, o


WINDOW_SHAPES = [
    # B, Hq, Hkv, Nq, Nk, window, sinks
    (1, 1, 1, 1, 1, 0, 0), (2, 4, 2, 1, 300, 100, 4), (1, 2, 1, 5, 5, 1, 0), (1, 2, 1, 130, 130, 1, 1),
    (1, 3, 1, 129, 129, 64, 0), (2, 2, 2, 257, 257, 0, 0), (1, 4, 2, 300, 300, 128, 0),
    (1, 4, 4, 384, 384, 127, 3), (1, 6, 2, 400, 400, 129, 130), (1, 7, 1, 200, 333, 90, 200),
    (1, 2, 1, 100, 640, 256, 5), (1, 1, 1, 640, 640, 200, 300), (1, 2, 2, 513, 513, 300, 128),
    (1, 2, 1, 150, 20, 8, 2), (1, 4, 1, 300, 130, 0, 0), (3, 2, 1, 127, 128, 5000, 7),
    (1, 16, 2, 70, 260, 33, 129),
]


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("shape", WINDOW_SHAPES)
def test_window_shapes(gpu, shape, d, t):
    B, Hq, Hkv, Nq, Nk, window, sinks = shape
    _window_case(gpu, t, B, Hq, Hkv, Nq, Nk, d, window, sinks, seed=Nq + Nk + window)


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("Nq,Nk,lens", [(300, 300, [300, 1, 0, 171]), (260, 260, [256, 128, 400, -3]),
                                        (64, 257, [257, 193, 194, 100]), (200, 90, [90, 0, 1, 89])])
def test_window_padded_batch(gpu, Nq, Nk, lens, t):
    """NaN and infinities behind each sequence's end; rows there stay as they were."""
    _window_case(gpu, t, 4, 4, 2, Nq, Nk, 64, 100, 3, lens=lens, seed=Nq)
    _window_case(gpu, t, 4, 2, 2, Nq, Nk, 128, 0, 0, lens=lens, tokens_first=True, seed=Nq + 1)


@pytest.mark.parametrize("d", [64, 128])
def test_window_strided(gpu, d):
    """Token-major tensors, as a projection leaves them, and slices of a fused one."""
    _window_case(gpu, torch.bfloat16, 2, 6, 2, 200, 333, d, 70, 9, tokens_first=True)
    B, N, Hq, Hkv = 2, 150, 4, 2
    qkv = torch.randn(B, N, Hq + 2 * Hkv, d, device="cuda").half()
    q, k, v = (x.transpose(1, 2) for x in qkv.split([Hq, Hkv, Hkv], 2))
    wide = torch.full((B, N, Hq + 1, d), 7.0, device="cuda", dtype=torch.half)
    o = wide[:, :, :Hq].transpose(1, 2)
    assert gpu.flash_window_fwd(q, k, v, o, B, Hq, Hkv, N, N, d, LOG2E / math.sqrt(d), gpu.Dtype.F16,
                                window=40, sinks=2, q_strides=q.stride()[:3], k_strides=k.stride()[:3],
                                v_strides=v.stride()[:3], o_strides=o.stride()[:3]) == 0
    dense = torch.empty(B, Hq, N, d, device="cuda", dtype=torch.half)
    assert gpu.flash_window_fwd(q.contiguous(), k.contiguous(), v.contiguous(), dense, B, Hq, Hkv, N, N,
                                d, LOG2E / math.sqrt(d), gpu.Dtype.F16, window=40, sinks=2) == 0
    _done(gpu)
    assert torch.equal(o, dense)
    assert (wide[:, :, Hq] == 7.0).all()  # the columns beside O


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
def test_window_large_scores(gpu, t):
    """Scores over hundreds of log2 units: the running maximum moves within the row."""
    _window_case(gpu, t, 1, 4, 2, 400, 400, 128, 200, 5, q_scale=30.0, seed=9)


def test_window_masked_keys_do_not_matter(gpu):
    """NaN and infinite K of keys that a row does not see leave it as it is."""
    B, H, N, d = 1, 2, 300, 64
    q = torch.randn(B, H, N, d, device="cuda").half()
    k, v = torch.randn_like(q), torch.randn_like(q)
    outs = []
    for bad in (False, True):
        kk = k.clone()
        if bad:
            kk[0, :, 150], kk[0, :, 151] = float("nan"), float("inf")
        o = torch.empty_like(q)
        assert gpu.flash_window_fwd(q, kk, v, o, B, H, H, N, N, d, 0.18, gpu.Dtype.F16, window=30,
                                    sinks=2) == 0
        outs.append(o)
    _done(gpu)
    sees = torch.zeros(N, dtype=torch.bool)
    sees[150:181] = True
    assert torch.equal(outs[0][:, :, ~sees], outs[1][:, :, ~sees])
    assert not torch.isfinite(outs[1][:, :, 150:180]).any()


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
def test_window_long_sampled(gpu, t):
    """Long prompts; rows around tile borders, at the ends and in between."""
    rows = [0, 1, 127, 128, 255, 256, 1023, 1024, 1025, 2047, 2500, 4094, 4095]
    _window_case(gpu, t, 1, 8, 2, 4096, 4096, 128, 1000, 4, rows=rows, seed=1)
    _window_case(gpu, t, 1, 4, 4, 4001, 4500, 64, 513, 140, rows=[r for r in rows if r < 4001], seed=2)
    _window_case(gpu, t, 2, 3, 1, 4096, 4096, 128, 0, 0, rows=rows, seed=3)


def test_window_late_rows_of_a_long_sequence(gpu):
    """The last rows of 300000 tokens, through a window and in full."""
    _window_case(gpu, torch.float16, 1, 2, 1, 4, 300000, 64, 1000, 130, seed=5)
    _window_case(gpu, torch.bfloat16, 1, 1, 1, 2, 200001, 128, 0, 0, seed=6)


PAIR_SHAPES = [
    # B, Hq, Hkv, Nq, Nk, window, sinks, lens: more row tiles than SMs, so that a CTA takes two, of
    # the same rows, of adjacent ones, and none where a sequence has ended
    (10, 16, 16, 129, 129, 0, 0, None), (6, 14, 2, 257, 257, 100, 3, None), (12, 12, 4, 150, 290, 70, 130, None),
    (5, 32, 2, 130, 60, 16, 2, None), (40, 4, 1, 130, 130, 0, 0, [130, 1, 0, 64, 128, 129, 127, -1] * 5),
    (9, 15, 3, 300, 300, 33, 5, [300, 0, 0, 0, 1, 257, 256, 129, 299]),
    (8, 8, 8, 384, 384, 128, 256, [0, 0, 0, 0, 0, 0, 0, 383]),
    (20, 8, 2, 200, 333, 90, 4, [333, 134, 133, 200] * 5), (3, 64, 64, 140, 140, 1, 0, [140, 128, 5]),
]


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("shape", PAIR_SHAPES)
def test_window_pairs_of_tiles(gpu, shape, d, t):
    B, Hq, Hkv, Nq, Nk, window, sinks, lens = shape
    assert (Nq + 127) // 128 * Hq * B > 148
    rows = sorted({0, 1, 63, 100, 127, 128, 129, 255, 256, Nq - 2, Nq - 1} & set(range(Nq)))
    _window_case(gpu, t, B, Hq, Hkv, Nq, Nk, d, window, sinks, lens=lens, rows=rows,
                 tokens_first=d == 64, seed=Nq + Hq)


@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 200), (520, 0)])
@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("d", [64, 128])
def test_window_halves_of_keys(gpu, d, t, window, sinks):
    """Few row tiles, whose keys are shared out: one to nine key tiles, odd and even, sequences that
    end within a tile and on its border, scores that make one half's share vanish."""
    B, Hq, N = 8, 2, 1100
    assert (N + 127) // 128 * Hq * B <= 148
    rows = [0, 1, 127, 128, 300, 511, 512, 639, 640, 800, 896, 1023, 1024, 1098, 1099]
    _window_case(gpu, t, B, Hq, 1, N, N, d, window, sinks, lens=[1100, 1025, 1024, 897, 640, 385, 129, 3],
                 rows=rows, seed=d + window)
    _window_case(gpu, t, 4, Hq, 2, N, N + 333, d, window, sinks, q_scale=20.0, rows=rows,
                 tokens_first=True, seed=d + window + 1)


def test_window_matches_flash_fwd(gpu):
    """Without a window it is the causal vc_flash_fwd."""
    B, H, N, d = 2, 3, 500, 128
    q, k, v = (torch.randn(B, H, N, d, device="cuda").to(torch.bfloat16) for _ in range(3))
    a, b = torch.empty_like(q), torch.empty_like(q)
    s = LOG2E / math.sqrt(d)
    assert gpu.flash_fwd(q, k, v, a, B * H, N, d, s, True, gpu.Dtype.BF16) == 0
    assert gpu.flash_window_fwd(q, k, v, b, B, H, H, N, N, d, s, gpu.Dtype.BF16) == 0
    _done(gpu)
    vmax = float(v.abs().max())
    assert (a.double() - b.double()).abs().max() <= 2 * (2 * 2.0 ** -8 * vmax + 2.0 ** -8 * vmax)


# ------------------------------------------------------------------ cache
class Cache:
    """A layer's cache in torch tensors, every code NaN and every scale 1 at first."""

    def __init__(self, gpu, pages, H, P, d):
        self.k, self.v = (torch.full((pages, H, P, d), 0x7F, dtype=torch.uint8, device="cuda")
                          for _ in range(2))
        self.ks, self.vs = (torch.ones(pages, H, device="cuda") for _ in range(2))
        self.handle = gpu.kv8_cache(self.k, self.v, self.ks, self.vs, pages, H, P, d)

    def host(self):
        return [x.cpu().numpy() for x in (self.k, self.ks, self.v, self.vs)]


def _table(lens, P, pages, rng, width=None):
    need = [-(-n // P) for n in lens]
    ids = rng.permutation(pages)[:sum(need)]
    table = np.full((len(lens), max(width or 1, max(need), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table


def _ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("P", [16, 32, 64, 128])
def test_append_exact(gpu, P, d, t):
    """Ragged tokens behind ragged prefixes, twice, with growing magnitudes (scales grow and the
    earlier tokens move), zeros, subnormals, infinities and NaN."""
    rng = np.random.default_rng(P + d)
    H, B = 3, 6
    start = [0, 1, P - 1, P, 2 * P + 5, 0]
    count = [1, 3 * P + 2, 2, 0, P, 2 * P]
    total = [a + b for a, b in zip(start, count)]
    later = [5, 1, P, 1, 0, 3]
    pages = sum(-(-(n + m) // P) for n, m in zip(total, later)) + 3
    table = _table([n + m for n, m in zip(total, later)], P, pages, rng)
    c = Cache(gpu, pages, H, P, d)
    want = c.host()
    # The prefix: what an earlier append left.
    steps = [(start, [0] * B, 1.0), (count, start, 4.0), (later, total, 100.0)]
    for new, at, size in steps:
        T = sum(new)
        x = [(torch.randn(max(T, 1), H, d, device="cuda") * size *
              torch.exp2(torch.randint(-6, 3, (max(T, 1), 1, 1), device="cuda").float())).to(t)
             for _ in range(2)]
        if size == 4.0:
            x[0][0, 0] = 0.0
            x[0][1, 1, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 1e-7]).to(t)
            x[1][3:6] = 0.0
        lens_out = _ints([-1] * B)
        cu = np.concatenate([[0], np.cumsum(new)])
        assert gpu.kv8_append(c.handle, x[0], x[1], T, _ints(table), table.shape[1], _ints(at), B,
                              max(max(new), 1), _dt(gpu, t), cu=_ints(cu), lens_out=lens_out) == 0
        _done(gpu)
        assert lens_out.tolist() == [a + n for a, n in zip(at, new)]
        plain.append(want[0], want[1], _f64(x[0]), table, at, new, P)
        plain.append(want[2], want[3], _f64(x[1]), table, at, new, P)
        for g, w, name in zip(c.host(), want, ("k", "k_scale", "v", "v_scale")):
            assert np.array_equal(g, w), (name, size, np.argwhere(g != w)[:4])


def test_append_nothing(gpu):
    """A step in which no sequence has new tokens: empty tensors, the lengths as they were."""
    rng = np.random.default_rng(5)
    c, table = _fill(gpu, [30, 7], 2, 16, 64, rng)
    before = c.host()
    for t, cu in ((torch.half, _ints([0, 0, 0])), (torch.bfloat16, None)):
        none = torch.empty(0, 2, 64, device="cuda", dtype=t)
        assert none.data_ptr() == 0
        lens = _ints([-1, -1])
        assert gpu.kv8_append(c.handle, none, none, 0, _ints(table), table.shape[1], _ints([30, 7]), 2,
                              4 if cu is not None else 0, _dt(gpu, t), cu=cu, lens_out=lens) == 0
        _done(gpu)
        assert lens.tolist() == [30, 7]
    for g, w in zip(c.host(), before):
        assert np.array_equal(g, w)
    assert gpu.kv8_append(c.handle, None, None, 1, _ints(table), table.shape[1], _ints([30, 7]), 1, 1,
                          gpu.Dtype.F16) == gpu.VCError.InvalidValue


def test_append_step_strided(gpu):
    """One token each, out of a fused projection, without offsets; extreme magnitudes keep their
    scales within range."""
    H, d, P, B = 2, 64, 32, 5
    rng = np.random.default_rng(3)
    start = [0, 31, 32, 7, 64]
    table = _table([n + 1 for n in start], P, 12, rng, width=4)
    c = Cache(gpu, 12, H, P, d)
    c.k.fill_(0x38)  # 1.0
    c.ks.fill_(2.0 ** -3)
    want = c.host()
    fused = torch.randn(B, 6 * d, device="cuda").to(torch.bfloat16)
    fused[1, :d] *= 1e30
    fused[2, :d] = 3e38
    fused[3, :2 * d] *= 1e-35
    fused[4, 3 * d] = 2.0 ** -133  # a bf16 subnormal
    assert gpu.kv8_append(c.handle, fused, fused[:, 2 * d:], B, _ints(table), 4, _ints(start), B, 1,
                          gpu.Dtype.BF16, k_stride=6 * d, v_stride=6 * d) == 0
    _done(gpu)
    x = _f64(fused).reshape(B, 6, d)
    plain.append(want[0], want[1], x[:, :2], table, start, [1] * B, P)
    plain.append(want[2], want[3], x[:, 2:4], table, start, [1] * B, P)
    for g, w in zip(c.host(), want):
        assert np.array_equal(g, w)


def test_append_scales_not_powers_of_two(gpu):
    """A page whose scale another quantiser chose keeps it while it is the larger one."""
    H, d, P = 1, 64, 16
    c = Cache(gpu, 1, H, P, d)
    c.k.fill_(0x40)  # 2.0
    c.v.fill_(0x41)
    c.ks.fill_(0.3)
    c.vs.fill_(1e-3)
    want = c.host()
    x = torch.randn(2, H, d, device="cuda").half()
    assert gpu.kv8_append(c.handle, x, x, 2, _ints([[0]]), 1, _ints([4]), 1, 2, gpu.Dtype.F16) == 0
    _done(gpu)
    got = c.host()
    plain.append(want[0], want[1], _f64(x), [[0]], [4], [2], P)
    plain.append(want[2], want[3], _f64(x), [[0]], [4], [2], P)
    assert got[1][0, 0] == np.float32(0.3) and np.array_equal(got[1], want[1]) and np.array_equal(got[3], want[3])
    # The fp32 quotient x / 0.3 may fall on the other side of a code's border than the float64 one:
    # by one code at most, and hardly ever.
    off = np.abs(got[0].astype(int) - want[0].astype(int))
    assert off.max() <= 1 and (off > 0).mean() < 0.01
    assert np.array_equal(got[2], want[2])


def test_append_reports_what_does_not_fit(gpu):
    """Page numbers, offsets and positions out of range are left out and reported; the rest is
    written."""
    H, d, P, B = 1, 64, 16, 6
    c = Cache(gpu, 8, H, P, d)
    x = torch.ones(8, H, d, device="cuda").half()
    table = np.array([[0, 1], [8, 2], [-1, 3], [4, 5], [6, 7], [2, 2]], np.int32)
    start = [0, 0, 0, -1, 31, 0]
    cu = [0, 1, 2, 3, 4, 7, 9]  # the fifth runs past its row's pages, the sixth past the tokens
    lens = _ints([-7] * B)
    assert gpu.kv8_append(c.handle, x, x, 8, _ints(table), 2, _ints(start), B, 3, gpu.Dtype.F16,
                          cu=_ints(cu), lens_out=lens) == 0
    torch.cuda.synchronize()
    assert gpu.kernel_error(True) == 4
    code = int(plain.to_e4m3(np.array([256.0]))[0])  # 1 / 2^-8
    k = c.k.cpu().numpy()
    # Slot 31's page holds earlier tokens at scale 1, which is the larger: 1.0 is code 0x38 there.
    assert (k[0, 0, 0] == code).all() and (k[7, 0, 15] == 0x38).all()
    k[0, 0, 0] = k[7, 0, 15] = 0x7F
    assert (k == 0x7F).all()
    assert lens.tolist() == [1, 1, 1, 0, 32, 0]


# ------------------------------------------------------------------ single tokens
def _fill(gpu, lens, H, P, d, rng, spare=2, width=None):
    pages = sum(-(-n // P) for n in lens) + spare
    table = _table(lens, P, pages, rng, width)
    c = Cache(gpu, pages, H, P, d)
    for codes, scales in ((c.k, c.ks), (c.v, c.vs)):
        x = plain.to_e4m3(rng.standard_normal((pages, H, P, d)) * 100)
        scales.copy_(torch.from_numpy((rng.uniform(0.5, 2, (pages, H)) * 2.0 ** -7).astype(np.float32)))
        for b, n in enumerate(lens):  # slots behind the last token: NaN
            if n % P:
                x[table[b, n // P], :, n % P:] = 0x7F
        codes.copy_(torch.from_numpy(x))
    return c, table


def _attn_case(gpu, c, table, lens, Hq, t, window, sinks, q_scale=1.0, check=True, ws=None, seed=0):
    B, H, P = len(lens), c.k.shape[1], c.k.shape[2]
    d = c.k.shape[3]
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn(B, Hq, d, device="cuda", generator=g) * q_scale).to(t)
    o = torch.full_like(q, 7.0)
    scale = LOG2E / math.sqrt(d)
    if ws is None:
        err, n = gpu.kv8_attn_workspace(c.handle, B, Hq)
        assert err == 0
        ws = torch.zeros(max(n, 256), dtype=torch.uint8, device="cuda")
    assert gpu.kv8_attn(c.handle, q, o, _ints(table), table.shape[1], _ints(lens), B, Hq, scale,
                        _dt(gpu, t), ws, ws.numel(), window=window, sinks=sinks) == 0
    _done(gpu)
    if not check:
        return q, o
    k, ks, v, vs = c.host()
    want = plain.cache_attn(_f64(q), k, ks, v, vs, table, lens, window, sinks, scale, P)
    kmax = 448 * ks.max()
    vmax = 448 * float(vs.max())
    smax = np.abs(_f64(q)).sum(-1).max() * kmax * scale
    tol = _tol(want, t, 2.0 ** -11, vmax, smax, d, max(lens))
    assert (np.abs(_f64(o) - want) <= tol).all(), (np.abs(_f64(o) - want).max(), tol.min())
    return q, o


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("P,H,G", [(16, 2, 1), (32, 1, 8), (64, 3, 3), (128, 1, 16), (16, 1, 7),
                                   (64, 1, 20), (32, 2, 9), (16, 1, 40)])
def test_attn_shapes(gpu, P, H, G, d, t):
    rng = np.random.default_rng(P * G + d)
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 130, 500, 1000]
    c, table = _fill(gpu, lens, H, P, d, rng, width=70)
    for window, sinks in ((0, 0), (1, 0), (64, 4), (100, 17), (999, 1), (200, 300)):
        _attn_case(gpu, c, table, lens, H * G, t, window, sinks, seed=window)


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
def test_attn_large_scores(gpu, t):
    rng = np.random.default_rng(5)
    lens = [700, 33, 1]
    c, table = _fill(gpu, lens, 2, 16, 128, rng)
    _attn_case(gpu, c, table, lens, 8, t, 0, 0, q_scale=40.0)
    _attn_case(gpu, c, table, lens, 8, t, 300, 2, q_scale=1e-4)


def test_attn_bf16_queries_beyond_fp16(gpu):
    """bf16 queries reach past fp16's range; the scales of K bring the scores back."""
    rng = np.random.default_rng(6)
    lens = [300, 45]
    c, table = _fill(gpu, lens, 1, 32, 64, rng)
    c.ks.mul_(2.0 ** -60)
    _attn_case(gpu, c, table, lens, 4, torch.bfloat16, 0, 0, q_scale=2.0 ** 60)
    c.ks.mul_(2.0 ** 100)
    _attn_case(gpu, c, table, lens, 4, torch.bfloat16, 0, 0, q_scale=2.0 ** -40)


def test_attn_uneven_value_scales(gpu):
    """Value scales many powers of two apart, zero among them: a page with a small scale keeps its
    precision where it holds the weight."""
    rng = np.random.default_rng(7)
    lens = [256]
    c, table = _fill(gpu, lens, 1, 16, 64, rng)
    scale = LOG2E / 8
    for exps in ([-20, 0], [20, -60], [0, None], [100, -100]):
        for i, e in enumerate(exps):
            c.vs[table[0, i::2].tolist()] = 0.0 if e is None else 2.0 ** e
        for heavy in (0, 1):  # the keys of these pages get all the weight
            q = torch.zeros(1, 4, 64, device="cuda").half()
            q[0, :, 0] = 8.0
            codes = c.k.clone()
            c.k[:, :, :, 0] = int(plain.to_e4m3(np.array([-448.0]))[0])
            c.k[table[0, heavy::2].tolist(), :, :, 0] = int(plain.to_e4m3(np.array([448.0]))[0])
            c.ks.fill_(1.0)
            o = torch.full((1, 4, 64), 7.0, device="cuda").to(torch.bfloat16)
            qb = q.to(torch.bfloat16)
            err, n = gpu.kv8_attn_workspace(c.handle, 1, 4)
            ws = torch.zeros(max(n, 256), dtype=torch.uint8, device="cuda")
            assert gpu.kv8_attn(c.handle, qb, o, _ints(table), table.shape[1], _ints(lens), 1, 4, scale,
                                gpu.Dtype.BF16, ws, ws.numel()) == 0
            _done(gpu)
            k, ks, v, vs = c.host()
            want = plain.cache_attn(_f64(qb), k, ks, v, vs, table, lens, 0, 0, scale, 16)
            big = 448 * (0.0 if exps[heavy] is None else 2.0 ** exps[heavy])
            # The heavy pages' weights are 2^-2600 above the others': only they count.
            assert (np.abs(_f64(o) - want) <= 2.0 ** -8 * np.abs(want) + big * 2.0 ** -10).all()
            c.k.copy_(codes)


def test_attn_nan_outside_the_window(gpu):
    """NaN codes that the mask hides, inside visible pages too, do not reach the output."""
    rng = np.random.default_rng(8)
    lens = [200, 37, 500]
    c, table = _fill(gpu, lens, 2, 64, 64, rng)
    for b, n in enumerate(lens):
        j = np.arange(4, n - 30)
        for x in (c.k, c.v):
            x[table[b, j // 64].tolist(), :, j % 64] = 0x7F
    _attn_case(gpu, c, table, lens, 4, torch.float16, 30, 4)


def test_attn_long_splits(gpu):
    """A long sequence beside short ones: the work is split along the tokens."""
    rng = np.random.default_rng(9)
    lens = [20011, 3, 1500, 0]
    c, table = _fill(gpu, lens, 1, 128, 64, rng)
    for t in TYPES.values():
        _attn_case(gpu, c, table, lens, 8, t, 0, 0)
        _attn_case(gpu, c, table, lens, 8, t, 9000, 128)


def test_attn_same_answer_each_time(gpu):
    rng = np.random.default_rng(10)
    lens = [5000, 17, 3333, 900]
    c, table = _fill(gpu, lens, 2, 16, 128, rng)
    err, n = gpu.kv8_attn_workspace(c.handle, 4, 16)
    ws = torch.zeros(max(n, 256), dtype=torch.uint8, device="cuda")
    outs = [_attn_case(gpu, c, table, lens, 16, torch.float16, 0, 0, check=False, ws=ws)[1]
            for _ in range(5)]
    assert all(torch.equal(outs[0], o) for o in outs)


def test_attn_workspace_serves_other_shapes(gpu):
    """One workspace, calls of different shapes in turn."""
    rng = np.random.default_rng(11)
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    for H, G, d, lens in ((2, 4, 128, [3000, 5]), (1, 16, 64, [100] * 40), (4, 2, 64, [7000]),
                          (2, 4, 128, [3000, 5])):
        c, table = _fill(gpu, lens, H, 32, d, rng)
        _attn_case(gpu, c, table, lens, H * G, torch.float16, 0, 0, ws=ws)


def test_attn_strided_rows(gpu):
    rng = np.random.default_rng(12)
    lens, Hq, d = [90, 300, 5], 4, 64
    c, table = _fill(gpu, lens, 2, 16, d, rng)
    fused = torch.randn(3, Hq * d + 256, device="cuda").half()
    out = torch.full((3, Hq * d + 64), 7.0, device="cuda").half()
    err, n = gpu.kv8_attn_workspace(c.handle, 3, Hq)
    ws = torch.zeros(max(n, 256), dtype=torch.uint8, device="cuda")
    dense = torch.empty(3, Hq, d, device="cuda").half()
    args = (_ints(table), table.shape[1], _ints(lens), 3, Hq, 0.18, gpu.Dtype.F16, ws, ws.numel())
    assert gpu.kv8_attn(c.handle, fused, out, *args, q_stride=fused.stride(0), o_stride=out.stride(0)) == 0
    assert gpu.kv8_attn(c.handle, fused[:, :Hq * d].contiguous(), dense, *args) == 0
    _done(gpu)
    assert torch.equal(out[:, :Hq * d].reshape(3, Hq, d), dense)
    assert (out[:, Hq * d:] == 7.0).all()


@pytest.mark.parametrize("B", [33, 300, 1500])
def test_attn_many_short_sequences(gpu, B):
    """More sequences than a warp has lanes, empty ones among them, in any order."""
    rng = np.random.default_rng(B)
    lens = rng.integers(0, 40, B).tolist()
    lens[0], lens[B // 2], lens[-1] = 0, 700, 0
    c, table = _fill(gpu, lens, 2, 16, 64, rng)
    _attn_case(gpu, c, table, lens, 6, torch.float16, 0, 0)
    _attn_case(gpu, c, table, lens, 6, torch.bfloat16, 17, 2)
    zeros = [0] * B
    q, o = _attn_case(gpu, c, table, zeros, 6, torch.float16, 0, 0, check=False)
    assert (o == 0).all()


def test_attn_very_long(gpu):
    """300000 tokens of one sequence; offsets, splits and joins of the longest kind."""
    rng = np.random.default_rng(31)
    lens = [300001]
    c, table = _fill(gpu, lens, 1, 128, 64, rng)
    _attn_case(gpu, c, table, lens, 2, torch.float16, 0, 0)
    _attn_case(gpu, c, table, lens, 16, torch.bfloat16, 200000, 4)


def test_attn_nan_query_stays_in_its_row(gpu):
    rng = np.random.default_rng(32)
    lens = [5000, 40]
    c, table = _fill(gpu, lens, 1, 32, 128, rng)
    q, clean = _attn_case(gpu, c, table, lens, 8, torch.float16, 0, 0)
    q2 = q.clone()
    q2[0, 3, 7] = float("nan")
    o = torch.empty_like(q2)
    err, n = gpu.kv8_attn_workspace(c.handle, 2, 8)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    assert gpu.kv8_attn(c.handle, q2, o, _ints(table), table.shape[1], _ints(lens), 2, 8,
                        LOG2E / math.sqrt(128), gpu.Dtype.F16, ws, n) == 0
    _done(gpu)
    assert torch.isnan(o[0, 3]).all()
    keep = torch.ones(2, 8, dtype=torch.bool)
    keep[0, 3] = False
    # The running maximum may move at other keys: fp32 roundings, then one of the output.
    assert (o[keep].double() - clean[keep].double()).abs().max() <= 2.0 ** -10 * clean.abs().max()


def test_layers_in_one_allocation(gpu):
    """Append and attention on two layers whose pages alternate in memory, K and V and the scales
    of both in one buffer each."""
    H, P, d, pages, Hq = 2, 32, 64, 9, 6
    one = H * P * d
    codes = torch.full((pages, 2, 2, one + 64), 0x7F, dtype=torch.uint8, device="cuda")
    scales = torch.full((pages, 2, 2, H + 3), 5.0, device="cuda")
    want = [codes.clone(), scales.clone()]
    caches = [gpu.kv8_cache(codes[0, i, 0], codes[0, i, 1], scales[0, i, 0], scales[0, i, 1], pages, H, P, d,
                            page_stride=4 * (one + 64), scale_stride=4 * (H + 3)) for i in range(2)]
    rng = np.random.default_rng(3)
    lens = [70, 33]
    table = _table(lens, P, pages, rng)
    ws = torch.zeros(gpu.kv8_attn_workspace(caches[0], 2, Hq)[1], dtype=torch.uint8, device="cuda")
    for i in range(2):
        x = [torch.randn(103, H, d, device="cuda").half() for _ in range(2)]
        q, o = torch.randn(2, Hq, d, device="cuda").half(), torch.empty(2, Hq, d, device="cuda").half()
        assert gpu.kv8_append(caches[i], x[0], x[1], 103, _ints(table), 3, _ints([0, 0]), 2, 70, gpu.Dtype.F16,
                              cu=_ints([0, 70, 103])) == 0
        assert gpu.kv8_attn(caches[i], q, o, _ints(table), 3, _ints(lens), 2, Hq, 0.18, gpu.Dtype.F16, ws,
                            ws.numel()) == 0
        _done(gpu)
        host = []
        for kv in range(2):
            ck = np.full((pages, H, P, d), 0x7F, np.uint8)
            sk = np.full((pages, H), 5.0, np.float32)
            plain.append(ck, sk, _f64(x[kv]), table, [0, 0], lens, P)
            want[0][:, i, kv, :one] = torch.from_numpy(ck.reshape(pages, one)).cuda()
            want[1][:, i, kv, :H] = torch.from_numpy(sk).cuda()
            host += [ck, sk]
        assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
        exp = plain.cache_attn(_f64(q), *host, table, lens, 0, 0, 0.18, P)
        assert np.abs(_f64(o) - exp).max() <= 2.0 ** -11 * 3 * 6 + 1e-4


def test_attn_reports_bad_pages_and_lengths(gpu):
    """A page number out of range hides its tokens; a length past the table is cut; both are
    reported."""
    rng = np.random.default_rng(13)
    lens = [100, 64]
    c, table = _fill(gpu, lens, 1, 16, 64, rng, width=7)
    for bad in (-1, table.max() + 100, 2 ** 31 - 1, -2 ** 31):
        t2 = table.copy()
        t2[0, 2] = bad
        q = torch.randn(2, 4, 64, device="cuda").half()
        o = torch.empty_like(q)
        err, n = gpu.kv8_attn_workspace(c.handle, 2, 4)
        ws = torch.zeros(max(n, 256), dtype=torch.uint8, device="cuda")
        args = (2, 4, 0.18, gpu.Dtype.F16, ws, ws.numel())
        assert gpu.kv8_attn(c.handle, q, o, _ints(t2), 7, _ints(lens), *args) == 0
        torch.cuda.synchronize()
        assert gpu.kernel_error(True) == 4
        k, ks, v, vs = c.host()
        keep = np.concatenate([np.arange(32), np.arange(48, 100)])
        kk = plain.E4M3[k[table[0, keep // 16], 0, keep % 16]] * ks[table[0, keep // 16], 0][:, None]
        vv = plain.E4M3[v[table[0, keep // 16], 0, keep % 16]] * vs[table[0, keep // 16], 0][:, None]
        want = np.stack([plain._row(x, kk, vv, 0.18) for x in _f64(q)[0]])
        assert np.abs(_f64(o)[0] - want).max() <= 0.02
    full = _ints(table[:1, :6].copy())
    outs = []
    for n_tok in (96, 1000, 2 ** 31 - 1):
        o = torch.empty(1, 4, 64, device="cuda").half()
        assert gpu.kv8_attn(c.handle, q[:1], o, full, 6, _ints([n_tok]), 1, 4, 0.18, gpu.Dtype.F16, ws,
                            ws.numel()) == 0
        torch.cuda.synchronize()
        assert gpu.kernel_error(True) == (0 if n_tok == 96 else 4)
        outs.append(o)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    o.fill_(7.0)
    assert gpu.kv8_attn(c.handle, q[:1], o, full, 6, _ints([-5]), 1, 4, 0.18, gpu.Dtype.F16, ws,
                        ws.numel()) == 0
    torch.cuda.synchronize()
    assert gpu.kernel_error(True) == 4 and (o == 0).all()


def test_cache_beyond_32_bit_offsets(gpu):
    """Pages gigabytes apart (page strides of a cache that interleaves many layers)."""
    H, P, d, stride = 1, 16, 64, (1 << 31) + 4096
    big = torch.empty(3 * stride, dtype=torch.uint8, device="cuda")
    ks, vs = torch.ones(3, H, device="cuda"), torch.ones(3, H, device="cuda")
    half = stride // 2 & ~15
    c = gpu.kv8_cache(big, big[half:], ks, vs, 3, H, P, d, page_stride=stride)
    table, n = _ints([[2, 1]]), 20
    x = [torch.randn(n, H, d, device="cuda").half() for _ in range(2)]
    assert gpu.kv8_append(c, x[0], x[1], n, table, 2, _ints([0]), 1, n, gpu.Dtype.F16) == 0
    assert gpu.kv8_copy_pages(gpu.kv8_layers([c]), _ints([2]), _ints([0]), 1) == 0
    q, o = torch.randn(1, 2, d, device="cuda").half(), [torch.empty(1, 2, d, device="cuda").half() for _ in range(2)]
    err, need = gpu.kv8_attn_workspace(c, 1, 2)
    ws = torch.zeros(max(need, 256), dtype=torch.uint8, device="cuda")
    for out, tab in zip(o, (table, _ints([[0, 1]]))):
        assert gpu.kv8_attn(c, q, out, tab, 2, _ints([n]), 1, 2, 0.18, gpu.Dtype.F16, ws, ws.numel()) == 0
    _done(gpu)
    assert torch.equal(o[0], o[1])
    codes = []
    for base, s in ((0, ks), (half, vs)):
        rows = [big[base + p * stride:base + p * stride + P * d].view(P, d).cpu().numpy() for p in (2, 1)]
        codes.append(np.concatenate([plain.E4M3[r] * float(s[p, 0]) for r, p in zip(rows, (2, 1))])[:n])
    want = np.stack([plain._row(r, codes[0], codes[1], 0.18) for r in _f64(q)[0]])
    assert np.abs(_f64(o[0])[0] - want).max() <= 0.01


# ------------------------------------------------------------------ pages
@pytest.mark.parametrize("layers,H,P,d", [(1, 1, 16, 64), (3, 2, 16, 128), (2, 8, 128, 128), (70, 1, 16, 64)])
def test_copy_pages(gpu, layers, H, P, d):
    """Layers in one allocation (wide page strides), more than one launch takes."""
    pages = 9
    one = H * P * d
    codes = torch.randint(0, 256, (pages, layers, 2, one), dtype=torch.uint8, device="cuda")
    scales = torch.rand(pages, layers, 2, H, device="cuda")
    cs = gpu.kv8_layers([gpu.kv8_cache(codes[0, i, 0], codes[0, i, 1], scales[0, i, 0], scales[0, i, 1],
                                       pages, H, P, d, page_stride=layers * 2 * one,
                                       scale_stride=layers * 2 * H) for i in range(layers)])
    want = [codes.clone(), scales.clone()]
    src, dst = [8, 3, 3, 5], [0, 2, 7, 5]
    for a, b in zip(src, dst):
        for w in want:
            w[b] = w[a]
    assert gpu.kv8_copy_pages(cs, _ints(src), _ints(dst), 4) == 0
    assert gpu.kv8_copy_pages(cs, _ints(src), _ints(dst), 0) == 0
    _done(gpu)
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    assert gpu.kv8_copy_pages(cs, _ints([9, 1, -1]), _ints([1, 4, 6]), 3) == 0
    torch.cuda.synchronize()
    assert gpu.kernel_error(True) == 4
    want[0][4], want[1][4] = want[0][1], want[1][1]
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])


# ------------------------------------------------------------------ refusals on a GPU
def test_host_pointers_are_refused(gpu):
    rng = np.random.default_rng(1)
    c, table = _fill(gpu, [30], 1, 16, 64, rng)
    host = np.zeros(1 << 14, np.uint8)
    at = (host.ctypes.data + 255) & ~255
    q = torch.zeros(1, 4, 64, device="cuda").half()
    ws = torch.zeros(1 << 24, dtype=torch.uint8, device="cuda")
    tail = (_ints(table), table.shape[1], _ints([30]), 1, 4, 0.1, gpu.Dtype.F16, ws, ws.numel())
    assert gpu.kv8_attn(c.handle, at, q, *tail) == gpu.VCError.InvalidValue
    assert gpu.kv8_attn(c.handle, q, at, *tail) == gpu.VCError.InvalidValue
    bad = gpu.kv8_cache(at, c.v, c.ks, c.vs, 2, 1, 16, 64)
    assert gpu.kv8_attn(bad, q, q, *tail) == gpu.VCError.InvalidValue
    assert gpu.kv8_append(bad, q, q, 1, _ints([[0]]), 1, _ints([0]), 1, 1, gpu.Dtype.F16) \
        == gpu.VCError.InvalidValue
    assert gpu.kv8_copy_pages(gpu.kv8_layers([c.handle]), at, at, 1) == gpu.VCError.InvalidValue
    assert gpu.flash_window_fwd(q, q, q, at, 1, 4, 4, 1, 1, 64, 0.1, gpu.Dtype.F16) \
        == gpu.VCError.InvalidValue
    _done(gpu)


def test_pinned_and_managed_memory_are_refused(gpu):
    rng = np.random.default_rng(2)
    c, table = _fill(gpu, [30], 1, 16, 64, rng)
    q = torch.zeros(1, 4, 64, device="cuda").half()
    ws = torch.zeros(1 << 24, dtype=torch.uint8, device="cuda")
    pinned = torch.zeros(1 << 14, dtype=torch.uint8).pin_memory()
    err, managed = gpu.vcMallocManaged(1 << 14)
    assert err == 0
    try:
        for other in (pinned, managed):
            tail = (_ints(table), table.shape[1], _ints([30]), 1, 4, 0.1, gpu.Dtype.F16, ws, ws.numel())
            assert gpu.kv8_attn(c.handle, other, q, *tail) == gpu.VCError.InvalidValue
            bad = gpu.kv8_cache(other, c.v, c.ks, c.vs, 2, 1, 16, 64)
            assert gpu.kv8_attn(bad, q, q, *tail) == gpu.VCError.InvalidValue
            assert gpu.kv8_append(c.handle, q, q, 1, other, 1, _ints([0]), 1, 1, gpu.Dtype.F16) \
                == gpu.VCError.InvalidValue
            assert gpu.kv8_copy_pages(gpu.kv8_layers([bad]), _ints([0]), _ints([1]), 1) \
                == gpu.VCError.InvalidValue
            assert gpu.flash_window_fwd(q, other, q, q, 1, 4, 4, 1, 1, 64, 0.1, gpu.Dtype.F16) \
                == gpu.VCError.InvalidValue
    finally:
        assert gpu.vcFree(managed) == 0
    _done(gpu)


def test_buffers_too_small_are_refused(gpu, dev):
    small = dev.alloc(4096)
    assert gpu.flash_window_fwd(small.ptr, small.ptr, small.ptr, small.ptr, 1, 4, 4, 64, 64, 64, 0.1,
                                gpu.Dtype.F16) == gpu.VCError.InvalidValue
    c = gpu.kv8_cache(small.ptr, small.ptr, small.ptr, small.ptr, 8, 1, 16, 64)
    big = dev.alloc(1 << 20)
    assert gpu.kv8_append(c, big.ptr, big.ptr, 1, big.ptr, 1, big.ptr, 1, 1, gpu.Dtype.F16) \
        == gpu.VCError.InvalidValue
    ok = gpu.kv8_cache(big.ptr, big.ptr, big.ptr, big.ptr, 8, 1, 16, 64)
    assert gpu.kv8_attn(ok, big.ptr, big.ptr, big.ptr, 1, big.ptr, 1, 1, 0.1, gpu.Dtype.F16, small.ptr,
                        1 << 20) == gpu.VCError.InvalidValue
    assert gpu.kv8_attn(ok, big.ptr, big.ptr, big.ptr, 1 << 19, big.ptr, 1, 1, 0.1, gpu.Dtype.F16,
                        big.ptr, 1 << 20) == gpu.VCError.InvalidValue


# ------------------------------------------------------------------ together
def test_serving_run(gpu):
    """Prompts through the window, into the cache, a fork that diverges, a freed sequence, a
    compaction, and single tokens at each step, for two layers with pages from one pool; the
    attention is compared with float64 over the codes that the cache holds, the codes with those of
    a plain append."""
    L, H, G, d, P, pages, window, sinks = 2, 2, 4, 64, 16, 40, 50, 3
    Hq, t, s2 = H * G, torch.float16, LOG2E / 8
    layers = [Cache(gpu, pages, H, P, d) for _ in range(L)]
    caches = gpu.kv8_layers([c.handle for c in layers])
    want = [c.host() for c in layers]
    err, pool = gpu.kv8_pool_create(pages, P)
    g = torch.Generator(device="cuda").manual_seed(4)
    ws = torch.zeros(gpu.kv8_attn_workspace(caches[0], 8, Hq)[1] or 256, dtype=torch.uint8, device="cuda")

    def copy(pairs):
        if not pairs:
            return
        src, dst = zip(*pairs)
        assert gpu.kv8_copy_pages(caches, _ints(src), _ints(dst), len(pairs)) == 0
        for w in want:
            for x in w:
                x[list(dst)] = x[list(src)]

    def table(seqs):
        out = np.full((len(seqs), 10), -1, np.int32)
        counts = [gpu.kv8_pool_pages(pool, s, out[i:i + 1], 10) for i, s in enumerate(seqs)]
        assert all(e == 0 for e, _, _ in counts)
        return out, [n for _, _, n in counts]

    def add(seqs, new):
        """Room for the new tokens, their K and V, and the appends."""
        before = table(seqs)[1]
        pairs = []
        for s, n in zip(seqs, new):
            err, pair = gpu.kv8_pool_extend(pool, s, n)
            assert err == 0
            pairs += [pair] if pair else []
        copy(pairs)
        tab, after = table(seqs)
        lens = _ints([0] * len(seqs))
        made = []
        for i in range(L):
            x = [torch.randn(sum(new), H, d, device="cuda", generator=g).to(t) for _ in range(2)]
            assert gpu.kv8_append(caches[i], x[0], x[1], sum(new), _ints(tab), 10, _ints(before), len(seqs),
                                  max(new), gpu.Dtype.F16, cu=_ints(np.concatenate([[0], np.cumsum(new)])),
                                  lens_out=lens) == 0
            plain.append(want[i][0], want[i][1], _f64(x[0]), tab, before, new, P)
            plain.append(want[i][2], want[i][3], _f64(x[1]), tab, before, new, P)
            made.append(x)
        assert lens.tolist() == after
        return tab, after, lens, made

    def step(seqs):
        tab, after, lens, _ = add(seqs, [1] * len(seqs))
        for i in range(L):
            q = torch.randn(len(seqs), Hq, d, device="cuda", generator=g).to(t)
            o = torch.empty_like(q)
            assert gpu.kv8_attn(caches[i], q, o, _ints(tab), 10, lens, len(seqs), Hq, s2, gpu.Dtype.F16, ws,
                                ws.numel(), window=window, sinks=sinks) == 0
            _done(gpu)
            for a, b in zip(layers[i].host(), want[i]):
                assert np.array_equal(a, b)
            k, ks, v, vs = want[i]
            exp = plain.cache_attn(_f64(q), k, ks, v, vs, tab, after, window, sinks, s2, P)
            assert np.abs(_f64(o) - exp).max() <= 2.0 ** -11 * 3 * 5 + 1e-4
        return after

    seqs = [gpu.kv8_pool_new(pool)[1] for _ in range(3)]
    new = [70, 5, 33]
    _, _, lens, made = add(seqs, new)
    for k, v in made:  # the prompts themselves, as a padded batch
        N = max(new)
        kk, vv = (torch.full((3, N, H, d), float("nan"), device="cuda", dtype=t) for _ in range(2))
        at = 0
        for b, n in enumerate(new):
            kk[b, :n], vv[b, :n] = k[at:at + n], v[at:at + n]
            at += n
        q = torch.randn(3, N, Hq, d, device="cuda", generator=g).to(t)
        o = torch.full_like(q, 7.0)
        views = [x.transpose(1, 2) for x in (q, kk, vv, o)]
        st = [x.stride()[:3] for x in views]
        assert gpu.flash_window_fwd(*views, 3, Hq, H, N, N, d, s2, gpu.Dtype.F16, window=window, sinks=sinks,
                                    lens=lens, q_strides=st[0], k_strides=st[1], v_strides=st[2],
                                    o_strides=st[3]) == 0
        _done(gpu)
        exp = plain.window_attn(*(_f64(x) for x in views[:3]), new, window, sinks, s2)
        for (b, h, i), w in exp.items():
            row = _f64(views[3][b, h, i])
            assert (row == 7.0).all() if w is None else np.abs(row - w).max() <= 2.0 ** -11 * 3 * 5 + 1e-4
    for _ in range(3):
        step(seqs)
    child = gpu.kv8_pool_fork(pool, seqs[0])[1]
    seqs.append(child)
    for _ in range(2):
        step(seqs)  # the first step gives one of the two a page of its own
    assert gpu.kv8_pool_free(pool, seqs.pop(1)) == 0
    src, dst = np.empty(pages, np.int32), np.empty(pages, np.int32)
    err, n = gpu.kv8_pool_compact(pool, src, dst, pages)
    assert err == 0 and n > 0
    copy(list(zip(src[:n].tolist(), dst[:n].tolist())))
    assert step(seqs) == [76, 39, 76]
    assert gpu.kv8_pool_destroy(pool) == 0


def test_decode_step_in_a_graph(gpu):
    """A decode step (append, attention) recorded into a runtime graph with the default stream, and
    the same calls captured by torch on its own stream; replayed as the lengths grow."""
    rng = np.random.default_rng(21)
    H, Hq, d, P, B = 2, 8, 64, 16, 3
    lens0 = [20, 1, 40]
    c, table = _fill(gpu, [n + 8 for n in lens0], H, P, d, rng)
    ref = Cache(gpu, c.k.shape[0], H, P, d)
    for a, b in zip((ref.k, ref.v, ref.ks, ref.vs), (c.k, c.v, c.ks, c.vs)):
        a.copy_(b)
    tab = _ints(table)
    lens, after = _ints(lens0), _ints([0] * B)
    x = torch.randn(B, H, d, device="cuda").half()
    q, o, o2 = torch.randn(B, Hq, d, device="cuda").half(), *(torch.empty(B, Hq, d, device="cuda").half() for _ in range(2))
    need = max(gpu.kv8_attn_workspace(c.handle, B, Hq)[1], 256)
    ws, ws2 = (torch.zeros(need, dtype=torch.uint8, device="cuda") for _ in range(2))

    def calls(cache, lens, after, out, ws, stream=None):
        assert gpu.kv8_append(cache, x, x, B, tab, table.shape[1], lens, B, 1, gpu.Dtype.F16, lens_out=after,
                              stream=stream) == 0
        assert gpu.kv8_attn(cache, q, out, tab, table.shape[1], after, B, Hq, 0.18, gpu.Dtype.F16, ws,
                            ws.numel(), window=30, sinks=2, stream=stream) == 0

    torch.cuda.synchronize()
    err, graph = gpu.vcGraphCreate()
    assert gpu.vcGraphBeginRecord(graph) == 0
    calls(c.handle, lens, after, o, ws)
    assert gpu.vcMemcpyAsync(lens, after, B * 4, gpu.VCMemcpyKind.DeviceToDevice) == 0
    assert gpu.vcGraphEndRecord(graph) == 0
    lens2, after2 = lens.clone(), after.clone()
    tg = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(tg):
        s = torch.cuda.current_stream().cuda_stream
        calls(ref.handle, lens2, after2, o2, ws2, s)
        lens2.copy_(after2)
    for i in range(5):
        x.copy_(torch.randn(B, H, d, device="cuda"))
        torch.cuda.synchronize()
        assert gpu.vcGraphLaunch(graph) == 0
        tg.replay()
        _done(gpu)
        now = [n + i + 1 for n in lens0]
        assert lens.tolist() == now and lens2.tolist() == now
        assert torch.equal(o, o2) and torch.equal(c.k, ref.k) and torch.equal(c.vs, ref.vs)
        k, ks, v, vs = c.host()
        want = plain.cache_attn(_f64(q), k, ks, v, vs, table, now, 30, 2, 0.18, P)
        assert np.abs(_f64(o) - want).max() <= 0.02
    assert gpu.vcGraphDestroy(graph) == 0


def test_two_streams_at_once(gpu):
    """The same cache read by two streams with a workspace each."""
    rng = np.random.default_rng(22)
    lens = [4000, 123, 900]
    c, table = _fill(gpu, lens, 2, 32, 128, rng)
    tab, ln = _ints(table), _ints(lens)
    q = torch.randn(3, 16, 128, device="cuda").half()
    need = max(gpu.kv8_attn_workspace(c.handle, 3, 16)[1], 256)
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [torch.zeros(need, dtype=torch.uint8, device="cuda") for _ in streams]
    outs = [[torch.empty_like(q) for _ in range(10)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(10):
        for s, w, o in zip(streams, ws, outs):
            assert gpu.kv8_attn(c.handle, q, o[i], tab, table.shape[1], ln, 3, 16, 0.12, gpu.Dtype.F16, w,
                                need, stream=s) == 0
    _done(gpu)
    first = outs[0][0]
    assert all(torch.equal(first, o) for row in outs for o in row)
    assert _attn_case(gpu, c, table, lens, 16, torch.float16, 0, 0)


def test_registry_launches(gpu):
    """The serving kernels through vcLaunchKernel give what the native entries give."""
    rng = np.random.default_rng(23)
    lens, Hq = [45, 10], 4
    c, table = _fill(gpu, [n + 2 for n in lens], 2, 16, 64, rng)
    d = Cache(gpu, c.k.shape[0], 2, 16, 64)
    for a, b in zip((d.k, d.v, d.ks, d.vs), (c.k, c.v, c.ks, c.vs)):
        a.copy_(b)
    tab, ln, W = _ints(table), _ints(lens), table.shape[1]
    x = torch.randn(2, 2, 64, device="cuda").half()
    q = torch.randn(2, Hq, 64, device="cuda").half()
    out = [[torch.zeros(2, Hq, 64, device="cuda").half() for _ in range(2)] for _ in range(2)]
    new = [_ints([0, 0]) for _ in range(2)]
    need = max(gpu.kv8_attn_workspace(c.handle, 2, Hq)[1], 256)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    p, i32, f32, i64 = gpu.ptr, gpu.i32, gpu.f32, gpu.i64
    src, dst = _ints([0]), _ints([1])
    lp = torch.randn(1, 4, 60, 64, device="cuda").half()
    dense = [4 * 60 * 64, 60 * 64, 64]
    import ctypes
    strides = (ctypes.c_int64 * 12)(*(dense * 4))
    lo = [torch.empty_like(lp) for _ in range(2)]

    def launch(name, args):
        err, k = gpu.vcGetKernel(name)
        assert err == 0
        assert gpu.vcLaunchKernel(k, 1, 1, args) == 0, name
        assert gpu.vcLaunchKernel(k, 1, 1, args[:-1]) == gpu.VCError.InvalidValue
        gpu.vcReleaseKernel(k)

    launch("vc.kv8_append", [gpu.structs(c.handle), p(x), p(x), i64(128), i64(128), i32(2), p(tab), i32(W),
                             p(ln), p(0), i32(2), i32(1), p(new[0]), i32(1)])
    launch("vc.kv8_attn", [gpu.structs(c.handle), p(q), i64(256), p(out[0][0]), i64(256), p(tab), i32(W),
                           p(new[0]), i32(2), i32(Hq), i32(20), i32(2), f32(0.18), i32(1), p(ws), i64(need)])
    launch("vc.kv8_copy_pages", [gpu.structs(gpu.kv8_layers([c.handle])), p(src), p(dst), i32(1)])
    launch("vc.flash_window", [p(lp), p(lp), p(lp), p(lo[0]), p(0), gpu.structs(strides), i32(1), i32(4),
                               i32(4), i32(60), i32(60), i32(64), i32(20), i32(2), f32(0.18), i32(1)])
    assert gpu.kv8_append(d.handle, x, x, 2, tab, W, ln, 2, 1, gpu.Dtype.F16, lens_out=new[1]) == 0
    assert gpu.kv8_attn(d.handle, q, out[1][0], tab, W, new[1], 2, Hq, 0.18, gpu.Dtype.F16, ws, need,
                        window=20, sinks=2) == 0
    assert gpu.kv8_copy_pages(gpu.kv8_layers([d.handle]), src, dst, 1) == 0
    assert gpu.flash_window_fwd(lp, lp, lp, lo[1], 1, 4, 4, 60, 60, 64, 0.18, gpu.Dtype.F16, window=20,
                                sinks=2) == 0
    _done(gpu)
    assert torch.equal(new[0], new[1]) and torch.equal(out[0][0], out[1][0]) and torch.equal(lo[0], lo[1])
    assert torch.equal(c.k, d.k) and torch.equal(c.vs, d.vs)
