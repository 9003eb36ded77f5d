"""The serving attentions at the ends of their documented ranges: value scales and
scores, against closed forms and the float64 forms of kv8_plain.py; and the same
bits from call to call."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv8_plain as plain
from test_gpu_serving import TYPES, Cache, _done, _dt, _f64, _fill, _ints

pytestmark = pytest.mark.gpu


def _attn_call(gpu, c, q, table, lens, scale, window=0, sinks=0):
    """One call over a cache as it is; q [B][Hq][d]."""
    B, Hq = q.shape[:2]
    o = torch.full_like(q, 7.0)
    ws = torch.zeros(gpu.kv8_attn_workspace(c.handle, B, Hq)[1], dtype=torch.uint8, device="cuda")
    assert gpu.kv8_attn(c.handle, q, o, _ints(table), table.shape[1], _ints(lens), B, Hq, scale,
                        _dt(gpu, q.dtype), ws, ws.numel(), window=window, sinks=sinks) == 0
    _done(gpu)
    return _f64(o)


def _code(x):
    return int(plain.to_e4m3(np.array([float(x)]))[0])


@pytest.mark.parametrize("Hq,d", [(1, 128), (9, 64), (20, 128)])
@pytest.mark.parametrize("n", [32, 128, 272, 5000, 90000])
@pytest.mark.parametrize("big,small", [(27, -100), (119, -100), (17, None), (119, None), (0, -100)])
def test_attn_value_scales_do_not_move_the_weights(gpu, big, small, n, Hq, d):
    """Equal scores over pages whose value scales are up to 2^219 apart (None: a page of scale 0, as
    memory comes): the pages with the small scale hold zeros, and their keys' share of the sum counts.
    One page holds ones: the first, the second, one of another warp, the last."""
    P = 16
    pages = -(-n // P)
    c = Cache(gpu, pages, 1, P, d)
    table = np.random.default_rng(n).permutation(pages).astype(np.int32)[None]
    c.k.fill_(_code(1.0))
    c.ks.fill_(2.0 ** -3)
    q = torch.randn(1, Hq, d, device="cuda").bfloat16()
    for at in sorted({0, 1, 2, 4, 9, pages - 1} & set(range(pages))):
        c.v.fill_(0)
        c.vs.fill_(0.0 if small is None else 2.0 ** small)
        c.v[table[0, at]] = _code(1.0)
        c.vs[table[0, at]] = 2.0 ** big
        # All weights are 1 / n: the output's rounding and the weights', all values of one sign.
        want = 2.0 ** big * min(P, n - at * P) / n
        got = _attn_call(gpu, c, q, table, [n], 0.1)
        assert (np.abs(got - want) <= want * (2.0 ** -8 + 2.0 ** -10)).all(), (at, got.min() / want, got.max() / want)


@pytest.mark.parametrize("exp", [119, 0, -100])
@pytest.mark.parametrize("n,heavy", [(600, 0), (600, 20), (40000, 5), (40000, 2499)])
def test_attn_lower_scores_keep_their_share(gpu, n, heavy, exp):
    """16 keys 10 log2 units above all others, at the ends of the range of value scales: the others are
    a good part of the sum."""
    P, d = 16, 64
    pages = -(-n // P)
    c = Cache(gpu, pages, 1, P, d)
    table = np.random.default_rng(n).permutation(pages).astype(np.int32)[None]
    c.k.fill_(0)
    c.k[:, :, :, 0] = _code(-2.0)
    c.k[table[0, heavy], :, :, 0] = _code(8.0)
    c.v.fill_(0)
    c.v[table[0, heavy]] = _code(1.0)
    c.vs.fill_(2.0 ** exp)
    q = torch.zeros(1, 3, d, device="cuda").bfloat16()
    q[:, :, 0] = 1.0
    want = 2.0 ** exp * P / (P + (n - P) * 2.0 ** -10)
    got = _attn_call(gpu, c, q, table, [n], 1.0)
    # The sum's n terms are exact powers of two; the output's rounding and the weights'.
    assert (np.abs(got - want) <= want * (2.0 ** -8 + 2.0 ** -10)).all(), got / want


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("size", [1e2, 1e4, 1e5, 1e6])
def test_attn_one_token_of_a_large_score(gpu, size, t):
    """A single key is the output whatever its score is: one weight, which is also the sum."""
    P, d, H, Hq = 16, 64, 4, 36
    rng = np.random.default_rng(int(size))
    for lens in ([1], [1, 1, 1]):
        B = len(lens)
        c = Cache(gpu, B, H, P, d)
        table = rng.permutation(B).astype(np.int32)[:, None]
        c.k.fill_(0)
        c.k[:, :, :, 0] = _code(1.0)
        c.v.copy_(torch.from_numpy(plain.to_e4m3(rng.standard_normal((B, H, P, d)) * 100)))
        c.vs.copy_(torch.from_numpy(rng.uniform(0.5, 2.0, (B, H)).astype(np.float32)))
        c.ks.copy_(torch.from_numpy(rng.uniform(0.5, 1.0, (B, H)).astype(np.float32)))
        q = torch.zeros(B, Hq, d, device="cuda")
        q[:, :, 0] = torch.from_numpy(rng.uniform(0.5, 1.0, (B, Hq)) * rng.choice([-1, 1], (B, Hq)))
        got = _attn_call(gpu, c, q.to(t), table, lens, size)
        v = plain.E4M3[c.v.cpu().numpy()][table[:, 0], :, 0] * c.vs.cpu().double().numpy()[table[:, 0], :, None]
        want = np.repeat(v, Hq // H, axis=1)
        # The weight's rounding to fp16, the exponentials and fp32 products, the output's.
        u = torch.finfo(t).eps / 2
        assert (np.abs(got - want) <= np.abs(want) * (u + 2.0 ** -11 + 2.0 ** -16) + 2.0 ** -24).all(), \
            (np.abs(got - want) / np.abs(want).clip(1e-9)).max()


def test_attn_zero_scores_of_large_factors(gpu):
    """Queries and K scales whose product is past fp32's range, at scores that are zero: the largest
    elements of one meet zeros of the other."""
    P, d, n = 16, 64, 100
    rng = np.random.default_rng(3)
    c, table = _fill(gpu, [n], 1, P, d, rng)
    q = torch.zeros(1, 4, d, device="cuda").bfloat16()
    q[:, :, 0] = 2.0 ** 100
    c.k[:, :, :, 0] = 0
    c.ks.fill_(2.0 ** 90)
    got = _attn_call(gpu, c, q, table, [n], 0.2)
    v = plain.E4M3[c.v.cpu().numpy()] * c.vs.cpu().double().numpy()[:, :, None, None]
    want = v[table[0]].transpose(0, 2, 1, 3).reshape(-1, d)[:n].mean(0)
    tol = 2.0 ** -8 * np.abs(want) + np.abs(v[np.isfinite(v)]).max() * (2.0 ** -10 + 2.0 ** -20)
    assert (np.abs(got - want) <= tol).all()


WINDOW_REPEATS = [
    # B, Hq, Hkv, Nq, Nk, d, window, sinks, lens: few row tiles, whose keys are shared, and many
    (1, 8, 2, 97, 97, 64, 64, 4, None), (1, 8, 1, 2000, 2000, 128, 0, 0, None),
    (4, 16, 4, 700, 1100, 128, 300, 130, None), (5, 16, 4, 1000, 1000, 128, 256, 4, [1000, 3, 0, 640, 129]),
    (2, 32, 8, 900, 2000, 64, 0, 0, None),
]


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("shape", WINDOW_REPEATS)
def test_window_same_answer_each_time(gpu, shape, t):
    """Call after call, with and without a wait between, and beside another stream's calls: the same
    bits, although the row tiles go to whichever CTA asks first."""
    B, Hq, Hkv, Nq, Nk, d, window, sinks, lens = shape
    q, k, v = (torch.randn(B, H, N, d, device="cuda").to(t) for H, N in ((Hq, Nq), (Hkv, Nk), (Hkv, Nk)))
    ln = None if lens is None else _ints(lens)
    streams = [None, torch.cuda.Stream()]
    outs = [torch.full_like(q, 7.0) for _ in range(24)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert gpu.flash_window_fwd(q, k, v, o, B, Hq, Hkv, Nq, Nk, d, 0.15, _dt(gpu, t), window=window,
                                    sinks=sinks, lens=ln, stream=streams[i >= 8 and i % 2]) == 0
        if i < 4:
            torch.cuda.synchronize()
    _done(gpu)
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("Hq,H,d,n,P", [(8, 2, 64, 200, 16), (32, 8, 128, 700, 64)])
def test_calls_that_follow_at_once_see_each_other(gpu, Hq, H, d, n, P, t):
    """Launches overlap the one before them: prompt attention, append of its output, page copies,
    attention over the copies, whose output is the next prompt's query, without a wait and with one
    after each call; on the default stream, on another, and in a graph."""
    pages = -(-n // P)
    rng = np.random.default_rng(n)
    ids = rng.permutation(2 * pages).astype(np.int32)
    src, dst = _ints(ids[:pages]), _ints(ids[pages:])
    x = [torch.randn(1, H, n, d, device="cuda").to(t) for _ in range(2)]
    q0 = torch.randn(1, Hq, n, d, device="cuda").to(t)

    def chain(rounds, after, stream=None):
        s = stream if stream is not None else torch.cuda.default_stream()
        with torch.cuda.stream(s):
            c = Cache(gpu, 2 * pages, H, P, d)
            q, o = q0.clone(), torch.zeros(1, Hq, n, d, device="cuda", dtype=t)
            one = [torch.zeros(1, Hq, d, device="cuda", dtype=t) for _ in range(2)]
            zero, lens = _ints([0]), _ints([0])
            ws = torch.zeros(gpu.kv8_attn_workspace(c.handle, 1, Hq)[1], dtype=torch.uint8, device="cuda")
            out = torch.zeros(rounds, 2, Hq, d, device="cuda", dtype=t)
            torch.cuda.synchronize()

            def go(i, s):
                assert gpu.flash_window_fwd(q, x[0], x[1], o, 1, Hq, H, n, n, d, 0.2, _dt(gpu, t), window=90, sinks=2,
                                            stream=s) == 0
                after()
                # The output's memory as tokens of the cache, V one row on.
                assert gpu.kv8_append(c.handle, o, o[:, :, 1:], n - 1, src.view(1, -1), pages, zero, 1, n - 1, _dt(gpu, t),
                                      lens_out=lens, k_stride=H * d, v_stride=H * d, stream=s) == 0
                after()
                assert gpu.kv8_copy_pages(gpu.kv8_layers([c.handle]), src, dst, pages, stream=s) == 0
                after()
                # Hq rows of the first head as queries, from row 0 and from row 1 on.
                for side, (table, to) in enumerate(((dst, one[0]), (src, one[1]))):
                    assert gpu.kv8_attn(c.handle, q[0, :, side], to, table.view(1, -1), pages, lens, 1, Hq, 0.2,
                                        _dt(gpu, t), ws, ws.numel(), window=60, sinks=1, stream=s) == 0
                    after()
            return c, q, one, out, go, s

    def run(rounds, after, stream=None):
        c, q, one, out, go, s = chain(rounds, after, stream)
        with torch.cuda.stream(s):
            for i in range(rounds):
                go(i, s)
                out[i, 0].copy_(one[0][0])
                out[i, 1].copy_(one[1][0])
                q[0, :, :2].copy_(torch.stack(one)[:, 0].transpose(0, 1))
        torch.cuda.synchronize()
        return out

    rounds = 40
    want = run(rounds, torch.cuda.synchronize)
    assert torch.isfinite(want).all() and want.abs().max() > 0.01
    assert not torch.equal(want[:, 0], want[:, 1])
    for stream in (None, torch.cuda.Stream()):
        assert torch.equal(run(rounds, lambda: None, stream), want)
    c, q, one, out, go, _ = chain(rounds, lambda: None)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(0, torch.cuda.current_stream())
        q[0, :, :2].copy_(torch.stack(one)[:, 0].transpose(0, 1))
    for i in range(rounds):
        graph.replay()
        out[i, 0].copy_(one[0][0])
        out[i, 1].copy_(one[1][0])
    _done(gpu)
    assert torch.equal(out, want)


def test_two_threads_at_once(gpu):
    """Calls of two host threads, each with a stream, a workspace and outputs of its own, over one
    cache: what one thread alone gets."""
    import threading
    rng = np.random.default_rng(41)
    lens = [900, 17, 300]
    c, table = _fill(gpu, lens, 2, 32, 128, rng)
    tab, ln = _ints(table), _ints(lens)
    q = torch.randn(3, 8, 128, device="cuda").half()
    p = torch.randn(1, 8, 500, 128, device="cuda").half()
    need = gpu.kv8_attn_workspace(c.handle, 3, 8)[1]
    torch.cuda.synchronize()
    results, errors = {}, []

    def work(name, count):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
            o = [torch.zeros_like(q) for _ in range(count)]
            w = [torch.zeros_like(p) for _ in range(count)]
        for i in range(count):
            errors.append(int(gpu.kv8_attn(c.handle, q, o[i], tab, table.shape[1], ln, 3, 8, 0.12, gpu.Dtype.F16, ws,
                                           need, stream=s)))
            errors.append(int(gpu.flash_window_fwd(p, p, p, w[i], 1, 8, 8, 500, 500, 128, 0.1, gpu.Dtype.F16,
                                                   window=100, stream=s)))
        s.synchronize()
        results[name] = o, w

    work("alone", 1)
    threads = [threading.Thread(target=work, args=(i, 60)) for i in range(2)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    _done(gpu)
    assert set(errors) == {0}
    (o,), (w,) = results["alone"]
    for i in range(2):
        assert all(torch.equal(x, o) for x in results[i][0]) and all(torch.equal(x, w) for x in results[i][1])
