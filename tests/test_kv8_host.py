"""The serving entries on the CPU: refusals (every argument check runs before
the GPU is asked for), the page pool against a model in Python, the cache's
index arithmetic, and the plain forms that the GPU tests compare with."""
from __future__ import annotations

import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

import kv8_plain as plain

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID = 1


def test_index_arithmetic(tmp_path):
    exe = tmp_path / "kv8_index"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror",
                    "-I" + os.path.join(ROOT, "vkcuda_b200", "csrc"),
                    os.path.join(ROOT, "tests", "hosts", "kv8_index_host.cpp"), "-o", str(exe)],
                   check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout == "PASS\n"


def test_plain_e4m3_matches_torch():
    import torch
    x = np.random.default_rng(0).standard_normal(20000) * np.exp2(
        np.random.default_rng(1).integers(-12, 10, 20000))
    x = np.concatenate([x, plain.E4M3[np.isfinite(plain.E4M3)], [0.0, 448.0, -448.0, 2.0 ** -10, 1.5 * 2.0 ** -9]])
    x = x[np.abs(x) <= 448].astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(plain.to_e4m3(x.astype(np.float64)), want)


# ------------------------------------------------------------------ refusals
BUF = np.zeros(1 << 16, np.uint8)
A = (BUF.ctypes.data + 255) & ~255


def _cache(vc, **kw):
    args = dict(k=A, v=A, k_scale=A, v_scale=A, num_pages=4, heads=2, page_size=16, head_dim=64)
    args.update(kw)
    return vc.kv8_cache(**args)


def _window(vc, **kw):
    a = dict(Q=A, K=A, V=A, O=A, B=1, Hq=4, Hkv=2, Nq=16, Nk=16, d=64, scale_log2=0.1,
             dtype=vc.Dtype.F16)
    a.update(kw)
    return vc.flash_window_fwd(**a)


@pytest.mark.parametrize("kw", [
    dict(Q=0), dict(K=0), dict(V=0), dict(O=0), dict(Q=A + 2), dict(O=A + 8), dict(B=0), dict(B=-1),
    dict(Hq=0), dict(Hkv=0), dict(Hq=3), dict(Nq=0), dict(Nk=0), dict(Nq=-1), dict(d=96), dict(d=32),
    dict(d=256), dict(dtype=0), dict(dtype=3), dict(window=-1), dict(sinks=-1), dict(lens=A + 1),
    dict(B=40000, Hq=2), dict(q_strides=[1024, 1024, 63]), dict(q_strides=[1024, 1024, 32]),
    dict(k_strides=[0, 0, 64]), dict(o_strides=[0, -1024, 64]), dict(v_strides=[0, 1024, 68]),
    dict(q_strides=[0, 1 << 39, 64]), dict(scale_log2=0.0), dict(scale_log2=-1.0),
    dict(scale_log2=float("nan")), dict(scale_log2=float("inf")), dict(Nk=(1 << 30) + 8)])
def test_window_refusals(vc, kw):
    assert _window(vc, **kw) == INVALID


@pytest.mark.parametrize("kw", [
    dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=0), dict(k=A + 8), dict(v_scale=A + 2),
    dict(num_pages=0), dict(heads=0), dict(heads=65536), dict(page_size=24), dict(page_size=256),
    dict(page_size=8), dict(head_dim=96), dict(head_dim=0), dict(page_stride=1024),
    dict(page_stride=2056), dict(scale_stride=1)])
def test_cache_refusals(vc, kw):
    c = _cache(vc, **kw)
    assert vc.kv8_append(c, A, A, 2, A, 4, A, 2, 1, vc.Dtype.F16) == INVALID
    assert vc.kv8_attn(c, A, A, A, 4, A, 1, 4, 0.1, vc.Dtype.F16, A, 1 << 30) == INVALID
    assert vc.kv8_copy_pages(vc.kv8_layers([c]), A, A, 1) == INVALID


@pytest.mark.parametrize("kw", [
    dict(K=0), dict(V=0), dict(K=A + 2), dict(tokens=-1), dict(tokens=1), dict(table=0),
    dict(table=A + 1), dict(table_width=0), dict(start=0), dict(B=-1), dict(max_new=-1),
    dict(dtype=0), dict(dtype=7), dict(k_stride=64), dict(v_stride=132), dict(cu=A + 2),
    dict(lens_out=A + 4096), dict(lens_out=A + 8192 + 4), dict(lens_out=A + 2)])
def test_append_refusals(vc, kw):
    a = dict(cache=_cache(vc), K=A, V=A, tokens=2, table=A + 8192, table_width=4, start=A + 4096, B=2,
             max_new=1, dtype=vc.Dtype.F16)
    a.update(kw)
    assert vc.kv8_append(**a) == INVALID


@pytest.mark.parametrize("kw", [
    dict(Q=0), dict(O=0), dict(Q=A + 2), dict(table=0), dict(lens=0), dict(table_width=0), dict(B=-1),
    dict(Hq=0), dict(Hq=3), dict(window=-1), dict(sinks=-1), dict(dtype=0), dict(q_stride=192),
    dict(o_stride=260), dict(workspace=0), dict(workspace=A + 16), dict(B=65536),
    dict(table_width=1 << 28), dict(scale_log2=0.0), dict(scale_log2=-0.5),
    dict(scale_log2=float("nan"))])
def test_attn_refusals(vc, kw):
    a = dict(cache=_cache(vc), Q=A, O=A, table=A, table_width=4, lens=A, B=1, Hq=4, scale_log2=0.1,
             dtype=vc.Dtype.F16, workspace=A, workspace_bytes=1 << 30)
    a.update(kw)
    assert vc.kv8_attn(**a) == INVALID


def test_copy_refusals(vc):
    one = vc.kv8_layers([_cache(vc)])
    assert vc.kv8_copy_pages(one, 0, A, 1) == INVALID
    assert vc.kv8_copy_pages(one, A, 0, 1) == INVALID
    assert vc.kv8_copy_pages(one, A, A + 2, 1) == INVALID
    assert vc.kv8_copy_pages(one, A, A, -1) == INVALID
    assert vc.kv8_copy_pages((vc.Kv8Cache * 0)(), A, A, 1) == INVALID
    two = vc.kv8_layers([_cache(vc), _cache(vc, num_pages=5)])
    assert vc.kv8_copy_pages(two, A, A, 1) == INVALID


def test_null_caches(vc):
    lib = vc.library()
    n = ctypes.c_size_t(0)
    assert lib.vc_kv8_attn_workspace(None, 1, 1, ctypes.byref(n)) == INVALID
    assert lib.vc_kv8_append(None, A, A, 128, 128, 1, A, 1, A, None, 1, 1, None, 1, None) == INVALID
    assert lib.vc_kv8_copy_pages(None, 1, A, A, 1, None) == INVALID
    c = _cache(vc)
    assert vc.kv8_attn_workspace(c, 1, 3)[0] == INVALID  # 3 query heads over 2 K/V heads
    assert vc.kv8_attn_workspace(c, -1, 4)[0] == INVALID


def test_registry_knows_the_serving_kernels(vc):
    for name in ("vc.flash_window", "vc.kv8_append", "vc.kv8_attn", "vc.kv8_copy_pages"):
        err, k = vc.vcGetKernel(name)
        assert err == 0 and k
        vc.vcReleaseKernel(k)


# ------------------------------------------------------------------ the pool
class Model:
    """The pool in plain Python: pages by sequence, lowest free page first."""

    def __init__(self, pages, size):
        self.pages, self.size, self.seqs, self.next = pages, size, {}, 1

    def held(self, p):
        return sum(p in s[0] for s in self.seqs.values())

    def free(self):
        return [p for p in range(self.pages) if not self.held(p)]

    def extend(self, s, n):
        pages, tokens = self.seqs[s]
        want = -(-(tokens + n) // self.size)
        copy = n > 0 and tokens % self.size != 0 and self.held(pages[-1]) > 1
        free = self.free()
        if want - len(pages) + copy > len(free):
            return None
        made = (-1, -1)
        pages = list(pages)
        if copy:
            made = (pages[-1], free.pop(0))
            pages[-1] = made[1]
        while len(pages) < want:
            pages.append(free.pop(0))
        self.seqs[s] = (pages, tokens + n)
        return made

    def compact(self):
        live = self.pages - len(self.free())
        moves = list(zip([p for p in range(live, self.pages) if self.held(p)],
                         [p for p in range(live) if not self.held(p)]))
        to = dict(moves)
        self.seqs = {s: ([to.get(p, p) for p in pages], t) for s, (pages, t) in self.seqs.items()}
        return moves


@pytest.mark.parametrize("seed", range(12))
def test_pool_against_model(vc, seed):
    rng = random.Random(seed)
    pages, size = rng.choice([1, 7, 40]), rng.choice([1, 16, 64])
    err, pool = vc.kv8_pool_create(pages, size)
    assert err == 0
    m = Model(pages, size)
    row = np.empty(pages, np.int32)
    src, dst = np.empty(pages, np.int32), np.empty(pages, np.int32)
    for _ in range(250):
        op = rng.choice(["new", "extend", "extend", "extend", "fork", "free", "compact"])
        s = rng.choice(list(m.seqs)) if m.seqs else None
        if op == "new" or s is None:
            assert vc.kv8_pool_new(pool) == (0, m.next)
            m.seqs[m.next] = ([], 0)
            m.next += 1
        elif op == "extend":
            n = rng.choice([0, 1, 1, size, rng.randrange(4 * size + 1)])
            want = m.extend(s, n)
            got = vc.kv8_pool_extend(pool, s, n)
            assert got == ((vc.VCError.OutOfMemory, None) if want is None else
                           (0, None if want[0] < 0 else want))
        elif op == "fork" and len(m.seqs) < 12:
            assert vc.kv8_pool_fork(pool, s) == (0, m.next)
            m.seqs[m.next] = m.seqs[s]
            m.next += 1
        elif op == "free":
            assert vc.kv8_pool_free(pool, s) == 0
            del m.seqs[s]
        elif op == "compact":
            want = m.compact()
            err, n = vc.kv8_pool_compact(pool, src, dst, pages)
            assert err == 0 and list(zip(src[:n].tolist(), dst[:n].tolist())) == want
        assert vc.kv8_pool_info(pool) == (0, len(m.free()), len(m.seqs))
        for q, (want, tokens) in m.seqs.items():
            err, n, t = vc.kv8_pool_pages(pool, q, row, pages)
            assert (err, n, t) == (0, len(want), tokens)
            assert row.tolist() == want + [-1] * (pages - n)
    assert vc.kv8_pool_destroy(pool) == 0


def test_pool_refusals(vc):
    assert vc.kv8_pool_create(0, 16)[0] == INVALID
    assert vc.kv8_pool_create(4, 0)[0] == INVALID
    assert vc.kv8_pool_new(None)[0] == INVALID
    assert vc.kv8_pool_destroy(None) == 0
    _, pool = vc.kv8_pool_create(4, 16)
    _, s = vc.kv8_pool_new(pool)
    assert vc.kv8_pool_fork(pool, 99)[0] == INVALID
    assert vc.kv8_pool_free(pool, 99) == INVALID
    assert vc.kv8_pool_extend(pool, 99, 1)[0] == INVALID
    assert vc.kv8_pool_extend(pool, s, -1)[0] == INVALID
    assert vc.kv8_pool_extend(pool, s, 1 << 62)[0] == vc.VCError.OutOfMemory
    assert vc.kv8_pool_extend(pool, s, 65)[0] == vc.VCError.OutOfMemory
    assert vc.kv8_pool_extend(pool, s, 64) == (0, None)
    row = np.empty(2, np.int32)
    assert vc.kv8_pool_pages(pool, s, row, 2)[0] == INVALID    # four pages do not fit
    assert vc.kv8_pool_pages(pool, s) == (0, 4, 64)
    _, t = vc.kv8_pool_new(pool)
    assert vc.kv8_pool_extend(pool, t, 1)[0] == vc.VCError.OutOfMemory
    assert vc.kv8_pool_pages(pool, t) == (0, 0, 0)              # nothing changed
    assert vc.kv8_pool_free(pool, s) == 0
    assert vc.kv8_pool_extend(pool, t, 1) == (0, None)
    # A compaction that does not fit says how many copies it has.
    _, u = vc.kv8_pool_new(pool)
    vc.kv8_pool_extend(pool, u, 16)
    vc.kv8_pool_free(pool, t)
    assert vc.kv8_pool_compact(pool, None, None, 0) == (INVALID, 1)
    assert vc.kv8_pool_pages(pool, u, row, 2) == (0, 1, 16) and row[0] == 1
    vc.kv8_pool_destroy(pool)
