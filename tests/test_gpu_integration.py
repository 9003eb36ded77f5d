"""The serving example of the integration notes runs as it is written: every call succeeds, and what the
cache and the attention hold is what the plain forms give."""
from __future__ import annotations

import math
import os
import textwrap

import numpy as np
import pytest
import torch

import kv8_plain as plain
from test_gpu_serving import Cache, _done, _f64, _ints

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Calls:
    """The binding, with the error codes of all calls kept."""

    def __init__(self, vc):
        self.vc, self.errors = vc, []

    def __getattr__(self, name):
        f = getattr(self.vc, name)
        if not name.startswith(("kv8_", "flash_")) or name == "kv8_cache":
            return f

        def call(*a, **k):
            out = f(*a, **k)
            self.errors.append((name, int(out[0] if isinstance(out, tuple) else out)))
            return out
        return call


def _example():
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    text = text[text.index("## 4a."):]
    block = text[text.index("    from vkcuda_b200 import vc\n"):text.index("\n* ")]
    return textwrap.dedent(block).replace("from vkcuda_b200 import vc\n", "")


def test_the_serving_example(gpu):
    pages, heads, q_heads, batch, n, width, P, d = 32, 2, 8, 3, 150, 4, 64, 128
    new = [70, 1, 130]
    total, most, bf = sum(new), max(new), torch.bfloat16
    c = Cache(gpu, pages, heads, P, d)

    def rand(*shape):
        return torch.randn(*shape, device="cuda").to(bf)

    # The pool gives the prompt the pages 0, 1, 2; the batch has others.
    tables = np.array([[10, 11, -1, -1], [12, -1, -1, -1], [13, 14, 15, -1]], np.int32)
    names = dict(vc=Calls(gpu), k=c.k, v=c.v, k_scale=c.ks, v_scale=c.vs, pages=pages, heads=heads, q_heads=q_heads,
                 batch=batch, n=n, width=width, scale_log2=1.4426950408889634 / math.sqrt(d),
                 row=torch.empty(width, dtype=torch.int32), table=_ints([[0] * width]), zero=_ints([0]),
                 q=rand(n, q_heads, d), k_new=rand(n, heads, d), v_new=rand(n, heads, d), o=rand(n, q_heads, d),
                 total=total, most=most, k_all=rand(total, heads, d), v_all=rand(total, heads, d),
                 tables=_ints(tables), starts=_ints([0] * batch), cu=_ints(np.concatenate([[0], np.cumsum(new)])),
                 lens=_ints([0] * batch), lens_next=_ints([0] * batch), k1=rand(batch, heads, d),
                 v1=rand(batch, heads, d), q1=rand(batch, q_heads, d), o1=rand(batch, q_heads, d),
                 workspace=torch.zeros(64 << 20, dtype=torch.uint8, device="cuda"))
    want = c.host()
    exec(_example(), names)
    _done(gpu)
    called = names["vc"].errors
    assert [e for e in called if e[1]] == [] and {x for x, _ in called} == {
        "kv8_attn_workspace", "kv8_pool_create", "kv8_pool_new", "kv8_pool_extend", "kv8_pool_pages",
        "flash_window_fwd", "kv8_append", "kv8_attn"}
    assert names["copy"] is None and (names["used"], names["tokens"]) == (3, n)
    after = [x + 1 for x in new]
    assert names["lens"].tolist() == new and names["lens_next"].tolist() == after
    for i, key in ((0, "k"), (2, "v")):
        plain.append(want[i], want[i + 1], _f64(names[key + "_new"]), [[0, 1, 2, -1]], [0], [n], P)
        plain.append(want[i], want[i + 1], _f64(names[key + "_all"]), tables, [0] * batch, new, P)
        plain.append(want[i], want[i + 1], _f64(names[key + "1"]), tables, new, [1] * batch, P)
    for g, w in zip(c.host(), want):
        assert np.array_equal(g, w)
    s = names["scale_log2"]
    exp = plain.cache_attn(_f64(names["q1"]), *want, tables, after, 4096, 4, s, P)
    assert np.abs(_f64(names["o1"]) - exp).max() <= 2.0 ** -8 * 4 + 2.0 ** -10 * 5
    exp = plain.window_attn(*(_f64(names[x]).transpose(1, 0, 2)[None] for x in ("q", "k_new", "v_new")), None, 4096, 4, s)
    got = _f64(names["o"])
    for (_, h, i), w in exp.items():
        assert np.abs(got[i, h] - w).max() <= 2.0 ** -8 * np.abs(w).max() + 2 * 2.0 ** -8 * 5
    assert gpu.kv8_pool_destroy(names["pool"]) == 0
