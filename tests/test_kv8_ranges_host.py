"""The serving entries at the ends of their ranges, on the CPU."""
from __future__ import annotations

import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID = 1
BUF = np.zeros(1 << 12, np.uint8)
A = (BUF.ctypes.data + 255) & ~255


def test_index_arithmetic_at_its_ends(tmp_path):
    exe = tmp_path / "kv8_ranges"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-I" + os.path.join(ROOT, "vkcuda_b200", "csrc"),
                    os.path.join(ROOT, "tests", "hosts", "kv8_ranges_host.cpp"), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout == "PASS\n"


@pytest.mark.parametrize("kw", [
    # Spans that wrap around 64 bits, to a few bytes.
    dict(Nq=1 << 26, q_strides=[1 << 37, 1 << 37, 1 << 37]),
    dict(Nk=(1 << 26) + 1, k_strides=[1 << 37, 1 << 37, 1 << 37]),
    dict(B=2, Nk=(1 << 26) + 1, v_strides=[1 << 37, 1 << 37, 1 << 37]),
    dict(Nq=(1 << 27) + 1, o_strides=[1 << 37, 1 << 37, 1 << 36])])
def test_window_spans_past_64_bits(vc, kw):
    a = dict(Q=A, K=A, V=A, O=A, B=1, Hq=4, Hkv=2, Nq=16, Nk=16, d=64, scale_log2=0.1, dtype=vc.Dtype.F16)
    a.update(kw)
    assert vc.flash_window_fwd(**a) == INVALID


@pytest.mark.parametrize("kw", [dict(num_pages=(1 << 25) + 1, page_stride=1 << 39),
                                dict(num_pages=(1 << 30) + 1, scale_stride=1 << 32),
                                dict(num_pages=(1 << 24) + 1, scale_stride=1 << 38)])
def test_cache_spans_past_64_bits(vc, kw):
    c = vc.kv8_cache(**dict(dict(k=A, v=A, k_scale=A, v_scale=A, num_pages=4, heads=2, page_size=16,
                                 head_dim=64), **kw))
    assert vc.kv8_append(c, A, A, 2, A, 4, A, 2, 1, vc.Dtype.F16) == INVALID
    assert vc.kv8_attn(c, A, A, A, 4, A, 1, 4, 0.1, vc.Dtype.F16, A, 1 << 30) == INVALID
    assert vc.kv8_copy_pages(vc.kv8_layers([c]), A, A, 1) == INVALID


def test_append_rows_past_64_bits(vc):
    c = vc.kv8_cache(A, A, A, A, 4, 2, 16, 64)
    for kw in (dict(k_stride=1 << 38), dict(v_stride=1 << 37)):
        assert vc.kv8_append(c, A, A, (1 << 26) + 1, A, 4, A, 1, 1, vc.Dtype.F16, **kw) == INVALID


def test_window_waits_cover_the_longest_pair(tmp_path):
    """A wait that lasts as long as a pair of row tiles grows with its keys: 4 s alone were too short
    from 2^28 keys on."""
    from vkcuda_b200 import build
    exe = tmp_path / "window_wait"
    cuda = os.path.join(os.path.dirname(os.path.dirname(build.nvcc())), "include")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I" + cuda, "-I" + os.path.join(ROOT, "vkcuda_b200", "csrc"),
                    os.path.join(ROOT, "tests", "hosts", "window_wait_host.cpp"), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout == "PASS\n"


def test_addresses_without_exceptions(vc):
    """Host arrays and ctypes objects, which most calls of the runtime get, reach their address by
    tests, not by a caught exception (0.15 instead of 0.65 us)."""
    import ctypes
    import sys
    array, words, raw = np.zeros(3), (ctypes.c_int * 3)(), bytearray(8)
    raised = []
    mon = sys.monitoring
    mon.use_tool_id(mon.PROFILER_ID, "addresses")
    mon.register_callback(mon.PROFILER_ID, mon.events.RAISE, lambda *a: raised.append(a))
    mon.set_events(mon.PROFILER_ID, mon.events.RAISE)
    try:
        got = [vc._addr(x) for x in (array, words, raw, 5, None)]
    finally:
        mon.set_events(mon.PROFILER_ID, 0)
        mon.free_tool_id(mon.PROFILER_ID)
    assert got[:2] == [array.ctypes.data, ctypes.addressof(words)] and got[3:] == [5, None]
    assert not raised
    assert [vc._at(x) for x in (array, words, 5, None)] == got[:2] + got[3:]


def test_documented_limits(vc):
    """The sizes that the header gives are taken as far as the check for a GPU goes (which a machine
    without one fails), and the next one is refused."""
    def window(**kw):
        a = dict(Q=A, K=A, V=A, O=A, B=1, Hq=1, Hkv=1, Nq=1, Nk=1, d=64, scale_log2=0.1, dtype=vc.Dtype.F16)
        a.update(kw)
        return vc.flash_window_fwd(**a)

    def attn(heads=1, **kw):
        a = dict(cache=vc.kv8_cache(A, A, A, A, 1, heads, 16, 64), Q=A, O=A, table=A, table_width=1, lens=A, B=1,
                 Hq=heads, scale_log2=0.1, dtype=vc.Dtype.F16, workspace=A, workspace_bytes=0)
        a.update(kw)
        return vc.kv8_attn(**a)

    refused = (INVALID,)
    if vc.vcInit() == 0:
        pytest.skip("with a GPU the host addresses are refused by themselves")
    assert window(B=65535) not in refused and window(B=65536) in refused
    assert window(Hq=65535) not in refused and window(Hq=32768, B=2) in refused
    assert window(Nq=1 << 30) not in refused and window(Nq=(1 << 30) + 1) in refused
    assert window(Nk=1 << 30) not in refused and window(Nk=(1 << 30) + 1) in refused
    assert attn(B=65535) not in refused and attn(B=65536) in refused
    assert attn(Hq=65535) not in refused and attn(Hq=65536) in refused
    assert attn(heads=65535) not in refused and attn(heads=65536) in refused
    most = ((1 << 31) - 1) // 16
    assert attn(table_width=most) not in refused and attn(table_width=most + 1) in refused
