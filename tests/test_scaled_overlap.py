"""CPU checks of what the append to block-scaled pages refuses because its workgroups, which run in
any order, would take from each other: the strided arithmetic against sets of bytes, and the C ABI's
refusals (pointers are checked, never followed)."""

import ctypes
import os
import random
import subprocess

import pytest

from helios_amd import build as hbuild
from helios_amd import qmm
from test_attention_abi import BAD, P, batch, heads, lib, q_heads  # noqa: F401
from test_serving_abi import append, e4m3, scales

HERE = os.path.dirname(os.path.abspath(__file__))
MB = 1 << 20


@pytest.fixture(scope="module")
def host():
    so = os.path.join(HERE, "_build", "liboverlap.so")
    src, dep = os.path.join(HERE, "overlap_host.cpp"), os.path.join(hbuild.CSRC, "overlap.h")
    if not os.path.exists(so) or any(os.path.getmtime(d) > os.path.getmtime(so) for d in (src, dep)):
        os.makedirs(os.path.dirname(so), exist_ok=True)
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fPIC", "-shared", "-I", hbuild.CSRC, src, "-o", so], check=True, capture_output=True)
    of = ctypes.CDLL(so)
    u = ctypes.c_uint64
    of.rt_overlap.argtypes = [u, u, u, u, ctypes.POINTER(u), ctypes.POINTER(u)]
    of.rt_rows_overlap.argtypes = [u] * 7
    return of


def strided(host, a, a_len, b, b_len, axes):
    three = ctypes.c_uint64 * 3
    return bool(host.rt_overlap(a, a_len, b, b_len, three(*[n for n, _ in axes]), three(*[s for _, s in axes])))


def taken(at, length, axes):
    starts = [at]
    for n, s in axes:
        starts = [x + i * s for x in starts for i in range(n)]
    return {x + j for x in starts for j in range(length)}


def test_strided_arrays_against_sets_of_bytes(host):
    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(4000):
        axes = [(rng.randint(1, 4), rng.choice([0, 1, 3, 4, 8, 12, 16, 24, 48, 64])) for _ in range(3)]
        a_len, b_len = rng.randint(1, 9), rng.randint(1, 9)
        a, b = 1000, 1000 + rng.randint(-300, 300)
        want = bool(taken(a, a_len, axes) & taken(b, b_len, axes))
        assert strided(host, a, a_len, b, b_len, axes) == want, (axes, a_len, b_len, b - a)
        seen[want] += 1
    assert min(seen) > 500


def test_rows_against_sets_of_bytes(host):
    rng = random.Random(2)
    seen = [0, 0]
    for _ in range(6000):
        rows = rng.randint(1, 6)
        a_len, b_len = rng.randint(1, 12), rng.randint(1, 12)
        sa, sb = a_len + rng.choice([0, 1, 10, 30]), b_len + rng.choice([0, 1, 10, 30])
        if rng.random() < 0.3:
            sa = sb = max(sa, sb)
        a, b = 1000, 1000 + rng.randint(-200, 200)
        want = bool(taken(a, a_len, [(rows, sa)]) & taken(b, b_len, [(rows, sb)]))
        assert bool(host.rt_rows_overlap(a, sa, a_len, b, sb, b_len, rows)) == want, (rows, sa, a_len, sb, b_len, b - a)
        seen[want] += 1
    assert min(seen) > 500


def test_the_largest_arrays(host):
    """No sum passes what the arithmetic holds, and what is apart is found so at once."""
    axes = [(1 << 30, 1 << 38), (65536, 1 << 10), (4096, 1 << 26)]
    assert strided(host, 1 << 46, 512, 1 << 46, 512, axes)
    assert strided(host, 1 << 46, 512, (1 << 46) + (3 << 38) + (7 << 26) + 511, 512, axes)
    assert not strided(host, 1 << 46, 512, (1 << 46) + (3 << 38) + (7 << 26) + 512, 512, axes)
    assert not host.rt_rows_overlap(1 << 40, 1 << 33, 1 << 20, (1 << 40) + (1 << 20), 1 << 33, 1 << 20, (1 << 24) - 1)
    assert host.rt_rows_overlap(1 << 40, 1 << 33, 1 << 20, (1 << 40) + (1 << 20) + 2, (1 << 33) - 2, 1 << 20, (1 << 24) - 1)


# e4m3() has 4 pages of 8 heads of 64 slots of 256 bytes: 512 KiB; scales() 4 bytes a head
APART = dict(pg=e4m3(v_dev=P + MB), sc=scales(k_dev=P + 4 * MB, v_dev=P + 5 * MB))


@pytest.mark.parametrize("pg", [e4m3(), e4m3(v_dev=P + 16), e4m3(v_dev=P + MB // 2 - 16), e4m3(v_dev=P - 64 * 256),
                                e4m3(v_dev=P + 8 * 64 * 512, token_stride=512, head_stride=64 * 512, page_stride=2 * 64 * 512),  # heads and pages of one run into others
                                e4m3(num_pages=1, v_dev=P + 7 * 64 * 256)])
def test_pages_that_share_bytes(lib, pg):
    assert append(lib, **{**APART, "pg": pg}) == BAD and "pages must not overlap" in qmm.last_error()


@pytest.mark.parametrize("at", [0, 1, 3, 4 * 8 * 4 - 1, -5])
def test_scales_that_share_bytes(lib, at):
    sc = scales(k_dev=P + 4 * MB, v_dev=P + 4 * MB + at)
    assert append(lib, **{**APART, "sc": sc}) == BAD and "scales must not overlap" in qmm.last_error()


K, V = heads(x_dev=P + 8 * MB), heads(x_dev=P + 9 * MB)  # rows of 4096 elements, 8 heads of 256


@pytest.mark.parametrize("out", [8 * MB, 9 * MB, 9 * MB + 4080, 8 * MB + 8192 + 4080, 8 * MB - 8176, 9 * MB - 16368])
def test_out_over_rows_of_keys_and_values(lib, out):
    q = q_heads(x_dev=P + 10 * MB, out_dev=P + out)
    assert append(lib, q=q, k=K, v=V, **APART) == BAD and "k's or v's rows" in qmm.last_error()


@pytest.mark.parametrize("kw", [dict(out_dev=P + 10 * MB + 16), dict(out_dev=P + 10 * MB - 8176), dict(out_dev=P + 10 * MB, out_stride=8192),
                                dict(out_dev=P + 10 * MB + 8192)])
def test_out_over_other_places_of_q(lib, kw):
    q = q_heads(**{"x_dev": P + 10 * MB, **kw})
    assert append(lib, q=q, k=K, v=V, **APART) == BAD and "be its x" in qmm.last_error()
