"""CPU check of how the attention kernels cut a launch into items: the host sizes the launch and
its partial sums for the slots and the most tiles that a batch of so many rows and requests can
have, and the device cuts the batch it finds.  An item past that number would be lost, and its
rows with it."""

import ctypes
import os
import subprocess

import numpy as np
import pytest

from helios_amd import build as hbuild

HERE = os.path.dirname(os.path.abspath(__file__))
NO_TILES = 0x40000000  # more rows than any request has


@pytest.fixture(scope="module")
def items():
    so = os.path.join(HERE, "_build", "libkvitems.so")
    src, dep = os.path.join(HERE, "kv_items_host.cpp"), os.path.join(hbuild.CSRC, "kv_index.h")
    if not os.path.exists(so) or any(os.path.getmtime(d) > os.path.getmtime(so) for d in (src, dep)):
        os.makedirs(os.path.dirname(so), exist_ok=True)
        subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                        "-I", hbuild.CSRC, src, "-o", so], check=True, capture_output=True)
    lib = ctypes.CDLL(so)
    i, p = ctypes.c_int, ctypes.c_void_p
    lib.kv_most_tiles.argtypes = [ctypes.c_int64, ctypes.c_int64, i, i, i]
    lib.kv_items.argtypes = [p, p, i, i, i, i, i, i, i, i, i, i, p, p]
    return lib


def cut(lib, rows, lens, table_keys, tokens, least, most, unit, slots, window, min_units, few_units):
    rows, lens = (np.ascontiguousarray(a, np.int32) for a in (rows, lens))
    tiles, splits = np.zeros_like(rows), np.zeros_like(rows)
    lib.kv_items(rows.ctypes.data, lens.ctypes.data, len(rows), table_keys, tokens, least, most, unit, slots, window, min_units,
                 few_units, tiles.ctypes.data, splits.ctypes.data)
    return tiles.astype(np.int64), splits.astype(np.int64)


def lengths(rng, n, most):
    """Lengths over the whole range, alike or not, some of them no lengths at all."""
    kind = rng.integers(4)
    if kind == 0:
        return np.full(n, rng.integers(0, most + 1))
    out = np.exp(rng.uniform(0, np.log(most), n)).astype(np.int64)
    if kind == 2:
        out[rng.integers(n)] = most
    if kind == 3:
        out[rng.random(n) < 0.2] = rng.choice([0, -1, -2 ** 31, 2 ** 31 - 1])
    return out


def test_items_fit_what_the_host_sizes(items):
    rng = np.random.default_rng(81)
    cuts = joined = 0
    for _ in range(6000):
        wide = bool(rng.integers(2))
        tokens = int(rng.choice([1, 2, 3, 4, 8, 16] + ([32, 64, 128] if wide else [])))
        requests = int(rng.choice([1, 2, 3, 8, 63, 64, 65, 200]))
        q = np.exp(rng.uniform(0, np.log(rng.choice([2, 20, 400])), requests)).astype(np.int64) * (rng.random(requests) < 0.9)
        rows = np.append(q, rng.integers(0, 40))  # the padding is a run too
        pages = int(rng.choice([1, 7, 300, 8192]))
        table_keys = 16 * pages if rng.random() < 0.9 else 1 << 30
        lens = np.append(lengths(rng, requests, table_keys), 0)
        split = int(rng.choice([1, 2, 16, 64]))
        least, most = (split, NO_TILES) if wide else (1, split - 1 if split > 1 else NO_TILES)
        window = int(rng.choice([0, 0, 1, 100, 1024, 1 << 30]))
        slots = int(rng.choice([1, 2, 16, 32, 64, 256, 512]))
        total = int(rows.sum())
        bound = items.kv_most_tiles(total, requests + 1, tokens, least, most)
        if wide:
            unit, min_units, few_units = 32, 8, 8
        else:
            unit, min_units, few_units = 64, 4, 2
        tiles, splits = cut(items, rows, lens, table_keys, tokens, least, most, unit, slots, window, min_units, few_units)
        counted = (rows >= least) & (rows <= most)
        assert (tiles == np.where(counted, -(-rows // tokens), 0)).all()
        assert tiles.sum() <= bound, (tiles.sum(), bound)
        assert (splits >= 1).all()
        if bound < slots:  # else the host makes no cuts
            assert (tiles * splits).sum() <= slots + bound, (tiles, splits, slots, bound)
            cuts += 1
            joined += int((splits[tiles > 0] > 1).any())
    assert cuts > 1000 and joined > 300


def test_items_of_the_largest_batches(items):
    """Where the sums of units pass what a float counts exactly."""
    for slots in (1, 17, 256, 511):
        rows = np.full(slots - 1, 1) if slots > 1 else np.array([1])
        for lens in (np.full(len(rows), (1 << 30) - 1), np.arange(len(rows)) * 1000003 % (1 << 30) + 1):
            tiles, splits = cut(items, rows, lens, 1 << 30, 1, 1, NO_TILES, 32, slots, 0, 8, 8)
            assert (tiles * splits).sum() <= slots + len(rows)
