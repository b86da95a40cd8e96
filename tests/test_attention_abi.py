"""CPU checks of the paged-cache calls: every refusal of the C ABI (pointers are checked,
never followed), the structs' layout, the Python checks that need no GPU, and the kernels'
index arithmetic (absent pages, clamped starts, key ranges, splits) compiled for the host."""

import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

from helios_amd import attention as A
from helios_amd import build as hbuild
from helios_amd import qmm

HERE = os.path.dirname(os.path.abspath(__file__))
P = 1 << 20  # a pointer-like value, 16-byte aligned; the calls under test refuse before use


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(hbuild.LIB_PATH):
        hbuild.build()
    return qmm.load_library()


def pages(**kw):
    f = dict(k_dev=P, v_dev=P, page_stride=8 * 16 * 256, token_stride=256, head_stride=16 * 256, num_pages=4, page_size=16,
             kv_heads=8, head_dim=256, dtype=0, k_scale=1.0, v_scale=1.0)
    f.update(kw)
    return A._Pages(**f)


def batch(**kw):
    f = dict(query_starts_dev=P, kv_lens_dev=P, block_tables_dev=P, requests=2, tokens=2, pages_per_request=4, table_stride=4)
    f.update(kw)
    return A._Batch(**f)


def heads(**kw):
    f = dict(x_dev=P, out_dev=None, weight_dev=None, x_stride=4096, out_stride=0, count=8, norm=1, eps=1e-6)
    f.update(kw)
    return A._Heads(**f)


def q_heads(**kw):
    return heads(**{"out_dev": P, "out_stride": 4096, "count": 16, **kw})


def attention(lib, pg=None, b=None, q=P, q_stride=4096, nq=16, scale=1.0, window=0, out=P, out_stride=4096, lse=None):
    return lib.gemma4_kv_attention(ctypes.byref(pg or pages()), ctypes.byref(b or batch()), q, q_stride, nq, scale, window,
                                   out, out_stride, lse, None)


def append(lib, pg=None, b=None, q=None, k=None, v=None, rope=None):
    ref = lambda s: None if s is None else ctypes.byref(s)  # noqa: E731
    return lib.gemma4_kv_append(ctypes.byref(pg or pages()), ctypes.byref(b or batch()), ref(q), ctypes.byref(k or heads()),
                                ctypes.byref(v or heads()), ref(rope), None)


BAD, NO = qmm.Status.INVALID_ARGUMENT, qmm.Status.UNSUPPORTED_CONFIG


@pytest.mark.parametrize("kw,status,text", [
    (dict(k_dev=None), BAD, "non-null k and v"),
    (dict(v_dev=None), BAD, "non-null k and v"),
    (dict(head_dim=96), NO, "head_dim"),
    (dict(head_dim=0), NO, "head_dim"),
    (dict(page_size=8), NO, "page_size"),
    (dict(page_size=48), NO, "page_size"),
    (dict(page_size=0), NO, "page_size"),
    (dict(page_size=1 << 17), NO, "page_size"),
    (dict(dtype=2), BAD, "dtype"),
    (dict(num_pages=0), BAD, "num_pages"),
    (dict(kv_heads=0), BAD, "kv_heads"),
    (dict(k_dev=P + 8), BAD, "16 bytes"),
    (dict(token_stride=260), BAD, "16 bytes"),
    (dict(token_stride=128), BAD, "shorter than head_dim"),
    (dict(head_stride=64), BAD, "shorter than head_dim"),
    (dict(page_stride=0), BAD, "shorter than head_dim"),
    (dict(token_stride=1 << 24), NO, "token_stride"),
    (dict(page_stride=1 << 41), NO, "2^40"),
    (dict(dtype=1, k_scale=0.0), BAD, "k_scale"),
    (dict(dtype=1, v_scale=float("nan")), BAD, "v_scale"),
    (dict(dtype=1, k_scale=float("inf")), BAD, "k_scale"),
    (dict(dtype=1, token_stride=264, head_stride=16 * 256), BAD, "16 bytes"),
])
def test_pages_are_checked(lib, kw, status, text):
    for call in (attention, append):
        assert call(lib, pg=pages(**kw)) == status
        assert text in qmm.last_error()


@pytest.mark.parametrize("kw,status,text", [
    (dict(query_starts_dev=None), BAD, "query_starts"),
    (dict(kv_lens_dev=None), BAD, "kv_lens"),
    (dict(block_tables_dev=None), BAD, "block_tables"),
    (dict(kv_lens_dev=P + 2), BAD, "4-byte"),
    (dict(requests=0), BAD, "requests"),
    (dict(requests=(1 << 20) + 1), BAD, "requests"),
    (dict(tokens=(1 << 24) + 1), NO, "tokens"),
    (dict(pages_per_request=0), BAD, "pages_per_request"),
    (dict(table_stride=3), BAD, "table_stride"),
    (dict(pages_per_request=(1 << 26) + 1, table_stride=(1 << 26) + 1), NO, "2^30"),
])
def test_batches_are_checked(lib, kw, status, text):
    for call in (attention, append):
        assert call(lib, b=batch(**kw)) == status
        assert text in qmm.last_error()


@pytest.mark.parametrize("kw,status,text", [
    (dict(nq=0), BAD, "q_heads"),
    (dict(nq=12), BAD, "q_heads"),
    (dict(scale=float("inf")), BAD, "scale"),
    (dict(scale=float("nan")), BAD, "scale"),
    (dict(window=(1 << 30) + 1), NO, "window"),
    (dict(q=None), BAD, "non-null q"),
    (dict(out=None), BAD, "non-null q"),
    (dict(q=P + 2), BAD, "16 bytes"),
    (dict(out=P + 8), BAD, "16 bytes"),
    (dict(lse=P + 1), BAD, "16 bytes"),
    (dict(q_stride=4095), BAD, "16 bytes"),
    (dict(q_stride=2048), BAD, "q_stride"),
    (dict(out_stride=2048), BAD, "out_stride"),
])
def test_attention_is_checked(lib, kw, status, text):
    assert attention(lib, **kw) == status
    assert text in qmm.last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(x_dev=None), "non-null"),
    (dict(x_dev=P + 8), "16 bytes"),
    (dict(weight_dev=P + 4), "16 bytes"),
    (dict(count=4), "kv_heads"),
    (dict(x_stride=1024), "stride"),
    (dict(x_stride=4097), "16 bytes"),
    (dict(norm=2), "norm"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(out_dev=P), "goes to the cache"),
])
def test_appended_heads_are_checked(lib, kw, text):
    assert append(lib, k=heads(**kw)) == BAD and text in qmm.last_error()
    assert append(lib, v=heads(**kw)) == BAD and text in qmm.last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(out_dev=None), "non-null"),
    (dict(out_dev=P + 8), "16 bytes"),
    (dict(out_stride=1024), "stride"),
    (dict(count=0), "count"),
])
def test_query_heads_are_checked(lib, kw, text):
    assert append(lib, q=q_heads(**kw)) == BAD and text in qmm.last_error()
    args = ctypes.byref(q_heads(**kw)), None, None, None, 3, 256, None
    assert lib.gemma4_qk_norm_rope(*args) == BAD and text in qmm.last_error()


@pytest.mark.parametrize("rope", [(P, 12, 128), (P, 136, 136), (P, 128, 120), (P, 64, 4), (P, 64, 200), (P, 64, 264),
                                  (P + 2, 64, 128), (None, 64, 128), (P, 8, 0)])
def test_rope_is_checked(lib, rope):
    r = A._Rope(*rope)
    assert append(lib, rope=r) == BAD and "rope" in qmm.last_error()
    assert lib.gemma4_qk_norm_rope(ctypes.byref(q_heads()), None, ctypes.byref(r), P, 3, 256, None) == BAD


def test_null_structs_and_empty_calls(lib):
    q, k = q_heads(), heads()
    b = ctypes.byref
    assert lib.gemma4_kv_attention(None, b(batch()), P, 4096, 16, 1.0, 0, P, 4096, None, None) == BAD
    assert lib.gemma4_kv_attention(b(pages()), None, P, 4096, 16, 1.0, 0, P, 4096, None, None) == BAD
    assert lib.gemma4_kv_append(None, b(batch()), None, b(k), b(k), None, None) == BAD
    assert lib.gemma4_kv_append(b(pages()), None, None, b(k), b(k), None, None) == BAD
    assert lib.gemma4_kv_append(b(pages()), b(batch()), None, None, b(k), None, None) == BAD
    assert lib.gemma4_kv_append(b(pages()), b(batch()), None, b(k), None, None, None) == BAD
    assert lib.gemma4_qk_norm_rope(None, None, None, None, 3, 256, None) == BAD
    assert lib.gemma4_qk_norm_rope(b(q), None, None, None, 3, 100, None) == NO
    assert lib.gemma4_qk_norm_rope(b(q), None, b(A._Rope(P, 64, 128)), None, 3, 256, None) == BAD
    assert "positions" in qmm.last_error()
    # nothing to do: no pointer is needed
    assert lib.gemma4_qk_norm_rope(b(q_heads(x_dev=None)), None, None, None, 0, 256, None) == qmm.Status.OK
    assert append(lib, b=batch(tokens=0), k=heads(x_dev=None)) == qmm.Status.OK
    assert attention(lib, b=batch(tokens=0), q=None, out=None) == qmm.Status.OK


def test_structs_match_the_header(tmp_path):
    names = {"Gemma4KvPages": A._Pages, "Gemma4KvBatch": A._Batch, "Gemma4Rope": A._Rope, "Gemma4Heads": A._Heads}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "gemma4_qmm.h"', "int main(void) {"]
    for c, py in names.items():
        lines.append(f'printf("{c} %zu", sizeof({c}));')
        lines += [f'printf(" %zu", offsetof({c}, {f}));' for f, _ in py._fields_]
        lines.append('printf("\\n");')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.join(hbuild.ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    said = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, (c, py) in zip(said, names.items()):
        assert line.split()[0] == c
        assert [int(v) for v in line.split()[1:]] == [ctypes.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_]


def test_python_refuses_host_tensors():
    import torch

    t = torch.zeros(4, 8, 256, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: A.qk_norm_rope(t, None, i), lambda: A.Rope(torch.zeros(8)), lambda: A.HeadNorm(torch.ones(256).bfloat16()),
                 lambda: A.KVBatch(i, i, i), lambda: A.PagedKVCache(t[None], t[None])):
        with pytest.raises(qmm.Gemma4Error) as e:
            call()
        assert e.value.status == BAD


# ------------------------------------------------------------------ index arithmetic

@pytest.fixture(scope="module")
def index():
    so = os.path.join(HERE, "_build", "libkvindex.so")
    src, dep = os.path.join(HERE, "kv_index_host.cpp"), os.path.join(hbuild.CSRC, "kv_index.h")
    if not os.path.exists(so) or any(os.path.getmtime(d) > os.path.getmtime(so) for d in (src, dep)):
        os.makedirs(os.path.dirname(so), exist_ok=True)
        subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                        "-I", hbuild.CSRC, src, "-o", so], check=True, capture_output=True)
    lib = ctypes.CDLL(so)
    i, p = ctypes.c_int, ctypes.c_void_p
    lib.kv_page_at.argtypes = [p, i, i, i]
    lib.kv_run_bound.argtypes = [p, i, i, i]
    lib.kv_visible.argtypes = lib.kv_split.argtypes = [i, i, i, i, p]
    return lib


def test_absent_pages(index):
    table = np.array([0, 3, -1, 4, 5, -2 ** 31, 2 ** 31 - 1, 2], np.int32)
    got = [index.kv_page_at(table.ctypes.data, at, 8, 5) for at in range(-3, 12)]
    # before the table, its entries (only 0..4 are pages of the cache), past it
    assert got == [-1, -1, -1, 0, 3, -1, 4, -1, -1, -1, 2, -1, -1, -1, -1]


def test_starts_are_clamped(index):
    starts = np.array([0, 5, 900, -7, 12], np.int32)
    got = [index.kv_run_bound(starts.ctypes.data, r, 4, 10) for r in range(6)]
    assert got == [0, 5, 10, 0, 10, 10]


def test_visible_keys_and_full_groups(index):
    rng = np.random.default_rng(3)
    out = (ctypes.c_int * 2)()
    for _ in range(400):
        kv, n = int(rng.integers(0, 80)), int(rng.integers(1, 20))
        window = int(rng.choice([0, 1, 2, 7, 16, 33, 1000]))
        pos0 = kv - int(rng.integers(1, 40))
        rows = range(pos0, pos0 + n)
        seen = [[j <= p and j < kv and (not window or j > p - window) for j in range(120)] for p in rows]
        some = [j for j in range(120) if any(s[j] for s in seen)]
        index.kv_visible(pos0, n, kv, window, out)
        if some:
            assert (out[0], out[1]) == (some[0], some[-1] + 1)
        else:
            assert out[0] >= out[1]
        last = pos0 + n - 1 < kv
        for key in range(0, 96, 16):
            if last:  # the kernels' rows are tokens of the cache
                assert bool(index.kv_all_visible(key, 16, pos0, n, window)) == all(all(s[key:key + 16]) for s in seen)


def test_splits_cover_every_tile_once(index):
    out = (ctypes.c_int * 2)()
    for tiles in list(range(0, 40)) + [100, 255, 1000]:
        for splits in (1, 2, 3, 7, 64, 128):
            for least in (1, 4, 8):
                at, used = 0, 0
                for s in range(splits):
                    index.kv_split(tiles, s, splits, least, out)
                    if out[1] > out[0]:
                        assert out[0] == at
                        at, used = out[1], used + 1
                assert at == tiles and used <= max(1, -(-tiles // least))


def test_header_says_what_the_library_has(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(hbuild.ROOT, "include", "gemma4_qmm.h")).read(), flags=re.S)
    for name in ("gemma4_qk_norm_rope", "gemma4_kv_append", "gemma4_kv_attention"):
        assert re.search(rf"Gemma4Status {name}\(", text) and hasattr(lib, name)


@pytest.mark.parametrize("tokens,requests,kv_heads,text", [
    (1 << 24, 1, 8, "2^24"),                      # tokens
    ((1 << 24) - 1, 1, 256, "2^31"),              # rows of q
    (1 << 20, 1 << 20, 16, "one launch"),         # a tile per request and KV head
])
def test_launches_too_large_are_refused(lib, tokens, requests, kv_heads, text):
    b = batch(tokens=tokens, requests=requests)
    pg = pages(kv_heads=kv_heads, page_stride=kv_heads * 16 * 256)
    assert attention(lib, pg=pg, b=b, nq=kv_heads, q_stride=kv_heads * 256, out_stride=kv_heads * 256) == NO
    assert text in qmm.last_error()
    if tokens >= 1 << 24:
        assert append(lib, pg=pg, b=b) == NO
        assert lib.gemma4_qk_norm_rope(ctypes.byref(q_heads()), None, None, None, tokens, 256, None) == NO
        assert text in qmm.last_error()


def test_the_attention_kernel_setting(lib):
    assert A.set_attention_kernel(2) == 0 and lib.gemma4_kv_set_attention_kernel(7) == 2  # 7 is taken as 0
    assert A.set_attention_kernel(0) == 0
    for bad in (-1, 3):
        with pytest.raises(ValueError):
            A.set_attention_kernel(bad)
