"""CPU checks of the block-scaled cache, the page pool and the sampling calls: every refusal of
the C ABI (pointers are checked, never followed), the structs' layout, the Python checks that
need no GPU, and the scales' arithmetic compiled for the host."""

import ctypes
import math
import os
import struct
import subprocess

import pytest

from helios_amd import attention as A
from helios_amd import build as hbuild
from helios_amd import paging, qmm, sampling
from test_attention_abi import BAD, NO, P, batch, heads, lib, pages, q_heads  # noqa: F401

HERE = os.path.dirname(os.path.abspath(__file__))
INF, NAN = float("inf"), float("nan")


def ref(s):
    return None if s is None else ctypes.byref(s)


# ------------------------------------------------------------------ block scales

def scales(**kw):
    f = dict(k_dev=P, v_dev=P, page_stride=8 * 4, head_stride=4, block=16)
    f.update(kw)
    return A._Scales(**f)


def e4m3(**kw):
    return pages(**{"dtype": 1, "page_size": 64, "page_stride": 8 * 64 * 256, "head_stride": 64 * 256, **kw})


def attention(lib, pg=None, sc=None, b=None):
    return lib.gemma4_kv_attention_scaled(ref(pg or e4m3()), ref(sc or scales()), ref(b or batch()), P, 4096, 16, 1.0, 0, P, 4096, None, None)


def append(lib, pg=None, sc=None, b=None, q=None, k=None, v=None):
    return lib.gemma4_kv_append_scaled(ref(pg or e4m3()), ref(sc or scales()), ref(b or batch()), ref(q), ref(k or heads()), ref(v or heads()), None, None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(k_dev=None), BAD, "non-null k and v scales"),
    (dict(v_dev=None), BAD, "non-null k and v scales"),
    (dict(block=0), NO, "block"),
    (dict(block=8), NO, "block"),
    (dict(block=48), NO, "block"),
    (dict(block=128), NO, "block"),
    (dict(block=512), NO, "block"),
    (dict(head_stride=3), BAD, "shorter than a page's blocks"),
    (dict(page_stride=3), BAD, "shorter than a page's blocks"),
    (dict(page_stride=(1 << 40) + 1), NO, "2^40"),
    (dict(head_stride=(1 << 40) + 1), NO, "2^40"),
])
def test_block_scales_are_checked(lib, kw, status, text):
    for call in (attention, append):
        assert call(lib, sc=scales(**kw)) == status
        assert text in qmm.last_error()


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=0), BAD, "E4M3"),
    (dict(dtype=7), BAD, "E4M3"),
    (dict(k_dev=None), BAD, "non-null k and v pages"),
    (dict(head_dim=96), NO, "head_dim"),
    (dict(page_size=8), NO, "page_size"),
    (dict(token_stride=260), BAD, "16 bytes"),
    (dict(num_pages=0), BAD, "num_pages"),
])
def test_scaled_pages_are_checked(lib, kw, status, text):
    for call in (attention, append):
        assert call(lib, pg=e4m3(**kw)) == status
        assert text in qmm.last_error()
        assert qmm.last_error().startswith("gemma4_kv_append_scaled" if call is append else "gemma4_kv_attention_scaled")


def test_scaled_calls_without_structs(lib):
    b, h = batch(), heads()
    assert lib.gemma4_kv_append_scaled(ref(e4m3()), None, ref(b), None, ref(h), ref(h), None, None) == BAD
    assert lib.gemma4_kv_append_scaled(None, ref(scales()), ref(b), None, ref(h), ref(h), None, None) == BAD
    assert lib.gemma4_kv_attention_scaled(ref(e4m3()), ref(scales()), None, P, 4096, 16, 1.0, 0, P, 4096, None, None) == BAD
    # the rest of the arguments as in the calls without scales
    assert append(lib, k=heads(count=4)) == BAD and "kv_heads" in qmm.last_error()
    assert append(lib, v=heads(eps=-1.0)) == BAD and "eps" in qmm.last_error()
    assert append(lib, q=q_heads(out_dev=None)) == BAD and "non-null" in qmm.last_error()
    assert append(lib, b=batch(requests=0)) == BAD and "requests" in qmm.last_error()
    # pages' own scales are not looked at
    assert append(lib, pg=e4m3(k_scale=NAN, v_scale=0.0), b=batch(tokens=0)) == 0
    assert attention(lib, pg=e4m3(k_scale=NAN, v_scale=0.0), b=batch(tokens=0)) == 0


def test_scaled_append_too_large_for_a_launch(lib):
    big = dict(tokens=(1 << 24) - 1, requests=1 << 20)
    assert append(lib, b=batch(**big)) == NO and "too large" in qmm.last_error()


@pytest.fixture(scope="module")
def scale():
    so = os.path.join(HERE, "_build", "libkvscale.so")
    src, dep = os.path.join(HERE, "kv_scale_host.cpp"), os.path.join(hbuild.CSRC, "kv_index.h")
    if not os.path.exists(so) or any(os.path.getmtime(d) > os.path.getmtime(so) for d in (src, dep)):
        os.makedirs(os.path.dirname(so), exist_ok=True)
        subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                        "-I", hbuild.CSRC, src, "-o", so], check=True, capture_output=True)
    return ctypes.CDLL(so)


def test_the_least_scale_that_holds_a_value(scale):
    f32 = lambda v: struct.unpack("f", struct.pack("f", v))[0]  # noqa: E731
    values = [m * 2.0 ** e for e in range(-149, 128) for m in (1.0, 1.25, 1.5, 1.75, f32(1.75000012), 1.99)]
    for v in [0.0, 448.0, f32(448.00003), 447.9999, f32(3.4028234663852886e38)] + [x for x in values if x < 3.5e38]:
        v = f32(v)
        byte = scale.kv_least_scale(struct.unpack("I", struct.pack("f", v))[0])
        assert 27 <= byte <= 207
        assert byte == 207 or v <= math.ldexp(448.0, byte - 127), v
        assert byte == 27 or v > math.ldexp(448.0, byte - 128), v
    assert [scale.kv_clamp_scale(b) for b in (0, 26, 27, 127, 207, 208, 255)] == [27, 27, 27, 127, 207, 207, 207]


# ------------------------------------------------------------------ the pool

def pool(**kw):
    f = dict(free_pages_dev=P, free_count_dev=P + 64, lens_dev=P + 128, block_tables_dev=P + 256, num_pages=10, page_size=64, requests=2,
             pages_per_request=4, table_stride=4)
    f.update(kw)
    return paging._Pool(**f)


def reserve(lib, p=None, new=P, starts=P, kv_lens=P, granted=P, rows=4, positions=P, slots=P):
    return lib.gemma4_kv_reserve(ref(p or pool()), new, starts, kv_lens, granted, rows, positions, slots, None)


def release(lib, p=None, lens=P, window=0):
    return lib.gemma4_kv_release(ref(p or pool()), lens, window, None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(free_pages_dev=None), BAD, "free_pages"),
    (dict(free_count_dev=None), BAD, "free_count"),
    (dict(lens_dev=None), BAD, "lens"),
    (dict(block_tables_dev=None), BAD, "block_tables"),
    (dict(lens_dev=P + 2), BAD, "4-byte"),
    (dict(page_size=8), NO, "page_size"),
    (dict(page_size=96), NO, "page_size"),
    (dict(num_pages=0), BAD, "num_pages"),
    (dict(num_pages=(1 << 30) + 1), BAD, "num_pages"),
    (dict(requests=0), BAD, "requests"),
    (dict(requests=(1 << 20) + 1), BAD, "requests"),
    (dict(pages_per_request=0), BAD, "pages_per_request"),
    (dict(table_stride=3), BAD, "table_stride"),
    (dict(table_stride=1 << 31), NO, "table_stride"),
    (dict(pages_per_request=(1 << 24) + 1, table_stride=(1 << 24) + 1), NO, "2^30"),
])
def test_pools_are_checked(lib, kw, status, text):
    for call in (reserve, release):
        assert call(lib, p=pool(**kw)) == status
        assert text in qmm.last_error()


@pytest.mark.parametrize("kw,status,text", [
    (dict(new=None), BAD, "new_tokens"),
    (dict(starts=None), BAD, "query_starts"),
    (dict(kv_lens=None), BAD, "kv_lens"),
    (dict(kv_lens=P + 128), BAD, "the pool's lens"),
    (dict(new=P + 1), BAD, "aligned"),
    (dict(granted=P + 2), BAD, "aligned"),
    (dict(positions=P + 1), BAD, "aligned"),
    (dict(slots=P + 4), BAD, "aligned"),
    (dict(rows=1 << 24), NO, "rows"),
])
def test_reserve_is_checked(lib, kw, status, text):
    assert reserve(lib, **kw) == status and text in qmm.last_error()
    assert lib.gemma4_kv_reserve(None, P, P, P, P, 0, None, None, None) == BAD


@pytest.mark.parametrize("kw,status,text", [
    (dict(lens=None), BAD, "lens"),
    (dict(lens=P + 1), BAD, "lens"),
    (dict(window=(1 << 30) + 1), NO, "window"),
])
def test_release_is_checked(lib, kw, status, text):
    assert release(lib, **kw) == status and text in qmm.last_error()
    assert lib.gemma4_kv_release(None, P, 0, None) == BAD


@pytest.mark.parametrize("kw", [dict(new=P + 4096), dict(new=P + 4096 + 8), dict(granted=P + 8192), dict(granted=P + 128), dict(positions=P + 4),
                                dict(slots=P + 256 + 24), dict(starts=P + 64), dict(positions=P + 32768 - 12)])
def test_reserve_writes_over_nothing(lib, kw):
    apart = dict(new=P + 12288, starts=P + 4096, kv_lens=P + 8192, granted=P + 16384, positions=P + 24576, slots=P + 32768)
    assert reserve(lib, **{**apart, **kw}) == BAD and "overlap" in qmm.last_error()


def test_release_reads_its_own_lens_only(lib):
    for lens in (P + 132, P + 124, P, P + 64, P + 256 + 28):
        assert release(lib, lens=lens) == BAD and "overlap" in qmm.last_error()
    assert release(lib, p=pool(free_count_dev=P + 36), lens=P + 4096) == BAD and "overlap" in qmm.last_error()


# ------------------------------------------------------------------ sampling

def logits(**kw):
    f = dict(x_dev=P, stride=1000, dtype=0, softcap=0.0)
    f.update(kw)
    return sampling._Logits(**f)


def sample(lib, of=None, rows=2, vocab=1000, u=P, heat=1.0, heats=None, out=P):
    return lib.gemma4_sample(ref(of or logits()), rows, vocab, u, heat, heats, out, None)


def verify(lib, of=None, draft=None, tokens=P, starts=P, requests=2, rows=4, vocab=1000, u=P, heat=1.0, heats=None, out=P, accepted=P):
    return lib.gemma4_verify_drafts(ref(of or logits()), ref(draft), tokens, starts, requests, rows, vocab, u, heat, heats, out, accepted, None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(of=logits(x_dev=None)), BAD, "non-null logits"),
    (dict(of=logits(x_dev=P + 1)), BAD, "aligned to their type"),
    (dict(of=logits(x_dev=P + 2, dtype=1)), BAD, "aligned to their type"),
    (dict(of=logits(dtype=2)), BAD, "BF16 or F32"),
    (dict(of=logits(stride=999)), BAD, "stride"),
    (dict(of=logits(stride=(1 << 40) + 1)), BAD, "stride"),
    (dict(of=logits(softcap=-1.0)), BAD, "softcap"),
    (dict(of=logits(softcap=NAN)), BAD, "softcap"),
    (dict(of=logits(softcap=INF)), BAD, "softcap"),
    (dict(vocab=0), NO, "vocab"),
    (dict(vocab=(1 << 24) + 1), NO, "vocab"),
    (dict(rows=(1 << 20) + 1), NO, "rows"),
    (dict(rows=1 << 20, vocab=1 << 24, of=logits(stride=1 << 24)), NO, "too large"),
    (dict(heat=-0.5), BAD, "temperature"),
    (dict(heat=NAN), BAD, "temperature"),
    (dict(heat=INF), BAD, "temperature"),
    (dict(u=None), BAD, "uniforms"),
    (dict(u=P + 2), BAD, "4-byte"),
    (dict(heats=P + 1), BAD, "4-byte"),
    (dict(out=None), BAD, "out_tokens"),
    (dict(out=P + 1), BAD, "4-byte"),
])
def test_sampling_is_checked(lib, kw, status, text):
    for call in (sample, verify):
        assert call(lib, **kw) == status
        assert text in qmm.last_error()
    assert sample(lib, rows=0) == 0 and verify(lib, rows=0) == 0


@pytest.mark.parametrize("kw,status,text", [
    (dict(tokens=None), BAD, "tokens"),
    (dict(starts=None), BAD, "query_starts"),
    (dict(accepted=None), BAD, "accepted"),
    (dict(tokens=P + 1), BAD, "4-byte"),
    (dict(starts=P + 2), BAD, "4-byte"),
    (dict(accepted=P + 2), BAD, "4-byte"),
    (dict(requests=0), BAD, "requests"),
    (dict(requests=(1 << 20) + 1), BAD, "requests"),
    (dict(draft=logits(x_dev=None)), BAD, "draft logits"),
    (dict(draft=logits(stride=10)), BAD, "draft logits"),
    (dict(draft=logits(dtype=1)), BAD, "one type"),
    (dict(draft=logits(softcap=-1.0)), BAD, "draft softcap"),
])
def test_verification_is_checked(lib, kw, status, text):
    assert verify(lib, **kw) == status and text in qmm.last_error()
    assert lib.gemma4_verify_drafts(None, None, P, P, 1, 1, 10, P, 1.0, None, P, P, None) == BAD


def test_tokens_are_written_over_nothing(lib):
    apart = dict(u=P + (1 << 20), heats=P + (2 << 20), out=P + (3 << 20))
    for kw in (dict(out=P + 3996), dict(out=P + (1 << 20) + 4), dict(out=P + (2 << 20) - 4)):
        assert sample(lib, **{**apart, **kw}) == BAD and "overlap" in qmm.last_error()
    apart.update(tokens=P + (4 << 20), starts=P + (5 << 20), accepted=P + (6 << 20), draft=logits(x_dev=P + (7 << 20)))
    for kw in (dict(out=P + (4 << 20)), dict(out=P + (5 << 20) + 8), dict(accepted=P + (3 << 20) + 12), dict(accepted=P + (1 << 20) + 28),
               dict(out=P + (7 << 20) + 7996), dict(accepted=P + (4 << 20) - 4)):
        assert verify(lib, **{**apart, **kw}) == BAD and "overlap" in qmm.last_error()


# ------------------------------------------------------------------ layout, Python's own checks

C_LAYOUT = r'''
#include "gemma4_qmm.h"
#include <stdio.h>
int main(void) {
    printf("%zu %zu %zu\n", sizeof(Gemma4KvScales), offsetof(Gemma4KvScales, page_stride), offsetof(Gemma4KvScales, block));
    printf("%zu %zu %zu\n", sizeof(Gemma4KvPool), offsetof(Gemma4KvPool, num_pages), offsetof(Gemma4KvPool, table_stride));
    printf("%zu %zu %zu\n", sizeof(Gemma4Logits), offsetof(Gemma4Logits, dtype), offsetof(Gemma4Logits, softcap));
}
'''


def test_struct_layout(tmp_path):
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text(C_LAYOUT)
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(hbuild.ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [tuple(map(int, line.split())) for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()]
    want = [(ctypes.sizeof(s), getattr(s, a).offset, getattr(s, b).offset) for s, a, b in
            ((A._Scales, "page_stride", "block"), (paging._Pool, "num_pages", "table_stride"), (sampling._Logits, "dtype", "softcap"))]
    assert got == want


def test_python_refuses_what_is_not_on_the_gpu():
    import torch

    ints, floats = torch.zeros(3, dtype=torch.int32), torch.zeros(2, 8)
    with pytest.raises(qmm.Gemma4Error, match="free_pages"):
        paging.PagePool(ints, ints, ints, ints.view(1, 3), 64)
    with pytest.raises(qmm.Gemma4Error, match="logits"):
        sampling.sample(floats, floats[:, 0])
    with pytest.raises(qmm.Gemma4Error, match="logits"):
        sampling.verify_drafts(floats, ints[:2], ints[:2], floats[:, :2])
    with pytest.raises(qmm.Gemma4Error, match="block scales"):
        A._block_scales(torch.zeros(1, 1, 1, dtype=torch.uint8), 1.0, torch.zeros(1, 1, 16, 64), 1, 2)


# ------------------------------------------------------------------ the sampling kernels' shares

@pytest.fixture(scope="module")
def shares():
    so = os.path.join(HERE, "_build", "libverifyindex.so")
    src, dep = os.path.join(HERE, "verify_index_host.cpp"), os.path.join(hbuild.CSRC, "verify_index.h")
    if not os.path.exists(so) or any(os.path.getmtime(d) > os.path.getmtime(so) for d in (src, dep)):
        os.makedirs(os.path.dirname(so), exist_ok=True)
        subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                        "-I", hbuild.CSRC, src, "-o", so], check=True, capture_output=True)
    return ctypes.CDLL(so)


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 31, 64, 240, 513, 4097])
@pytest.mark.parametrize("vocab", [1, 7, 2048, 2049, 6001, 50001, 262144])
def test_every_part_is_taken_once(shares, rows, vocab):
    """Of each row and of each request; waves past the last row take none."""
    import numpy as np

    parts = shares.verify_stats(rows, vocab, None)
    assert parts in (-(-vocab // 2048), -(-vocab // 512))
    seen = np.zeros((rows, parts), np.int32)
    assert shares.verify_stats(rows, vocab, ctypes.c_void_p(seen.ctypes.data)) == parts and (seen == 1).all()
    seen[:] = 0
    assert 1 <= shares.verify_rest(rows, parts, ctypes.c_void_p(seen.ctypes.data)) <= max(1, -(-256 // rows)) and (seen == 1).all()
