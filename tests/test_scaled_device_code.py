"""Checks on the compiled gfx950 code of the attention over block-scaled pages and of the
sampling kernels (CPU only: hipcc cross-compiles).  The attention's are those of
test_attention_device_code.py, on the kernels that read scales."""

import re

import pytest

from helios_amd import build as hbuild
from test_attention_device_code import _vgprs
from test_device_code import _blocks, _check_dma_hazards, _dmas_in_flight_at_barriers, _kernel_meta, _kernels

DIMS = (64, 128, 256, 512)


@pytest.fixture(scope="module")
def scaled_asm():
    return hbuild.device_asm("kv_scaled.hip")


def test_dma_sgpr_hazards_covered(scaled_asm):
    kernels = list(_kernels(scaled_asm, "tile_kernel"))
    assert len(kernels) == len(DIMS)
    _check_dma_hazards(kernels)


@pytest.mark.parametrize("d", DIMS)
def test_k_has_landed_at_every_barrier(scaled_asm, d):
    assert _dmas_in_flight_at_barriers(scaled_asm, f"tile_kernelILi{d}ELb1E") == {}


@pytest.mark.parametrize("d", DIMS)
def test_steps_stay_in_registers(scaled_asm, d):
    steps = [ins for ins, _ in _blocks(scaled_asm, f"tile_kernelILi{d}ELb1E") if sum(i.startswith("v_mfma") for i in ins) >= d // 16]
    assert len(steps) >= 2  # an even and an odd tile's
    for ins in steps:
        assert not any(i.startswith("scratch_") for i in ins)


def test_products_in_asm_wait_for_their_operands(scaled_asm):
    (name, lines), = [k for k in _kernels(scaled_asm, "tile_kernelILi512ELb1E")]
    products = 0
    for i, line in enumerate(lines):
        if not re.match(r"v_mfma_f32_32x32x16_bf16 a\[", line):
            continue
        products += 1
        a, b = (_vgprs(t.strip(",")) for t in line.split()[2:4])
        waits, j = 0, i - 1
        while j >= 0 and waits < 2:
            op = lines[j].split()[0]
            if op == "s_nop":
                waits += int(lines[j].split()[1]) + 1
            elif not op.endswith(":"):
                if op.startswith("v_") and not op.startswith("v_mfma"):
                    written = set().union(*[_vgprs(t.strip(",")) for t in lines[j].split()[1:3 if "swap" in op else 2]])
                    assert not written & (a | b), f"{name}: {lines[j]!r} feeds {line!r}"
                waits += 1
            j -= 1
    assert products >= 2 * 32  # an even and an odd tile's


def test_register_and_lds_budgets(scaled_asm):
    """As the planner counts on: two workgroups of 16-row tiles per CU up to head_dim 256 and no
    scratch; two 128-row tiles up to 128, one of two waves per SIMD at 256."""
    seen = 0
    for m in re.finditer(r"- \.agpr_count:.*?\.group_segment_fixed_size:\s+(\d+).*?\.name:\s+\S+?(tile|rows16)_kernelILi(\d+)E\S*"
                         r".*?\.private_segment_fixed_size:\s+(\d+).*?\.vgpr_count:\s+(\d+)", scaled_asm, re.S):
        lds, kind, d, private, vgprs = int(m.group(1)), m.group(2), int(m.group(3)), int(m.group(4)), int(m.group(5))
        assert lds <= 160 * 1024
        if kind == "rows16":
            assert private == 0 and vgprs <= (512 if d == 512 else 256), (d, vgprs, private)
        elif d <= 256:
            assert private == 0 and vgprs <= 256 and (d == 256 or lds <= 80 * 1024), (d, vgprs, private, lds)
        seen += 1
    assert seen == 2 * len(DIMS)


@pytest.mark.parametrize("source", ["kv_scaled_append.hip", "kv_pool.hip", "verify.hip"])
def test_no_scratch(source):
    meta = list(_kernel_meta(hbuild.device_asm(source)))
    assert meta
    for name, vgprs, private in meta:
        assert private == 0 and vgprs <= 128, f"{name}: {vgprs} VGPRs, {private} bytes of scratch"
