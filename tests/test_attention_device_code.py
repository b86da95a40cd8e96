"""Checks on the attention kernels' compiled gfx950 code (CPU only: hipcc cross-compiles).

The 128-row tile orders its LDS DMAs and its waits itself: every DMA a wave issued must have
landed at the barrier before other waves read the tile, its scalar operands must not come
from a VALU write within the hazard window, and its step must hold everything in registers
(a reload from scratch would wait for the loads of V, and count among them)."""

import re

import pytest

from helios_amd import build as hbuild
from test_device_code import _blocks, _check_dma_hazards, _dmas_in_flight_at_barriers, _kernel_meta, _kernels

TILES = [(d, f) for d in (64, 128, 256, 512) for f in (0, 1)]


@pytest.fixture(scope="module")
def tile_asm():
    return hbuild.device_asm("kv_tile.hip")


def test_tile_dma_sgpr_hazards_covered(tile_asm):
    kernels = list(_kernels(tile_asm, "tile_kernel"))
    assert len(kernels) == len(TILES)
    _check_dma_hazards(kernels)


@pytest.mark.parametrize("d,fp8", TILES)
def test_tile_k_has_landed_at_every_barrier(tile_asm, d, fp8):
    assert _dmas_in_flight_at_barriers(tile_asm, f"tile_kernelILi{d}ELb{fp8}E") == {}


@pytest.mark.parametrize("d,fp8", TILES)
def test_tile_steps_stay_in_registers(tile_asm, d, fp8):
    steps = [ins for ins, _ in _blocks(tile_asm, f"tile_kernelILi{d}ELb{fp8}E") if sum(i.startswith("v_mfma") for i in ins) >= d // 16]
    assert len(steps) >= 2  # an even and an odd tile's
    for ins in steps:
        assert not any(i.startswith("scratch_") for i in ins)
        assert any(" lds" in i for i in ins) or not any("a[" in i for i in ins if i.startswith("v_mfma"))


def _vgprs(tok: str):
    m = re.match(r"v\[(\d+):(\d+)\]$", tok)
    if m:
        return set(range(int(m.group(1)), int(m.group(2)) + 1))
    m = re.match(r"v(\d+)$", tok)
    return {int(m.group(1))} if m else set()


@pytest.mark.parametrize("fp8", [0, 1])
def test_products_in_asm_wait_for_their_operands(tile_asm, fp8):
    """The products with accumulators in AGPRs are asm, which the compiler's hazard recognizer
    cannot see into: no VALU write of an operand within two wait states before one."""
    (name, lines), = [k for k in _kernels(tile_asm, f"tile_kernelILi512ELb{fp8}E")]
    products = 0
    for i, line in enumerate(lines):
        if not re.match(r"v_mfma_f32_32x32x16_bf16 a\[", line):
            continue
        products += 1
        a, b = (_vgprs(t.strip(",")) for t in line.split()[2:4])
        assert len(a) == 4 and len(b) == 4, line
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


def test_attention_register_and_lds_budgets(tile_asm):
    """The 16-row kernel: no scratch, two workgroups of four waves per CU up to head_dim 256
    (256 VGPRs), as the planner counts on; every tile fits the CU's LDS."""
    meta = [(n, v, p) for n, v, p in _kernel_meta(hbuild.device_asm("kv_attention.hip")) if "rows16_kernel" in n]
    assert len(meta) == 8
    for name, vgprs, private in meta:
        assert private == 0, f"{name} spills to scratch"
        assert vgprs <= (512 if "ILi512E" in name else 256), f"{name}: {vgprs} VGPRs"
    lds = [int(v) for v in re.findall(r"\.group_segment_fixed_size:\s+(\d+)", tile_asm)]
    assert len(lds) >= len(TILES) and max(lds) <= 160 * 1024
    for name, vgprs, private in _kernel_meta(hbuild.device_asm("kv_heads.hip")):
        assert private == 0 and vgprs <= 80, f"{name}: {vgprs} VGPRs"


def test_two_tiles_of_small_heads_share_a_cu(tile_asm):
    """The planner counts on it: at most 256 VGPRs and half of the LDS up to head_dim 128; one
    workgroup of two waves per SIMD at 256."""
    seen = 0
    for m in re.finditer(r"- \.agpr_count:.*?\.group_segment_fixed_size:\s+(\d+).*?\.name:\s+\S+tile_kernelILi(\d+)E.*?\.vgpr_count:\s+(\d+)",
                         tile_asm, re.S):
        lds, d, vgprs = (int(m.group(i)) for i in (1, 2, 3))
        if d <= 256:
            assert vgprs <= 256, (d, vgprs)
        if d <= 128:
            assert lds <= 80 * 1024, (d, lds)
        seen += 1
    assert seen == len(TILES)
