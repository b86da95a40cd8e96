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
