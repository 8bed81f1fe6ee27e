"""CPU checks of the compiled kernels of differential attention, RMS norm and
dropout (no GPU): no scratch memory and no spills, and the registers that leave
the waves a SIMD which their launch bounds and comments count on."""

from __future__ import annotations

import re

import pytest

from tests import isa

SOURCES = ["fjx_diffattn.hip", "fjx_diffattn_bwd.hip", "fjx_rmsnorm.hip", "fjx_dropout.hip"]


def metadata(src):
    meta, name = {}, None
    for line in isa.assembly(src):
        m = re.match(r"\s*\.(name|private_segment_fixed_size|vgpr_spill_count|sgpr_spill_count|vgpr_count):\s+(\S+)", line)
        if m and m.group(1) == "name":
            name = m.group(2)
        elif m and name:
            meta.setdefault(name, {})[m.group(1)] = int(m.group(2))
    return {n: m for n, m in meta.items() if "vgpr_count" in m}


@pytest.fixture(scope="module")
def resources():
    return {src: metadata(src) for src in SOURCES}


@pytest.mark.parametrize("src", SOURCES)
def test_no_scratch_and_no_spills(resources, src):
    assert resources[src]
    for name, m in resources[src].items():
        assert m["private_segment_fixed_size"] == 0 and m["vgpr_spill_count"] == 0, (name, m)


def test_waves_a_simd_of_the_attention(resources):
    """bf16 at 32 channels: three waves a SIMD forward (170 registers a lane of
    512), two in the backward kernels (256)."""
    found = 0
    for src, most in (("fjx_diffattn.hip", 170), ("fjx_diffattn_bwd.hip", 256)):
        for name, m in resources[src].items():
            if re.search(r"(fwd|dq|dkv|dbias)_kernelI", name) and "DF16bLi32E" in name:
                found += 1
                assert m["vgpr_count"] <= most, (name, m)
    assert found == 2 + 2 + 6 + 1
