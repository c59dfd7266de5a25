"""The compiled 8-bit product and GroupNorm kernels (CPU: gfx950 assembly, analysed by tests/isa_sched.py).

A tile's K loop is a ring of two to four stages, one trip per round: a load is issued a round less a step ahead of the wait that
retires it. A wait that the compiler adds (an LDS read that it takes for one of a load's bytes) would drop that to nothing.
"""
from __future__ import annotations

import re
import shutil

import pytest

import isa_sched


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    from sdvk_amd import build as b

    if shutil.which(b.hipcc()) is None:
        pytest.skip("no hipcc for the gfx950 assembly")
    d = tmp_path_factory.mktemp("isa")
    return {src: isa_sched.compile_asm(src, d / (src + ".s")) for src in ("gemm_i8.hip", "groupnorm.hip")}


def test_ring_loops(asm):
    loops = [l for l in isa_sched.loops(asm["gemm_i8.hip"]) if "gemm_i8_tile_kernel" in l.kernel]
    assert len(loops) == 12  # six builds, two types of C
    for l in loops:
        stages = int(re.search(r"Li(\d+)EEEv", l.kernel).group(1))
        step = l.mfma // stages
        assert l.scratch == 0 and l.mfma == step * stages, l.kernel
        # (the last quarter of a step's products may be issued behind the next wait)
        assert l.min_distance >= (stages - 1) * step - step // 4, (l.kernel, l.distances)


@pytest.mark.parametrize("src", ["gemm_i8.hip", "groupnorm.hip"])
def test_resources(asm, src):
    for k in isa_sched.resources(asm[src]):
        assert k.scratch == 0, (k.kernel, k.scratch)  # (values past 256 registers lie in the other 256)
        assert k.lds <= 160 * 1024 and k.waves_per_simd * 4 * 64 >= k.max_threads, (k.kernel, k.lds, k.vgpr)
