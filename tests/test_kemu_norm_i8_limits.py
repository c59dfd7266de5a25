"""CPU checks of GroupNorm, the quantiser and the 8-bit product at the edges of their documentation (tests/norm_i8_limits.py), on the
kernel emulator (tests/kemu), under two schedules as in tests/test_kemu_norm_i8.py."""
from __future__ import annotations

import re
import shutil

import pytest

import isa_sched
import norm_i8_limits
from bwd_ref import rng_of
from test_kemu_norm_i8 import ORDERS, check, emulator  # noqa: F401


@pytest.mark.parametrize("op", list(norm_i8_limits.CASES))
def test_limits_on_emulator(emulator, op):  # noqa: F811
    check([dict(op=op, orders=ORDERS, **c) for c in norm_i8_limits.CASES[op]])


@pytest.mark.parametrize("case", norm_i8_limits.CASES["codes"] + norm_i8_limits.GPU_CASES["codes"], ids=str)
def test_rows_tell_the_mistake(case):
    """Every row of the quantiser's cases has codes that the mistake it is made for gets wrong."""
    norm_i8_limits.rows_of(rng_of(11), case["rows"], case["cols"], case.get("typ", "f32"), case["kind"])


def test_product_rounds_to_fp32_first(tmp_path):
    """No fp16 result of the product is rounded from the fma itself (gfx950 assembly): the builds and their ways to store would differ."""
    from sdvk_amd import build as b

    if shutil.which(b.hipcc()) is None:
        pytest.skip("no hipcc for the gfx950 assembly")
    isa_sched.compile_asm("gemm_i8.hip", tmp_path / "gemm_i8.s")
    text = (tmp_path / "gemm_i8.s").read_text()
    assert "v_cvt_f16_f32" in text and not re.findall(r"v_fma_mix\w*_f16", text)
