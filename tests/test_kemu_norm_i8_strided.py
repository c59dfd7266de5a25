"""CPU checks of GroupNorm, the quantiser and the 8-bit product where a launch has fewer workgroups than units, so that workgroups stride:
on the GPU that takes more than 2^20 units, or 2^23 tiles of every build; here a copy of the sources has both limits at three."""
from __future__ import annotations

import json
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

import norm_i8_ref
from test_kemu_norm_i8 import KEMU, ORDERS, check, emulator  # noqa: F401

CSRC = KEMU.parent.parent / "sdvk_amd" / "csrc"
LIMITS = {"constexpr uint32_t kMaxGrid = 1u << 20;": "constexpr uint32_t kMaxGrid = 3;", "tiles(b) < (1u << 23)": "tiles(b) < 3u"}


@pytest.fixture(scope="module")
def few(emulator, tmp_path_factory):  # noqa: F811
    """The emulator with those limits, for the processes that the tests start."""
    d = tmp_path_factory.mktemp("few")
    shutil.copytree(CSRC, d / "csrc")
    found = []
    for name in ("groupnorm.hip", "gemm_i8.hip"):
        text = (d / "csrc" / name).read_text()
        for a, b in LIMITS.items():
            found += [a] * text.count(a)
            text = text.replace(a, b)
        (d / "csrc" / name).write_text(text)
    assert sorted(found) == sorted([*LIMITS, "constexpr uint32_t kMaxGrid = 1u << 20;"])
    env = {"KEMU_CSRC": str(d / "csrc"), "KEMU_OUT": str(d / "out")}
    subprocess.run([sys.executable, str(KEMU / "kemu_build.py")], env={**os.environ, **env}, check=True, capture_output=True, timeout=900)
    with pytest.MonkeyPatch.context() as m:
        for k, v in env.items():
            m.setenv(k, v)
        yield


@pytest.mark.parametrize("op", ["groupnorm", "groupnorm_bwd", "quantize", "product"])
def test_strided_on_emulator(few, op):
    check([dict(op=op, orders=ORDERS, **c) for c in norm_i8_ref.CASES[op]])


LAST = """import json, sys
sys.path[:0] = json.loads(sys.argv[1])
import norm_i8_ref
from bwd_cases import Backend
be = Backend()
norm_i8_ref.OPS[sys.argv[2]](be, **json.loads(sys.argv[3]))
kernel, grid = be.E.last_launch()
print(kernel, grid[0])
"""


@pytest.mark.parametrize("op,case,kernel", [
    ("groupnorm", dict(P=300, C=64, G=32, yoff=1), "gn_apply_any_kernel"), ("groupnorm_bwd", dict(P=19, C=640, G=8, gap=3), "gn_bwd_apply_any_kernel"),
    ("quantize", dict(rows=20, cols=37), "quantize_rows_any_kernel"), ("quantize", dict(rows=9, cols=2048), "quantize_rows_kernel"),
    # aligned, and more tiles than any build may have
    ("product", dict(M=800, N=700, K=16), "gemm_i8_any_kernel")])
def test_grids_are_few(few, op, case, kernel):
    """The limits are in force: a call's last launch is a kernel that strides, of three workgroups."""
    paths = [str(p) for p in (KEMU.parent.parent, KEMU.parent, KEMU)]
    r = subprocess.run([sys.executable, "-c", LAST, json.dumps(paths), op, json.dumps(case)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert kernel in r.stdout and r.stdout.split()[-1] == "3", r.stdout
