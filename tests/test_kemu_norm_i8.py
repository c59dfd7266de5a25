"""CPU checks of the GroupNorm, quantiser and 8-bit product kernels on the kernel emulator (tests/kemu): the cases of
tests/norm_i8_ref.py against 64-bit formulas, on guarded buffers, under two schedules (one wave operation per wave per pass;
wave-major with lanes, waves and workgroups reversed, so a missing barrier changes the result under one of them)."""
from __future__ import annotations

import json
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest

import norm_i8_chain
import norm_i8_ref

KEMU = Path(__file__).resolve().parent / "kemu"
ORDERS = [0, 7]


@pytest.fixture(scope="module")
def emulator():
    if not Path(os.environ.get("KEMU_CXX", "/opt/rocm/llvm/bin/clang++")).exists():
        pytest.skip("no host clang++ for the emulation build")
    sys.path.insert(0, str(KEMU))
    import kemu_build

    return kemu_build.build()


def run(spec):
    return subprocess.run([sys.executable, str(KEMU / "norm_i8_cases.py"), json.dumps(spec)], capture_output=True, text=True, timeout=900)


def check(specs):
    with ThreadPoolExecutor(max(1, min(8, os.cpu_count() or 1))) as ex:
        results = list(ex.map(run, specs))
    failed = [f"{json.dumps(s)}\n{(r.stdout + r.stderr).strip()[-1200:]}" for s, r in zip(specs, results)
              if r.returncode != 0 or r.stdout.count("OK ") != len(ORDERS)]
    assert not failed, "\n\n".join(failed)


@pytest.mark.parametrize("op", list(norm_i8_ref.CASES))
def test_kernels_on_emulator(emulator, op):
    check([dict(op=op, orders=ORDERS, **c) for c in norm_i8_ref.CASES[op]])


def test_chain_on_emulator(emulator):
    """The operators run together, around each other and the existing ones."""
    check([dict(op=op, orders=ORDERS) for op in norm_i8_chain.OPS])
