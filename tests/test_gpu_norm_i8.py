"""GroupNorm, the quantiser and the 8-bit product on the GPU: the cases of tests/norm_i8_ref.py against 64-bit formulas."""
import json

import pytest

import norm_i8_ref
from sdvk_amd import ops
from test_gpu_bwd import Backend

pytestmark = pytest.mark.gpu


@pytest.fixture
def backend(gpu):
    ops.tuning_reset()
    return Backend(gpu)


ALL = [(op, c) for op in norm_i8_ref.CASES for c in norm_i8_ref.CASES[op] + norm_i8_ref.GPU_CASES.get(op, [])]


@pytest.mark.parametrize("op,case", ALL, ids=[f"{op}-{json.dumps(c)}" for op, c in ALL])
def test_operator(backend, op, case):
    print(op, json.dumps(case), flush=True)
    norm_i8_ref.OPS[op](backend, **case)
