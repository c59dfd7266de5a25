"""GroupNorm, the quantiser and the 8-bit product on the GPU at the edges of their documentation: tests/norm_i8_limits.py."""
import json

import pytest

import norm_i8_limits
from sdvk_amd import ops
from test_gpu_bwd import Backend

pytestmark = pytest.mark.gpu


@pytest.fixture
def backend(gpu):
    ops.tuning_reset()
    return Backend(gpu)


ALL = [(op, c) for op in norm_i8_limits.OPS for c in norm_i8_limits.CASES.get(op, []) + norm_i8_limits.GPU_CASES.get(op, [])]


@pytest.mark.parametrize("op,case", ALL, ids=[f"{op}-{json.dumps(c)}" for op, c in ALL])
def test_limits(backend, op, case):
    print(op, json.dumps(case), flush=True)
    norm_i8_limits.OPS[op](backend, **case)
