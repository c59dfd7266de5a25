"""The backward operators on the GPU: the cases of tests/bwd_ref.py against 64-bit formulas."""
import json

import numpy as np
import pytest

import bwd_ref
from sdvk_amd import ops
from sdvk_amd._lib import call
from sdvk_amd.hip import DeviceBuffer, synchronize

pytestmark = pytest.mark.gpu


class Handle:
    def __init__(self, arr):
        self.b = DeviceBuffer.from_array(arr)
        self.ptr = self.b.value


class Backend:
    def __init__(self, lib):
        self.lib = lib

    def buf(self, arr):
        return Handle(np.ascontiguousarray(arr).reshape(-1))

    def get(self, h, dtype, n):
        synchronize()
        return h.b.download(dtype, n)

    def at(self, h, byte):
        return h.ptr + byte

    def call(self, name, *args):
        call(name, *args)

    def value(self, name, *args):
        return getattr(self.lib, name)(*args)

    def tune(self, name, value):
        ops.tuning_set(name, value)


@pytest.fixture
def backend(gpu):
    ops.tuning_reset()
    yield Backend(gpu)
    ops.tuning_reset()


ALL = [(op, c) for op in bwd_ref.CASES for c in bwd_ref.CASES[op] + bwd_ref.GPU_CASES.get(op, [])]


@pytest.mark.parametrize("op,case", ALL, ids=[f"{op}-{json.dumps(c)}" for op, c in ALL])
def test_backward(backend, op, case):
    print(op, json.dumps(case), flush=True)
    bwd_ref.OPS[op](backend, **case)
