"""One case of tests/bwd_ref.py or tests/bwd_block.py on the kernel emulator, in a process of its own (a fault in an emulated kernel ends
that process with the emulator's report):

    python tests/kemu/bwd_cases.py '<json: {"op": name, "orders": [...], ...parameters}>'
"""
from __future__ import annotations

import json
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
sys.path[:0] = [str(HERE.parent), str(HERE)]

import bwd_block  # noqa: E402
import bwd_ref  # noqa: E402
import emu as kemu  # noqa: E402


class Backend:
    """The C-ABI on guarded host buffers: the byte past a buffer's 16-byte-rounded end is on a PROT_NONE page."""

    def __init__(self):
        self.E = kemu.Emu()

    def buf(self, arr):
        return self.E.buf(arr)

    def get(self, b, dtype, n):
        return b.get(dtype, n)

    def at(self, b, byte):
        return b.ptr + byte

    def call(self, name, *args):
        self.E.call(name, *args)

    def value(self, name, *args):
        return getattr(self.E.lib, name)(*args)

    def tune(self, name, value):
        assert self.E.lib.mi_tuning_set(name.encode(), None if value is None else value.encode()) == 0


def main(argv):
    spec = json.loads(argv[1])
    orders, op = spec.pop("orders"), spec.pop("op")
    be = Backend()
    from sdvk_amd import _lib
    _lib.load = lambda: be.E.lib  # sdvk_amd.ops on the emulated library
    for o in orders:
        be.E.order(o, bool(o))
        {**bwd_ref.OPS, **bwd_block.OPS}[op](be, **spec)
        print(f"OK order {o}", flush=True)


if __name__ == "__main__":
    main(sys.argv)
