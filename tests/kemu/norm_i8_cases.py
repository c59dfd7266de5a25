"""One case of tests/norm_i8_ref.py, norm_i8_limits.py or norm_i8_chain.py on the kernel emulator, in a process of its own (a fault in an emulated
kernel ends that process with the emulator's report):

    python tests/kemu/norm_i8_cases.py '<json: {"op": name, "orders": [...], ...parameters}>'
"""
from __future__ import annotations

import json
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
sys.path[:0] = [str(HERE.parent.parent), str(HERE.parent), str(HERE)]

import norm_i8_chain  # noqa: E402
import norm_i8_limits  # noqa: E402
import norm_i8_ref  # noqa: E402
from bwd_cases import Backend  # noqa: E402


def main(argv):
    spec = json.loads(argv[1])
    orders, op = spec.pop("orders"), spec.pop("op")
    be = Backend()
    from sdvk_amd import _lib
    _lib.load = lambda: be.E.lib  # sdvk_amd.ops on the emulated library
    for o in orders:
        be.E.order(o, bool(o))
        {**norm_i8_ref.OPS, **norm_i8_limits.OPS, **norm_i8_chain.OPS}[op](be, **spec)
        print(f"OK order {o}", flush=True)


if __name__ == "__main__":
    main(sys.argv)
