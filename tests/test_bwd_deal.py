"""The dealing of attention's backward work (blocks, shares and parts) on the host: tests/kemu/deal_check.cpp."""
from __future__ import annotations

import subprocess

from test_kemu_bwd import KEMU, emulator  # noqa: F401  (fixture)


def test_every_tile_once_and_every_part_written(emulator, tmp_path):  # noqa: F811
    import kemu_build

    exe = tmp_path / "deal_check"
    flags = [f for f in kemu_build.FLAGS if f != "-fPIC"]
    r = subprocess.run([kemu_build.CXX, *flags, "-I", str(kemu_build.OUT / "src"), "-I", str(KEMU / "include"), "-I", str(KEMU),
                        "-I", str(kemu_build.ROOT / "include"), str(KEMU / "deal_check.cpp"), "-o", str(exe), str(kemu_build.LIB),
                        f"-Wl,-rpath,{kemu_build.OUT}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout.startswith("OK "), (r.stdout + r.stderr)[-2000:]
    print(r.stdout)
