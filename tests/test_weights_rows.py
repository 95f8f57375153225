"""Where the attention weights' chunk kernel reads its query rows, replayed on the CPU
from its plans and its own walk (tests/native/weights_rows.cpp): groups 1 to 128, cut
and whole units.  No GPU is used."""
import os
import subprocess

from gpu_offloading_amd import _lib
from gpu_offloading_amd.build import ARCH, CSRC, INCLUDE, LIB_DIR, hipcc

HERE = os.path.dirname(os.path.abspath(__file__))


def test_rows_are_read_within_their_unit(tmp_path):
    _lib.load()
    exe = str(tmp_path / "weights_rows")
    res = subprocess.run([hipcc(), "-x", "hip", "--cuda-host-only", f"--offload-arch={ARCH}", "-O2",
                          "-std=c++17", f"-I{INCLUDE}", f"-I{CSRC}",
                          os.path.join(HERE, "native", "weights_rows.cpp"), "-o", exe,
                          "-L" + LIB_DIR, "-l:libkvc.so", "-Wl,-rpath," + LIB_DIR],
                         capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
    res = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.startswith("ok "), (res.stdout, res.stderr[-2000:])
