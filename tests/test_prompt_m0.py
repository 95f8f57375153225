"""Build-time check of the prompt attention's and the attention weights' AMD
assembly (built here with hipcc): their direct-to-LDS loads take their LDS address from M0, which the inline
assembly writes and cannot declare clobbered (hipcc reserves M0).  So nothing the
compiler generates may use M0: every instruction naming M0 is one of the kernel's
own `s_mov_b32 m0, sN`, directly followed by a direct-to-LDS load, every such load
is directly preceded by one, and no instruction that reads M0 implicitly
appears."""
import os
import re
import subprocess

import pytest

from test_prefill_m0 import HIPCC, IMPLICIT_M0, LDS_DMA, ROOT, _instructions


@pytest.mark.skipif(not os.access(HIPCC, os.X_OK), reason="hipcc not available")
@pytest.mark.parametrize("source", ["prompt", "weights"])
def test_only_the_direct_lds_loads_use_m0(tmp_path, source):
    out = tmp_path / (source + ".s")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang",
                    "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "gpu_offloading_amd", "csrc"),
                    "--cuda-device-only", "-S",
                    os.path.join(ROOT, "gpu_offloading_amd", "csrc", source + ".hip"),
                    "-o", str(out)], check=True, capture_output=True)
    ins = list(_instructions(out.read_text()))
    set_m0 = re.compile(r"^s_mov_b32 m0, s\d+$")
    n_dma = 0
    for i, code in enumerate(ins):
        assert not IMPLICIT_M0.match(code), code
        if LDS_DMA.match(code):
            n_dma += 1
            assert i > 0 and set_m0.match(ins[i - 1]), (ins[i - 1], code)
        if re.search(r"\bm0\b", code):
            assert set_m0.match(code), code
            assert i + 1 < len(ins) and LDS_DMA.match(ins[i + 1]), (code, ins[i + 1:i + 2])
    assert n_dma > 0
