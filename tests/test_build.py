"""What the built library holds: no packed fp32 arithmetic (build.py compiles without it; some of its forms have given wrong results on gfx950)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")
def test_no_packed_fp32_instructions_in_the_library(tmp_path):
    lib = str(tmp_path / "libgsx.so")
    shutil.copy(os.path.join(ROOT, "gaussian-splatting-cuda_amd", "libgsx.so"), lib)
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)   # one code object for each source, beside the copy
    objects = sorted(f for f in os.listdir(tmp_path) if f.endswith("gfx950"))
    from importlib import import_module
    assert len(objects) >= len(import_module("gaussian-splatting-cuda_amd.build").HIP_SOURCES) - 1   # (gsx_capi.hip has no kernel)
    packed, seen = re.compile(r"\bv_pk_(add|mul|fma)_f32\b"), 0
    for f in objects:
        p = subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(tmp_path / f)], stdout=subprocess.PIPE, text=True)
        for line in p.stdout:
            seen += "v_fma_f32" in line
            assert not packed.search(line), "%s: %s" % (f, line.strip())
        assert p.wait() == 0
    assert seen > 1000   # (the listing is one of kernels)
