"""The float32 tiles of the adapters as the compiler makes them (no GPU needed: hipcc cross-compiles): nothing in scratch memory, and no run of memory
instructions in front of the products of a slice."""
import os
import re
import shutil
import subprocess

import pytest

from scattermoe_amd import _build

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")


def test_memory_instructions_stand_between_products(tmp_path):
    out = tmp_path / "adapters_f32.s"
    subprocess.run([_build._hipcc()] + _build.HIPCC_FLAGS + ["--cuda-device-only", "-S", "-o", str(out), os.path.join(_build.CSRC, "adapters_f32.hip")],
                   check=True, stderr=subprocess.DEVNULL)
    text = out.read_text()
    kernels = re.findall(r"^(_ZN4smoe\d+adapter_(?:tiles|runs)_f32_kernel\w+):(.*?)^\.Lfunc_end", text, re.S | re.M)
    assert len(kernels) == 6
    for name, body in kernels:
        assert "scratch_" not in body, name
        loops = [b for b in re.split(r"^\.LBB\w+:", body, flags=re.M) if b.count("v_mfma") >= 16 and "s_barrier" in b]
        assert loops, name
        for loop in loops:
            ops = re.findall(r"v_mfma|ds_read|ds_write|global_load", loop)
            first, last = ops.index("v_mfma"), len(ops) - 1 - ops[::-1].index("v_mfma")
            run = longest = 0
            for op in ops[first:last]:
                run = 0 if op == "v_mfma" else run + 1
                longest = max(longest, run)
            assert longest <= 4, (name, longest)
