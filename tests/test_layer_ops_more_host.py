"""More of the adapters, norms and the gate without a GPU: their GPU tests of precision on the emulated build of the kernels."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EMU = os.path.join(ROOT, "tests", "emu")
sys.path.insert(0, EMU)

import build_emu  # noqa: E402

emulated = pytest.mark.skipif(not os.path.exists(build_emu.CXX), reason="host clang++ of the ROCm toolchain not found: the emulated build needs it")
FILES = ["tests/test_gpu_lora_parts.py"]


@emulated
def test_gpu_tests_pass_on_the_emulated_kernels():
    """The GPU tests of these files, run on the device code compiled for the host (tests/emu)."""
    build_emu.build()
    runs = [subprocess.Popen([sys.executable, os.path.join(EMU, "gpu_tests_on_emu.py"), f, "-k", "not graph and not stream and not long"], cwd=ROOT,
                             stdout=subprocess.PIPE, stderr=subprocess.STDOUT) for f in FILES]
    for f, p in zip(FILES, runs):
        log = p.communicate(timeout=900)[0].decode()
        assert p.returncode == 0, f + log[-3000:]
