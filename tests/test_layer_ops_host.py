"""The adapters, norms and the gate without a GPU: what the C ABI refuses before any launch, what the entry functions refuse on
their arguments alone, and their GPU tests on the emulated build of the kernels (also against guard pages)."""
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EMU = os.path.join(ROOT, "tests", "emu")
sys.path.insert(0, EMU)

import build_emu  # noqa: E402

EINVAL, ESHAPE, EALIGN, EUNSUPPORTED = -1, -2, -3, -4
P = 4096  # an address that is never reached


def test_c_abi_refusals_of_the_gate(lib):
    f = lib.moe_gg_route_gate
    assert f(P, 2, -1, 8, 2, 0, 1, 1.0, P, P, None) == EINVAL
    assert f(P, 3, 4, 8, 2, 0, 1, 1.0, P, P, None) == EINVAL
    assert f(P, 2, 4, 8, 2, 2, 1, 1.0, P, P, None) == EINVAL
    assert f(P, 2, 4, 8, 9, 0, 1, 1.0, P, P, None) == ESHAPE
    assert f(P, 2, 4, 769, 2, 0, 1, 1.0, P, P, None) == EUNSUPPORTED
    assert f(P, 2, 4, 100, 65, 0, 1, 1.0, P, P, None) == EUNSUPPORTED
    assert f(P, 2, (1 << 24) + 1, 8, 2, 0, 1, 1.0, P, P, None) == EUNSUPPORTED
    assert f(None, 2, 4, 8, 2, 0, 1, 1.0, P, P, None) == EINVAL and f(P, 2, 4, 8, 2, 0, 1, 1.0, None, P, None) == EINVAL
    assert f(P + 2, 2, 4, 8, 2, 0, 1, 1.0, P, P, None) == EALIGN
    assert f(None, 2, 0, 8, 2, 0, 1, 1.0, None, None, None) == 0
    b = lib.moe_gg_route_gate_backward
    assert b(P, P, 2, P, 4, 8, 9, 0, 1, 1.0, P, None) == ESHAPE
    assert b(P, P, 2, None, 4, 8, 2, 0, 1, 1.0, P, None) == EINVAL
    assert b(P, P, 0, P, 4, 8, 2, 0, 1, 1.0, P + 1, None) == EALIGN
    assert b(None, None, 2, None, 0, 8, 2, 0, 1, 1.0, None, None) == 0


def norm(lib, y=P, ldy=64, res=P, ldr=64, post=P, gate=P, kind=1, pre=P, alpha=1.0, h=P, z=P, T=4, d=64, dtype=0, stream=0, weights=0):
    return lib.moe_gg_block_norm(y, ldy, res, ldr, post, gate, kind, pre, alpha, 1.0, 1e-6, h, z, T, d, dtype, stream, weights, None)


def test_c_abi_refusals_of_the_norms(lib):
    assert norm(lib, T=-1) == EINVAL and norm(lib, dtype=2) == EINVAL and norm(lib, stream=1) == EINVAL and norm(lib, weights=1) == EINVAL and norm(lib, kind=3) == EINVAL
    assert norm(lib, d=16385) == EUNSUPPORTED and norm(lib, T=(1 << 21) + 1) == EUNSUPPORTED
    assert norm(lib, ldy=63) == ESHAPE and norm(lib, ldr=63) == ESHAPE
    for absent in ("res", "h", "z", "gate"):
        assert norm(lib, **{absent: None}) == EINVAL
    assert norm(lib, kind=0) == EINVAL                       # a gate without its kind
    assert norm(lib, y=None, h=None, post=None, gate=None, kind=0, alpha=2.0) == EINVAL  # the norm alone does not scale
    assert norm(lib, y=None, post=None, gate=None, kind=0) == EINVAL                   # nor writes a stream
    assert norm(lib, y=P + 1) == EALIGN and norm(lib, stream=2, h=P + 2) == EALIGN and norm(lib, weights=2, pre=P + 2) == EALIGN
    assert norm(lib, T=0, y=None, res=None) == 0
    ws = lib.moe_gg_block_norm_backward_workspace(4, 64)
    assert ws >= 3 * 4 * 64 * 4

    def back(gh=P, gz=P, y=P, h=P, post=P, gate=P, kind=1, pre=P, gy=P, gres=P, gpost=P, ggate=P, gpre=P, T=4, work=P, nbytes=ws):
        return lib.moe_gg_block_norm_backward(gh, 64, gz, 64, y, 64, h, 64, post, gate, kind, pre, 1.0, 1.0, 1e-6, gy, gres, gpost, ggate, gpre, T, 64, 0, 0, 0,
                                              work, nbytes, None)
    for absent in ("gz", "gy", "gres", "h", "gpost", "ggate", "gpre", "work", "y"):
        assert back(**{absent: None}) == EINVAL, absent
    assert back(nbytes=ws - 1) == EINVAL and back(work=P + 16) == EALIGN


def test_c_abi_refusals_of_the_adapters(lib):
    ws = lib.moe_gg_lora_add_workspace(600, 2, 16, 24, 4)
    assert ws > 0 and lib.moe_gg_lora_add_workspace(600, 2, 16, 24, 129) == 0 and lib.moe_gg_lora_add_workspace(6, 2, 16, 24, 4) == 0

    def add(y=P, ldy=24, x=P, ldx=16, a=P, b=P, scales=None, perm=P, offsets=P, L=2, T=600, K=16, N=24, R=4, out=P, ldo=24, h=None, dtype=0, work=P, nbytes=ws):
        return lib.moe_gg_lora_add(y, ldy, x, ldx, a, b, scales, perm, offsets, L, T, K, N, R, out, ldo, h, dtype, work, nbytes, None)
    for absent in ("y", "x", "a", "b", "perm", "offsets", "out", "work"):
        assert add(**{absent: None}) == EINVAL, absent
    assert add(T=-1) == EINVAL and add(dtype=2) == EINVAL and add(nbytes=ws - 1) == EINVAL
    assert add(ldy=23, ldo=23) == ESHAPE and add(ldx=15) == ESHAPE and add(ldo=32) == ESHAPE and add(R=0) == ESHAPE and add(K=0) == ESHAPE
    for big in (dict(R=129), dict(L=768), dict(T=(1 << 20) + 1), dict(K=(1 << 17) + 1), dict(N=(1 << 17) + 1)):
        assert add(**big) == EUNSUPPORTED
    assert add(x=P + 1) == EALIGN and add(work=P + 8) == EALIGN and add(scales=P + 2) == EALIGN
    assert add(T=0, y=None) == 0
    wb = lib.moe_gg_lora_backward_workspace(600, 2, 16, 24, 4, 0)

    def back(go=P, ldg=24, x=P, ldx=16, perm=P, offsets=P, h=None, gin=None, ld_in=16, gx=P, ld_gx=16, ga=P, gb=P, work=P, nbytes=wb):
        return lib.moe_gg_lora_backward(go, ldg, x, ldx, P, P, None, perm, offsets, 2, 600, 16, 24, 4, h, gin, ld_in, gx, ld_gx, ga, gb, 0, work, nbytes, None)
    for absent in ("go", "x", "perm", "offsets", "gx", "ga", "gb", "work"):
        assert back(**{absent: None}) == EINVAL, absent
    assert back(ldg=23) == ESHAPE and back(gin=P, ld_in=15) == ESHAPE and back(gin=P, ld_in=24) == ESHAPE and back(nbytes=wb - 1) == EINVAL
    p = lib.moe_gg_lora_plan
    assert p(P, 4, 768, P, P, P, None) == EUNSUPPORTED and p(P, 4, -1, P, P, P, None) == EINVAL and p(None, 4, 2, P, P, P, None) == EINVAL
    assert p(P + 1, 4, 2, P, P, P, None) == EALIGN


def test_there_is_no_cpu_path():
    import applied_ai_amd as A

    x = torch.zeros(4, 16, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        A.rms_norm(x, torch.zeros(16, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        A.route_gate(torch.zeros(4, 8), 2)
    with pytest.raises(RuntimeError):
        A.lora_plan(torch.zeros(4, dtype=torch.int32), 2)


FILES = ["tests/test_gpu_lora.py", "tests/test_gpu_norm.py", "tests/test_gpu_gate.py"]


@pytest.mark.skipif(not os.path.exists(build_emu.CXX), reason="host clang++ of the ROCm toolchain not found: the emulated build needs it")
def test_gpu_tests_pass_on_the_emulated_kernels():
    """The GPU tests of these operators, run on the device code compiled for the host (tests/emu)."""
    build_emu.build()
    runs = [subprocess.Popen([sys.executable, os.path.join(EMU, "gpu_tests_on_emu.py"), f, "-k", "not graph and not stream and not long"], cwd=ROOT,
                             stdout=subprocess.PIPE, stderr=subprocess.STDOUT) for f in FILES]
    for f, p in zip(FILES, runs):
        log = p.communicate(timeout=900)[0].decode()
        assert p.returncode == 0, f + log[-3000:]


@pytest.mark.skipif(not os.path.exists(build_emu.CXX), reason="host clang++ of the ROCm toolchain not found: the emulated build needs it")
def test_random_calls_against_guard_pages():
    """Random calls with every tensor against an inaccessible page and LDS that starts as NaN, plans of nonsense among them."""
    build_emu.build()
    runs = [subprocess.Popen([sys.executable, os.path.join(EMU, "fuzz_layer_ops.py"), str(10 + i), "40", "wide"], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                             env=dict(os.environ, EMU_GUARD=guard, EMU_LDS_POISON="1")) for i, guard in enumerate(("end", "start"))]
    for p in runs:
        log = p.communicate(timeout=900)[0].decode()
        assert p.returncode == 0 and "done 40" in log, log[-2000:]


@pytest.mark.skipif(not os.path.exists(build_emu.CXX), reason="host clang++ of the ROCm toolchain not found: the emulated build needs it")
def test_no_data_race_between_the_waves_of_a_workgroup():
    """Every kernel of these operators under the race check of tests/emu (each wave a fiber of the thread sanitizer): no two
    accesses by different waves to the same LDS or global bytes without a barrier between them."""
    out = os.path.dirname(build_emu.build_race_check())
    exe = os.path.join(out, "race_layer_ops")
    objs = [os.path.join(out, f.replace(".hip", ".emu.o")) for f in build_emu.sources()] + [os.path.join(out, f + ".o") for f in ("race_selftest", "emu_core")]
    subprocess.run([build_emu.CXX, "-fsanitize=thread", "-x", "c++", os.path.join(EMU, "race_layer_ops.cpp"), "-x", "none", "-o", exe] + objs + ["-ldl", "-lpthread"], check=True)
    for seed in ("0", "5"):
        p = subprocess.run([exe], env=dict(os.environ, EMU_SEED=seed), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=900)
        log = p.stdout.decode()
        assert p.returncode == 0 and "data race" not in log and "returned an error: 0" in log, log[-3000:]
