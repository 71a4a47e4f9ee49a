"""The gradients of the norms around a block where rows have no columns, and where a workgroup adds up many rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("T", [1, 300])
@pytest.mark.parametrize("weights", [BF, F32])
def test_rows_without_columns(T, weights):
    """A gate per row is the only argument with elements: its gradient is an empty sum, zero."""
    import applied_ai_amd as A
    from applied_ai_amd import ops

    y, gate = torch.empty(T, 0, dtype=BF).cuda(), torch.ones(T, 1, dtype=weights).cuda()
    h, z = A.block_norm(y, y, None, gate)
    assert h.shape == (T, 0) and z is None
    got = A.block_norm_backward(y, None, y, y, None, gate)
    assert got[3].shape == (T, 1) and got[3].dtype == weights and not got[3].any()
    old = torch.full((T + 1, 1), float("nan"), dtype=weights).cuda()
    kind = 2 if weights == F32 else 0
    rc = A._lib.lib().moe_gg_block_norm_backward(None, 0, None, 0, None, 0, None, 0, None, gate.data_ptr(), 2, None, 1.0, 1.0, 1e-6, None, None, None,
                                                 old.data_ptr(), None, T, 0, 0, 0, kind, None, 0, ops._stream_ptr(old.device))
    assert rc == 0 and not old[:T].any() and bool(old[T].isnan().all())


# Rows of +1 and -1, gradients of small whole numbers, eps = 0: mean(v^2) is 1, so normed rows are the rows and every term of the
# weights' and gates' gradients is a whole number. A row lost or taken twice is off by one at least.
# Where d is a power of two all of it is exact. Else 1 / d is rounded: with it, the root, the quotient and the products a term is
# off by 10 * 2^-24 at most, and a sum over T rows takes at most T / 512 + 1 steps in a workgroup and 48 over the workgroups:
# ROUNDS * 2^-24 of the magnitudes for T up to 8192, which stays below 1 / 8 for the sizes here.
ROUNDS = 10 + 17 + 48
SIZES = [(2100, 24), (530, 520)]
LONG = [(4200, 64), (4200, 512), (2300, 333), (1100, 640), (1300, 1500), (1200, 2048), (1100, 3000), (1200, 4096), (1100, 5120), (1100, 7168), (1200, 8192), (1100, 9000),
        (1050, 12288), (1100, 16384)]


def whole(g, shape, dtype, lo=-2, hi=3):
    return torch.randint(lo, hi, shape, generator=g, device=g.device).to(dtype)


def signs(g, shape, dtype):
    return (torch.randint(0, 2, shape, generator=g, device=g.device) * 2 - 1).to(dtype)


def summed(what, got, terms, dim, exact):
    """got against the sum of terms (64 bits)."""
    want, room = terms.sum(dim), 0.0 if exact else ROUNDS * 2.0 ** -24 * terms.abs().sum(dim)
    off = (got.double().reshape(want.shape) - want).abs()
    assert bool((off <= room).all()), (what, float(off.max()), int((off > room).sum()))


def rowwise(what, got, want, magnitude):
    """Results of every row: half a step of their type, and 64 roundings of what they are the difference of."""
    off = (got.double() - want).abs() - torch.finfo(got.dtype).eps / 2 * (1 + 2.0 ** -10) * want.abs() - 64 * 2.0 ** -24 * magnitude
    assert bool((off <= 0).all()), (what, float(off.max()), int((off > 0).sum()))


def check_many_rows(T, d, dtype, stream, gate, seed=0):
    import applied_ai_amd as A

    print("norm, many rows", T, d, dtype, stream, gate, flush=True)
    g = torch.Generator(device=torch.empty(0).cuda().device).manual_seed(T + d + seed)
    exact = d & (d - 1) == 0
    y, h = signs(g, (T, d), dtype), signs(g, (T, d), stream)
    gz, gh = whole(g, (T, d), dtype), whole(g, (T, d), stream)
    w = signs(g, (d,), F32)
    # the norm in front of the next block
    _, gres, _, _, gpre = A.block_norm_backward(gh, gz, y, h, None, None, w, eps=0.0)
    h64, gz64, gh64 = h.double(), gz.double(), gh.double()
    summed("gradient of w_pre", gpre, gz64 * h64, 0, exact)
    t = gz64 * w.double()
    part = h64 * (t * h64).mean(1, keepdim=True)
    rowwise("gradient of the stream", gres, gh64 + t - part, gh64.abs() + t.abs() + part.abs())
    # the norm behind the block, with its gate
    y64 = y.double()
    v = signs(g, (d,) if gate == "channel" else (T, 1), F32) if gate else None
    gy, gres, gpost, ggate, _ = A.block_norm_backward(gh, None, y, h, w, v, None, eps=0.0)
    assert torch.equal(gres, gh)
    gate64 = v.double() if gate else torch.ones(1, 1, dtype=torch.float64, device=y.device)
    summed("gradient of w_post", gpost, gh64 * gate64 * y64, 0, exact)
    if gate:
        summed("gradient of the gate", ggate, gh64 * y64 * w.double(), 0 if gate == "channel" else 1, exact)
    t = gh64 * gate64 * w.double()
    part = y64 * (t * y64).mean(1, keepdim=True)
    rowwise("gradient of y", gy, t - part, t.abs() + part.abs())
    # the norm alone
    gx, gw = A.rms_norm_backward(gz, y, w, eps=0.0)
    summed("gradient of the weight", gw, gz64 * y64, 0, exact)
    t = gz64 * w.double()
    part = y64 * (t * y64).mean(1, keepdim=True)
    rowwise("gradient of x", gx, t - part, t.abs() + part.abs())


@pytest.mark.parametrize("gate", [None, "channel", "row"])
@pytest.mark.parametrize("T,d", SIZES)
def test_many_rows_to_a_workgroup(T, d, gate):
    check_many_rows(T, d, BF, F32, gate)
    check_many_rows(T, d, FP, FP, gate)


@pytest.mark.parametrize("gate", ["channel", "row"])
@pytest.mark.parametrize("T,d", LONG)
def test_many_long_rows_to_a_workgroup(T, d, gate):
    check_many_rows(T, d, BF, BF, gate)
    check_many_rows(T, d, FP, F32, gate)


@pytest.mark.parametrize("d", [512, 3000, 4096, 5120, 9000])
def test_many_long_rows_of_any_values(d):
    """The same loops on random values, elementwise."""
    from test_gpu_norm import run

    T = 2300 if d <= 512 else 1100
    run((T, d, BF, F32, F32, True, True, "channel"))
    run((T, d, FP, FP, FP, True, True, "row"))


def test_long_tensors_weight_gradients():
    """More than 2^31 elements: every row enters the weights' gradients once."""
    import applied_ai_amd as A

    T, d = 270000, 8192
    g = torch.Generator(device="cuda").manual_seed(3)
    y, gz = torch.empty(T, d, dtype=BF, device="cuda"), torch.empty(T, d, dtype=BF, device="cuda")
    for i in range(0, T, 30000):  # the generator's whole numbers take 8 bytes each
        y[i:i + 30000], gz[i:i + 30000] = signs(g, (min(30000, T - i), d), BF), whole(g, (min(30000, T - i), d), BF)
    assert y.numel() > 2 ** 31
    w = torch.ones(d, device="cuda")
    want = sum((y[i:i + 10000].float() * gz[i:i + 10000].float()).sum(0, dtype=torch.float64) for i in range(0, T, 10000))
    assert float(want.abs().max()) < 2 ** 24
    gpre = A.block_norm_backward(None, gz, y, y, None, None, w, eps=0.0)[4]
    assert torch.equal(gpre.double(), want)
    del gpre
    _, _, gpost, ggate, _ = A.block_norm_backward(gz, None, y, y, w, w, None, eps=0.0)
    assert torch.equal(gpost.double(), want) and torch.equal(ggate.double(), want)
