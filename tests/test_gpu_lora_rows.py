"""Low-rank adapters over many rows: every row enters every result once. Whole numbers throughout, so that nothing is rounded: x and the
output's gradient have one entry other than zero in a row, a and b are -1, 0 and 1, and every sum is a whole number of at most
eight bits (checked below), which both 16-bit types hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def check(T, K, N, R, L, dtype, runs, keep, seed=0):
    import applied_ai_amd as A

    print("lora, many rows", T, K, N, R, L, dtype, runs, keep, flush=True)
    dev = torch.empty(0).cuda().device
    g = torch.Generator(device=dev).manual_seed(T + K + N + R + seed)
    ints = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device=dev)  # noqa: E731
    t = torch.arange(T, device=dev)
    ids = (t * (L + 1) // T if runs else ints(0, L + 1, T)) - 1
    kc, nc, xv, gv = ints(0, K, T), ints(0, N, T), ints(0, 2, T) * 2 - 1, ints(0, 2, T) * 2 - 1
    x, go = torch.zeros(T, K, dtype=dtype, device=dev), torch.zeros(T, N, dtype=dtype, device=dev)
    x[t, kc], go[t, nc] = xv.to(dtype), gv.to(dtype)
    a, b = ints(-1, 2, L, R, K), ints(-1, 2, L, N, R)
    plan = A.lora_plan(ids.to(torch.int32), L)
    who, live = ids.clamp(min=0), (ids >= 0)[:, None]
    h = a[who, :, kc] * xv[:, None] * live              # [T, R]
    u = b[who, nc] * gv[:, None] * live
    out, hk = A.lora_add(torch.zeros_like(go), x, a.to(dtype), b.to(dtype), plan, return_h=True)
    assert torch.equal(hk.long(), h)
    rows = torch.cat([t[:300], t[T // 2:T // 2 + 300], t[-300:]])
    assert R <= 256 and torch.equal(out[rows].long(), (b[who[rows]].double() @ h[rows].double()[:, :, None])[:, :, 0].long())
    del out
    gx, ga, gb = A.lora_backward(go, x, a.to(dtype), b.to(dtype), plan, h=hk if keep else None)
    assert torch.equal(gx[rows].long(), (a.double().transpose(1, 2).contiguous()[who[rows]] @ u[rows].double()[:, :, None])[:, :, 0].long())
    want_a, want_b = torch.zeros(L * K, R, dtype=torch.int64, device=dev), torch.zeros(L * N, R, dtype=torch.int64, device=dev)
    want_a.index_add_(0, who * K + kc, u * xv[:, None])
    want_b.index_add_(0, who * N + nc, h * gv[:, None])
    assert int(want_a.abs().max()) <= 256 and int(want_b.abs().max()) <= 256 and bool((want_b != 0).any())
    assert torch.equal(ga.long(), want_a.reshape(L, K, R).transpose(1, 2)), "grad_a"
    assert torch.equal(gb.long(), want_b.reshape(L, N, R)), "grad_b"


@pytest.mark.parametrize("shape", [(600, 40, 33, 7, 2), (1100, 24, 300, 16, 1), (1300, 72, 264, 40, 3)], ids=str)
def test_every_row_once(shape):
    check(*shape, BF, True, True)
    check(*shape, FP, False, False)


@pytest.mark.parametrize("shape", [(8192, 64, 1024, 16, 1), (8193, 64, 1024, 16, 1), (8193, 1000, 4096, 128, 5), (20000, 333, 300, 8, 70), (33000, 512, 2560, 64, 2)], ids=str)
@pytest.mark.parametrize("runs", [True, False], ids=["runs", "mixed"])
def test_every_row_once_in_long_batches(shape, runs):
    check(*shape, BF, runs, True)
    check(*shape, FP, runs, False)


def test_long_tensors_gradients():
    """More than 2^31 elements of the output's gradient."""
    assert 140000 * 16384 > 2 ** 31
    check(140000, 64, 16384, 8, 3, BF, False, True)
