"""Low-rank adapters: h and u enter the products in full, not in the type of the matrix instructions' operands.

h and u are made with 24 significant bits, p * 2^8 + q + r * 2^-8 (p below 2^8, q below 2^7), and every result is the difference
of two of them that agree in p and q. An operand of two parts of bf16 holds p and q and rounds r * 2^-8, which lies between 56 / 256
and 72 / 256, to a multiple of 1 / 2: it loses most of the result.

Tolerance: every term and every sum is a multiple of 2^-8 below 2^17, so fp32 sums are exact but for a unit of 2^-8 in each of at most
four that pass 2^16; two operand parts of fp16 are off by 2^-22 of the largest, 2 * 2^-22 * 2^16 for two of them; and half a step
of the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
TOL = 4 * 2.0 ** -8 + 2 * 2.0 ** -6
SHAPES = [(20, 9, 70, 2, 3), (40, 70, 9, 17, 2), (530, 33, 66, 5, 2), (48, 40, 80, 40, 2), (530, 72, 40, 100, 3)]  # T, K, N, R, L


def digits(g, n):
    """[n, 3]: p in [129, 255], q in [65, 127], both odd, and r in [56, 72]."""
    p, q = (torch.randint(lo, hi, (n, 1), generator=g) * 2 + 1 for lo, hi in ((64, 128), (32, 64)))
    return torch.cat([p, q, torch.randint(56, 73, (n, 1), generator=g)], 1).double()


def pick(g, n, k):
    return torch.randperm(n, generator=g)[:k]


def near(got, want, what):
    off = (got.double().cpu() - want).abs() - TOL - torch.finfo(got.dtype).eps / 2 * want.abs()
    assert bool((off <= 0).all()), (what, float(off.max()), int((off > 0).sum()))


def rows(g, T, L):
    """ids of every row, and two rows of each adapter."""
    ids = torch.arange(T) % (L + 1)
    ids = torch.where(ids == L, torch.full_like(ids, -1), ids)[torch.randperm(T, generator=g)].to(torch.int32)
    return ids, [(ids == e).nonzero()[pick(g, int((ids == e).sum()), 2), 0].tolist() for e in range(L)]


def tensors(T, K, N, R, L, seed):
    g = torch.Generator().manual_seed(seed + T + K + N + R)
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    ids, pairs = rows(g, T, L)
    return g, ids, pairs, dict(y=z(T, N), x=z(T, K), a=z(L, R, K), b=z(L, N, R), go=z(T, N))


def device(c, dtype):
    return {k: v.to(dtype).cuda() for k, v in c.items()}


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_result_of_two_ranks_that_nearly_cancel(shape, dtype):
    import applied_ai_amd as A

    T, K, N, R, L = shape
    g, ids, _, c = tensors(*shape, seed=1)
    print("parts, forward", shape, dtype, flush=True)
    v, sign = digits(g, T), torch.randint(0, 2, (N,), generator=g).double() * 2 - 1
    col, (i, j) = pick(g, K, 3), pick(g, R, 2).tolist()
    c["x"][:, col] = v
    c["a"][:, i, col] = torch.tensor([256.0, 1.0, 2.0 ** -8]).double()
    c["a"][:, j, col] = torch.tensor([256.0, 1.0, 0.0]).double()
    c["b"][:, :, i], c["b"][:, :, j] = sign, -sign
    d = device(c, dtype)
    out, h = A.lora_add(d["y"], d["x"], d["a"], d["b"], A.lora_plan(ids.cuda(), L), return_h=True)
    live = (ids >= 0).double()[:, None]
    want = v[:, 2:] * 2.0 ** -8 * sign * live
    near(out, want, "out")
    # and the gradient of x: u of the same two ranks
    g, ids, _, c = tensors(*shape, seed=2)
    col = pick(g, N, 3)
    c["go"][:, col] = v
    c["b"][:, col, i] = torch.tensor([256.0, 1.0, 2.0 ** -8]).double()
    c["b"][:, col, j] = torch.tensor([256.0, 1.0, 0.0]).double()
    sign = torch.randint(0, 2, (K,), generator=g).double() * 2 - 1
    c["a"][:, i], c["a"][:, j] = sign, -sign
    d = device(c, dtype)
    gx = A.lora_backward(d["go"], d["x"], d["a"], d["b"], A.lora_plan(ids.cuda(), L))[0]
    near(gx, v[:, 2:] * 2.0 ** -8 * sign * (ids >= 0).double()[:, None], "grad_x")


@pytest.mark.parametrize("keep", [True, False], ids=["kept", "again"])
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients_of_two_rows_that_nearly_cancel(shape, dtype, keep):
    import applied_ai_amd as A

    T, K, N, R, L = shape
    print("parts, gradients", shape, dtype, keep, flush=True)
    # grad_b: two rows with nearly the same h and opposite gradients of the output
    g, ids, pairs, c = tensors(*shape, seed=3)
    col, sign = pick(g, K, 3), torch.randint(0, 2, (N,), generator=g).double() * 2 - 1
    c["a"][:, :, col] = torch.tensor([256.0, 1.0, 2.0 ** -8]).double()
    want = torch.zeros(L, N, R).double()
    for e, (s, t) in enumerate(pairs):
        v = digits(g, 1)[0]
        c["x"][s, col], c["x"][t, col[:2]] = v, v[:2]
        c["go"][s], c["go"][t] = sign, -sign
        want[e] = v[2] * 2.0 ** -8 * sign[:, None]
    d, plan = device(c, dtype), A.lora_plan(ids.cuda(), L)
    h = A.lora_add(d["y"], d["x"], d["a"], d["b"], plan, return_h=True)[1] if keep else None
    near(A.lora_backward(d["go"], d["x"], d["a"], d["b"], plan, h=h)[2], want, "grad_b")
    # grad_a: two rows with nearly the same u and opposite x
    g, ids, pairs, c = tensors(*shape, seed=4)
    col, sign = pick(g, N, 3), torch.randint(0, 2, (K,), generator=g).double() * 2 - 1
    c["b"][:, col] = torch.tensor([256.0, 1.0, 2.0 ** -8]).double()[:, None]
    want = torch.zeros(L, R, K).double()
    for e, (s, t) in enumerate(pairs):
        v = digits(g, 1)[0]
        c["go"][s, col], c["go"][t, col[:2]] = v, v[:2]
        c["x"][s], c["x"][t] = sign, -sign
        want[e] = v[2] * 2.0 ** -8 * sign
    d, plan = device(c, dtype), A.lora_plan(ids.cuda(), L)
    near(A.lora_backward(d["go"], d["x"], d["a"], d["b"], plan, h=torch.zeros(T, R).cuda() if keep else None)[1], want, "grad_a")
