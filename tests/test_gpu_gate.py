"""The router's gate (route_gate, route_gate_backward): ids exactly, weights and gradients against the definition in 64 bits.

Tolerances: exponentials and logarithms of fp32 (2 units of 2^-23 each, and 2^-24 of an exponent's argument, below 64 here),
sums of at most 768 terms in at most 12 + 6 steps: 128 * 2^-23 of a weight; a gradient as much of the magnitudes that enter it,
and half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")
REL = 128 * 2.0 ** -23


def make(T, E, dtype=torch.float32, off=0, seed=0):
    g = torch.Generator().manual_seed(T * 1000 + E + seed)
    logits = (torch.randn(T, E, generator=g) * 2).to(dtype)
    if off:
        logits[:, torch.randperm(E, generator=g)[:off]] = -INF
    return logits


def order(logits, k):
    return torch.sort(logits.double(), dim=1, descending=True, stable=True).indices[:, :k]


def weights64(v, ids, score, renormalize, scale):
    lp = torch.log_softmax(v, 1) if score == "softmax" else torch.nn.functional.logsigmoid(v)
    of = lp.gather(1, ids)
    w = scale * (torch.softmax(of, 1) if renormalize else torch.exp(of))
    return torch.where(torch.isnan(w), torch.zeros_like(w), w)  # rows of -inf alone


def backward_tolerance(v, ids, gw, score, renormalize, scale):
    w = weights64(v, ids, score, renormalize, 1.0)
    dot = (w * gw.abs()).sum(1, keepdim=True)
    mag = torch.zeros_like(v).scatter_add(1, ids, scale * w * (gw.abs() + (dot if renormalize else 0)))
    if score == "softmax" and not renormalize:
        mag = mag + scale * torch.nan_to_num(torch.softmax(v, 1)) * dot
    # the oracle's own rounding: log_softmax's gradient subtracts softmax(v) * sum, terms of at most scale * sum |gw| in 53 bits that
    # cancel for experts not chosen (where the result is exactly zero)
    return REL * mag + 2.0 ** -48 * scale * gw.abs().sum(1, keepdim=True)


CASES = [(1, 8, 2), (5, 8, 8), (33, 7, 3), (9, 16, 1), (65, 20, 5), (17, 64, 6), (10, 65, 4), (30, 128, 8), (7, 256, 8), (3, 257, 64), (4, 768, 16), (1, 1, 1)]


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k", CASES)
def test_forward_and_backward(T, E, k, score, renormalize):
    import applied_ai_amd as A

    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        print("gate", T, E, k, score, renormalize, dtype, flush=True)
        logits = make(T, E, dtype)
        dev = logits.cuda()
        w, ids = A.route_gate(dev, k, score, renormalize, 2.5)
        want_ids = order(logits, k)
        assert torch.equal(ids.cpu().long(), want_ids)
        want = weights64(logits.double(), want_ids, score, renormalize, 2.5)
        assert bool(((w.double().cpu() - want).abs() <= REL * want + 1e-37).all())
        gw = torch.randn(T, k, generator=torch.Generator().manual_seed(E))
        got = A.route_gate_backward(gw.cuda(), dev, ids, score, renormalize, 2.5)
        v = logits.double().requires_grad_()
        weights64(v, want_ids, score, renormalize, 2.5).backward(gw.double())
        assert got.dtype == dtype
        tol = backward_tolerance(logits.double(), want_ids, gw.double(), score, renormalize, 2.5) + torch.finfo(dtype).eps / 2 * v.grad.abs()
        assert bool(((got.double().cpu() - v.grad).abs() <= tol + (2.0 ** -24 if dtype == torch.float16 else 1e-37)).all())


def test_ties_go_to_the_lower_expert_as_in_route_topk():
    import applied_ai_amd as A

    for E, k in ((8, 3), (64, 9), (200, 30)):
        logits = torch.randint(-2, 3, (40, E), generator=torch.Generator().manual_seed(E)).float()
        logits[0] = 0
        _, ids = A.route_gate(logits.cuda(), k)
        assert torch.equal(ids.cpu().long(), order(logits, k))
        assert torch.equal(ids, A.route_topk(logits.cuda(), k)[0])


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_experts_switched_off(score, renormalize):
    """Logits of -inf: chosen only for want of others, with weight and gradient 0; a row of nothing else gives zeros."""
    import applied_ai_amd as A

    for E, k, off in ((8, 4, 3), (12, 6, 10), (100, 8, 95)):
        logits = make(9, E, off=off)
        logits[4] = -INF
        logits[6] = torch.finfo(torch.float32).min  # the lowest number is a number
        w, ids = A.route_gate(logits.cuda(), k, score, renormalize, 1.0)
        want_ids = order(logits, k)
        assert torch.equal(ids.cpu().long(), want_ids)
        chosen = logits.gather(1, want_ids)
        assert not w.cpu()[chosen == -INF].any() and not w[4].any() and bool(w.isfinite().all())
        rows = [r for r in range(9) if r != 6]  # (there log p itself is beyond fp32 for the sigmoid)
        want = weights64(logits.double(), want_ids, score, renormalize, 1.0)
        assert bool(((w.double().cpu() - want).abs() <= REL * want + 1e-37)[rows].all())
        g = A.route_gate_backward(torch.ones(9, k).cuda(), logits.cuda(), ids, score, renormalize, 1.0)
        assert bool(g.isfinite().all()) and not g[4].any() and not g.cpu()[logits == -INF].any()


def test_sigmoid_scores_that_underflow_are_still_renormalised():
    import applied_ai_amd as A

    logits = -200 + torch.randn(6, 32, generator=torch.Generator().manual_seed(2))
    w, ids = A.route_gate(logits.cuda(), 4, "sigmoid")
    want = weights64(logits.double(), ids.cpu().long(), "sigmoid", True, 1.0)
    assert bool(((w.double().cpu() - want).abs() <= 2 * REL * want).all())  # arguments of 200 instead of 64: 2^-24 * 200 more


def test_rows_of_nan_stay_alone_and_ids_in_range():
    import applied_ai_amd as A

    for E in (8, 100):
        logits = make(5, E)
        logits[2, 1] = float("nan")
        logits[3] = float("nan")
        w, ids = A.route_gate(logits.cuda(), 3)
        assert bool(((ids >= 0) & (ids < E)).all()) and torch.equal(ids.cpu()[[0, 1, 4]].long(), order(logits[[0, 1, 4]], 3))
        assert bool(w[[0, 1, 4]].isfinite().all()) and all(len(set(r)) == 3 for r in ids.cpu().tolist())


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_backward_with_ids_out_of_range_or_named_twice(score, renormalize):
    """An id outside [0, E) takes no part; one named twice is two terms of the sums."""
    import applied_ai_amd as A

    E, k, T = 20, 4, 6
    logits = make(T, E)
    ids = order(logits, k).to(torch.int32)
    ids[1, 2], ids[2, 0], ids[3, 1] = -1, E, ids[3, 0]
    gw = torch.randn(T, k, generator=torch.Generator().manual_seed(8))
    got = A.route_gate_backward(gw.cuda(), logits.cuda(), ids.cuda(), score, renormalize, 1.5).double().cpu()
    for t in range(T):
        live = [(int(i), float(g)) for i, g in zip(ids[t], gw[t]) if 0 <= i < E]
        v = logits[t:t + 1].double().requires_grad_()
        at, g = torch.tensor([[i for i, _ in live]]), torch.tensor([[g for _, g in live]]).double()
        weights64(v, at, score, renormalize, 1.5).backward(g)
        tol = backward_tolerance(logits[t:t + 1].double(), at, g, score, renormalize, 1.5) + 2.0 ** -24 * v.grad.abs() + 1e-37
        assert bool(((got[t:t + 1] - v.grad).abs() <= tol).all()), t


def test_no_rows_and_refusals():
    import applied_ai_amd as A

    w, ids = A.route_gate(torch.empty(0, 8).cuda(), 2)
    assert w.shape == ids.shape == (0, 2)
    assert A.route_gate_backward(w, torch.empty(0, 8).cuda(), ids).shape == (0, 8)
    logits = make(4, 8).cuda()
    for bad in (dict(k=0), dict(k=9), dict(score="relu"), dict(logits=logits.double()), dict(logits=logits[0])):
        with pytest.raises(ValueError):
            A.route_gate(**dict(dict(logits=logits, k=2), **bad))
    with pytest.raises(RuntimeError):
        A.route_gate(torch.zeros(2, 769).cuda(), 2)
    with pytest.raises(RuntimeError):
        A.route_gate(torch.zeros(2, 100).cuda(), 65)
    with pytest.raises(ValueError):
        A.route_gate_backward(torch.zeros(4, 2).cuda(), logits, torch.zeros(4, 3, dtype=torch.int32).cuda())
