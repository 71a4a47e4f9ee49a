"""The norms around a block (block_norm, rms_norm and their gradients) against the definition in 64 bits; gradients by automatic
differentiation of it.

Tolerances, elementwise: half a step of the result's type, and (d + 64) * 2^-23 of the magnitudes that enter it: the
row sums of d terms in fp32 (d * 2^-24 at most, halved by the root, used twice) and the few products around them; sums over T
rows add T * 2^-23 of the summed magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def make(T, d, dtype, stream, weights, post, pre, gate, pad=0, seed=0):
    g = torch.Generator().manual_seed(10 * T + d + seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    c = dict(y=(r(T, d + pad) * 2).to(dtype)[:, :d], res=(r(T, d + pad) * 3).to(stream)[:, :d], gh=(r(T, d) * 0.3).to(stream), gz=(r(T, d + pad) * 0.3).to(dtype)[:, :d],
             post=(1 + 0.1 * r(d)).to(weights) if post else None, pre=(1 + 0.1 * r(d)).to(weights) if pre else None,
             gate=r(d).to(weights) if gate == "channel" else torch.rand(T, 1, generator=g).to(weights) if gate == "row" else None)
    return c


def cuda(t):
    if t is None or t.is_contiguous():
        return None if t is None else t.cuda()
    wide = torch.zeros(t.shape[0], t.stride(0), dtype=t.dtype).cuda()
    wide[:, :t.shape[1]] = t.contiguous().cuda()
    return wide[:, :t.shape[1]]


def norm(v, w, eps):
    return v / torch.sqrt((v * v).mean(1, keepdim=True) + eps) * w


def forward64(c, alpha, beta, eps):
    y, res = c["y"].double(), c["res"].double()
    n = norm(y, c["post"].double(), eps) if c["post"] is not None else y
    part = beta * (n * c["gate"].double() if c["gate"] is not None else n)
    h = alpha * res + part
    rel = (y.shape[1] + 64) * 2.0 ** -23
    th = rel * ((alpha * res).abs() + part.abs())
    z = tz = None
    if c["pre"] is not None:
        w = c["pre"].double()
        z = norm(h, w, eps)
        r = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
        # h off by th: its own place, and the root of the mean square through |h| th
        tz = r * th * w.abs() + z.abs() * (rel + r * r * (h.abs() * th).mean(1, keepdim=True))
        tz = tz + half(c["y"].dtype) * z.abs() + tiny(c["y"].dtype)
    return h, th + half(c["res"].dtype) * h.abs() + tiny(c["res"].dtype), z, tz


def half(dt):
    return torch.finfo(dt).eps / 2 * (1 + 2.0 ** -10)


def tiny(dt):
    return 2.0 ** -24 if dt == FP else 0.0


def backward64(c, h, alpha, beta, eps, has_y=True, has_gh=True):
    """Gradients at the stored stream h (in its type), and their tolerances."""
    d, T = h.shape[1], h.shape[0]
    h64 = h.double()
    leaf = {k: c[k].double().requires_grad_() if c[k] is not None else None for k in ("y", "post", "gate", "pre")}
    if has_y:
        n = norm(leaf["y"], leaf["post"], eps) if leaf["post"] is not None else leaf["y"]
        part = beta * (n * leaf["gate"] if leaf["gate"] is not None else n)
        before = ((h64 - part.detach()) / alpha).requires_grad_()
        now = alpha * before + part
    else:
        before = h64.clone().requires_grad_()
        now = before
    total = (now * c["gh"].double()).sum() if has_gh else (now * 0).sum()
    if leaf["pre"] is not None:
        total = total + (norm(now, leaf["pre"], eps) * c["gz"].double()).sum()
    total.backward()
    rel = 2 * (d + 64) * 2.0 ** -23
    # magnitudes of everything that enters, with absolute values throughout
    mag = c["gh"].double().abs() if has_gh else torch.zeros_like(h64)
    out = {}
    if leaf["pre"] is not None:
        r = 1 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + eps)
        g = (c["gz"].double() * c["pre"].double()).abs()
        mag = mag + r * (g + (h64 * r).abs() * (g * (h64 * r).abs()).mean(1, keepdim=True))
        out["pre"] = (leaf["pre"].grad, (rel + T * 2.0 ** -23) * (c["gz"].double() * h64 * r).abs().sum(0))
    out["res"] = (before.grad, rel * alpha * mag)
    if has_y:
        y = c["y"].double()
        r = 1 / torch.sqrt((y * y).mean(1, keepdim=True) + eps) if leaf["post"] is not None else torch.ones(T, 1).double()
        yn, w = (y * r).abs(), (c["post"].double().abs() if leaf["post"] is not None else 1.0)
        gate = c["gate"].double().abs() if leaf["gate"] is not None else 1.0
        g = beta * mag * gate * w
        out["y"] = (leaf["y"].grad, rel * r * (g + (yn * (g * yn).mean(1, keepdim=True) if leaf["post"] is not None else 0)))
        if leaf["post"] is not None:
            out["post"] = (leaf["post"].grad, (rel + T * 2.0 ** -23) * (beta * mag * gate * yn).sum(0))
        if leaf["gate"] is not None:
            t = beta * mag * yn * w
            out["gate"] = (leaf["gate"].grad, (rel + T * 2.0 ** -23) * t.sum(0) if leaf["gate"].shape == (d,) else rel * t.sum(1, keepdim=True))
    types = dict(y=c["y"].dtype, res=h.dtype, **{k: c[k].dtype for k in ("post", "gate", "pre") if c[k] is not None})
    return {k: (v, t + half(types[k]) * v.abs() + tiny(types[k])) for k, (v, t) in out.items()}


def near(got, want, tol, what):
    got = got.double().cpu()
    off = (got - want).abs() - tol
    assert got.shape == want.shape and bool((off <= 0).all()), (what, float(off.max()), int((off > 0).sum()), got.numel())


CASES = [  # T, d, rows, stream, weights, post, pre, gate
    (1, 64, BF, BF, BF, True, True, None), (5, 4096, BF, F32, BF, True, True, "channel"), (9, 512, FP, FP, F32, True, True, "row"), (3, 2048, FP, F32, FP, False, True, "channel"),
    (7, 1032, BF, BF, F32, True, False, None), (2, 1, BF, BF, BF, True, True, "row"), (6, 77, BF, F32, F32, True, True, "channel"), (4, 1030, FP, FP, FP, True, True, "row"),
    (2, 5000, BF, BF, BF, False, True, None), (3, 2001, FP, F32, F32, True, True, "channel"), (2, 8200, FP, F32, FP, True, True, "channel"), (130, 72, BF, BF, BF, True, True, "channel"),
    (1100, 16, BF, F32, BF, True, True, "row"), (2, 1500, BF, BF, BF, False, False, "row"), (600, 640, FP, FP, FP, True, True, "channel"), (1, 9001, BF, BF, BF, True, True, "channel"),
    (2, 16384, BF, BF, BF, True, True, None),
]


def run(case, pad=0, alpha=1.0, beta=0.5, eps=1e-6, has_gh=True):
    import applied_ai_amd as A

    c = make(*case, pad=pad)
    print("norm", case, flush=True)
    d = {k: cuda(v) for k, v in c.items()}
    h, z = A.block_norm(d["y"], d["res"], d["post"], d["gate"], d["pre"], alpha, beta, eps)
    want_h, th, want_z, tz = forward64(c, alpha, beta, eps)
    assert h.dtype == c["res"].dtype
    near(h, want_h, th, "h")
    if z is not None:
        assert z.dtype == c["y"].dtype
        near(z, want_z, tz, "z")
    else:
        assert c["pre"] is None
    got = A.block_norm_backward(d["gh"] if has_gh else None, d["gz"] if c["pre"] is not None else None, d["y"], h, d["post"], d["gate"], d["pre"], alpha, beta, eps)
    want = backward64(c, h.cpu(), alpha, beta, eps, has_gh=has_gh)
    for name, g in zip(("y", "res", "post", "gate", "pre"), got):
        if name in want:
            near(g, *want[name], "gradient of " + name)
        else:
            assert g is None, name


@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_backward(case):
    run(case)


def test_scales_rows_apart_and_no_stream_gradient():
    run((11, 136, BF, F32, BF, True, True, "channel"), pad=8, alpha=1.7, beta=0.25, eps=1e-5)
    run((11, 136, FP, FP, F32, True, True, "row"), pad=3, alpha=0.5, beta=2.0, has_gh=False)
    run((6, 520, BF, BF, BF, False, True, None), pad=1, alpha=1.0, beta=1.0)


@pytest.mark.parametrize("T,d,dtype,stream,weights", [(1, 64, BF, BF, BF), (7, 4096, BF, F32, F32), (5, 333, FP, FP, FP), (520, 128, FP, F32, FP)])
def test_the_norm_alone(T, d, dtype, stream, weights):
    import applied_ai_amd as A

    c = make(T, d, dtype, stream, weights, False, True, None, pad=2)
    g = {k: cuda(v) for k, v in c.items()}
    z = A.rms_norm(g["res"], g["pre"], 1e-6, dtype)
    x, w = c["res"].double(), c["pre"].double()
    want = norm(x, w, 1e-6)
    near(z, want, (d + 64) * 2.0 ** -23 * want.abs() + half(dtype) * want.abs() + tiny(dtype), "z")
    for has in (True, False):
        gx, gw = A.rms_norm_backward(g["gz"], g["res"], g["pre"], 1e-6, grad_x=g["gh"] if has else None)
        want = backward64(c, c["res"], 1.0, 1.0, 1e-6, has_y=False, has_gh=has)
        near(gx, *want["res"], "gradient of x")
        near(gw, *want["pre"], "gradient of the weight")


def test_rows_of_zeros_and_rows_that_are_not_finite():
    """A row of zeros is normed to zeros with finite gradients; NaN and infinities stay in their row."""
    import applied_ai_amd as A

    c = make(6, 264, BF, BF, BF, True, True, None)
    c["y"][1] = 0
    c["res"][1] = 0
    c["y"][4] = float("nan")
    c["res"][2, 7] = float("inf")
    d = {k: cuda(v) for k, v in c.items()}
    h, z = A.block_norm(d["y"], d["res"], d["post"], None, d["pre"])
    assert not h[1].any() and not z[1].any() and bool(z[4].isnan().all()) and bool(h[2, :7].isfinite().all())
    clean = {k: (v[[0, 3, 5]] if k in ("y", "res", "gh", "gz") else v) for k, v in c.items()}
    want_h, th, want_z, tz = forward64(clean, 1.0, 1.0, 1e-6)
    near(h[[0, 3, 5]], want_h, th, "h")
    near(z[[0, 3, 5]], want_z, tz, "z")
    g = A.block_norm_backward(d["gh"], d["gz"], d["y"], h, d["post"], None, d["pre"])
    assert bool(g[0][1].isfinite().all()) and bool(g[1][[0, 1, 3, 5]].isfinite().all())


def test_no_rows():
    import applied_ai_amd as A

    c = make(0, 64, BF, BF, BF, True, True, "channel")
    d = {k: cuda(v) for k, v in c.items()}
    h, z = A.block_norm(d["y"], d["res"], d["post"], d["gate"], d["pre"])
    assert h.shape == z.shape == (0, 64)
    g = A.block_norm_backward(d["gh"], d["gz"], d["y"], h, d["post"], d["gate"], d["pre"])
    assert g[0].shape == g[1].shape == (0, 64) and not g[2].any() and not g[3].any() and not g[4].any()


def test_same_inputs_give_the_same_bits():
    import applied_ai_amd as A

    c = make(700, 320, BF, BF, F32, True, True, "channel")
    d = {k: cuda(v) for k, v in c.items()}
    h, _ = A.block_norm(d["y"], d["res"], d["post"], d["gate"], d["pre"])
    first = A.block_norm_backward(d["gh"], d["gz"], d["y"], h, d["post"], d["gate"], d["pre"])
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, A.block_norm_backward(d["gh"], d["gz"], d["y"], h, d["post"], d["gate"], d["pre"])))


def test_refusals():
    import applied_ai_amd as A

    c = make(4, 64, BF, BF, BF, True, True, "channel")
    d = {k: cuda(v) for k, v in c.items()}
    for bad in (dict(y=d["y"].float()), dict(residual=d["res"].half()), dict(post_weight=d["post"][:32]), dict(gate=d["gate"].float()),
                dict(gate=d["gate"][:, None].contiguous()), dict(pre_weight=d["pre"].half())):
        args = dict(y=d["y"], residual=d["res"], post_weight=d["post"], gate=d["gate"], pre_weight=d["pre"])
        with pytest.raises(ValueError):
            A.block_norm(**dict(args, **bad))
    with pytest.raises(ValueError):
        A.block_norm_backward(d["gh"], None, d["y"], d["res"], d["post"], d["gate"], d["pre"])
    with pytest.raises(RuntimeError):  # wider than the kernels cover
        A.rms_norm(torch.zeros(1, 16392, dtype=BF).cuda(), torch.zeros(16392, dtype=BF).cuda())
    with pytest.raises(ValueError):
        A.rms_norm(torch.zeros(1, 64).cuda(), torch.zeros(64).cuda())  # fp32 rows need the result's type
