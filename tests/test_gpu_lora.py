"""Low-rank adapters (lora_plan, lora_add, lora_backward) against their definition in 64 bits, adapter by adapter.

Tolerances, elementwise, from the arithmetic: one rounding of the result (half a step of its type); fp32 sums of n terms,
n * 2^-23 of the sum of magnitudes; h and u as two 16-bit parts, off by 2^-17 (bf16: half a step of half a step, 2^-9 * 2^-9,
doubled) of their magnitude (fp16 keeps more, and at least 2^-22 of the largest of its rank)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def make(T, K, N, R, L, ids, dtype=BF, pad=0, seed=0, std=1.0):
    g = torch.Generator().manual_seed(1000 + seed + T + 7 * K + 11 * N + 13 * R + 17 * L)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    c = dict(x=(r(T, K + pad) * std).to(dtype)[:, :K], a=(r(L, R, K) / max(K, 1) ** 0.5).to(dtype), b=(r(L, N, R) * 0.3).to(dtype),
             y=r(T, N + pad).to(dtype)[:, :N], go=(r(T, N + pad) * 0.2).to(dtype)[:, :N], gx=(r(T, K) * 0.2).to(dtype),
             scales=torch.rand(L, generator=g) * 1.5 + 0.5)
    if ids == "random":
        c["ids"] = torch.randint(-1, L, (T,), generator=g, dtype=torch.int32)
    elif ids == "runs":
        c["ids"] = (torch.arange(T) * max(L - 1, 1) // max(T, 1)).to(torch.int32)  # the last adapter has no rows
    elif ids == "one":
        c["ids"] = torch.full((T,), L // 2, dtype=torch.int32)
    else:
        c["ids"] = torch.tensor([-1, L, 2 ** 31 - 1, -2 ** 31], dtype=torch.int64).to(torch.int32)[torch.arange(T) % 4]
    return c


def on_gpu(c):
    """The inputs on the device, with the row strides they have here."""
    d = {}
    for k, v in c.items():
        if v.dim() == 2 and not v.is_contiguous():
            wide = torch.empty(v.shape[0], v.stride(0), dtype=v.dtype).cuda()
            wide[:, :v.shape[1]] = v.contiguous().cuda()
            d[k] = wide[:, :v.shape[1]]
        else:
            d[k] = v.cuda()
    return d


def forward64(c):
    """out, h and their tolerances."""
    x, a, b, y, s = (c[n].double() for n in ("x", "a", "b", "y", "scales"))
    (T, K), (L, R) = x.shape, a.shape[:2]
    half = torch.finfo(c["y"].dtype).eps / 2
    h, th = torch.zeros(T, R, dtype=torch.float64), torch.zeros(T, R, dtype=torch.float64)
    out, tol = y.clone(), torch.zeros_like(y)
    for e in range(L):
        rows = (c["ids"] == e).nonzero()[:, 0]
        h[rows] = x[rows] @ a[e].T
        th[rows] = (K + 2) * 2.0 ** -23 * (x[rows].abs() @ a[e].abs().T)
        out[rows] += s[e] * (h[rows] @ b[e].T)
        part = s[e] * (h[rows].abs() @ b[e].abs().T)
        tol[rows] = (2.0 ** -17 + (2 * R + 4) * 2.0 ** -23) * part + s[e] * (th[rows] @ b[e].abs().T) + 2.0 ** -23 * y[rows].abs()
    tol += half * out.abs() * (1 + 2.0 ** -10) + (2.0 ** -24 if c["y"].dtype == FP else 0)
    return out, h, tol, th


def backward64(c, h64, with_base=True):
    x, a, b, go, s, gx0 = (c[n].double() for n in ("x", "a", "b", "go", "scales", "gx"))
    (T, K), (L, R), N = x.shape, a.shape[:2], b.shape[1]
    dt = c["x"].dtype
    half, tiny = torch.finfo(dt).eps / 2 * (1 + 2.0 ** -10), (2.0 ** -24 if dt == FP else 0)
    gx = gx0.clone() if with_base else torch.zeros_like(gx0)
    tx = 2.0 ** -23 * gx.abs()
    ga, gb, ta, tb = torch.zeros_like(a), torch.zeros_like(b), torch.zeros_like(a), torch.zeros_like(b)
    for e in range(L):
        rows = (c["ids"] == e).nonzero()[:, 0]
        if not len(rows):
            continue
        n, g, xr, h = len(rows), go[rows], x[rows], h64[rows]
        u = s[e] * (g @ b[e])
        tu = s[e] * (N + 2) * 2.0 ** -23 * (g.abs() @ b[e].abs()) + 2.0 ** -17 * u.abs() + 2.0 ** -22 * u.abs().max(0).values
        gx[rows] += u @ a[e]
        tx[rows] += tu @ a[e].abs() + (2 * R + 4) * 2.0 ** -23 * (u.abs() @ a[e].abs())
        ga[e] = u.T @ xr
        ta[e] = tu.T @ xr.abs() + (2 * n + 4) * 2.0 ** -23 * (u.abs().T @ xr.abs())
        gb[e] = s[e] * (g.T @ h)
        th = (K + 2) * 2.0 ** -23 * (xr.abs() @ a[e].abs().T) + 2.0 ** -17 * h.abs() + 2.0 ** -22 * h.abs().max(0).values
        tb[e] = s[e] * (g.abs().T @ th + (2 * n + 4) * 2.0 ** -23 * (g.abs().T @ h.abs()))
    return [(v, t + half * v.abs() + tiny) for v, t in ((gx, tx), (ga, ta), (gb, tb))]


def near(got, want, tol, what):
    got = got.double().cpu()
    off = (got - want).abs() - tol
    assert got.shape == want.shape and bool((off <= 0).all()), (what, float(off.max()), int((off > 0).sum()), got.numel())


SHAPES = [  # T, K, N, R, L, ids
    (1, 64, 64, 16, 1, "one"), (1, 1, 1, 1, 1, "one"), (3, 8, 24, 8, 5, "random"), (17, 200, 136, 16, 3, "random"), (33, 65, 39, 5, 4, "random"),
    (64, 520, 264, 16, 40, "random"), (40, 128, 320, 24, 130, "random"), (20, 72, 80, 128, 2, "random"), (18, 136, 70, 100, 3, "random"),
    (50, 96, 128, 40, 2, "one"), (25, 64, 72, 8, 3, "none"), (512, 72, 88, 16, 4, "runs"), (530, 64, 264, 20, 3, "random"), (700, 40, 33, 7, 2, "one"),
    (1100, 24, 40, 33, 3, "runs"), (520, 48, 64, 96, 70, "random"),
]


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(shape, dtype):
    import applied_ai_amd as A

    c = make(*shape, dtype=dtype)
    d = on_gpu(c)
    print("lora", shape, dtype, flush=True)
    plan = A.lora_plan(d["ids"], shape[4])
    out, h = A.lora_add(d["y"], d["x"], d["a"], d["b"], plan, d["scales"], return_h=True)
    want, h64, tol, th = forward64(c)
    near(h, h64, th, "h")
    near(out, want, tol, "out")
    got = A.lora_backward(d["go"], d["x"], d["a"], d["b"], plan, d["scales"], h=h, grad_x=d["gx"])
    for g, (v, t), what in zip(got, backward64(c, h64), ("grad_x", "grad_a", "grad_b")):
        near(g, v, t, what)
    # without what the forward pass kept and without the shared projection's part
    got = A.lora_backward(d["go"], d["x"], d["a"], d["b"], plan, d["scales"])
    for g, (v, t), what in zip(got, backward64(c, h64, with_base=False), ("grad_x", "grad_a", "grad_b")):
        near(g, v, t, what + " alone")


@pytest.mark.parametrize("shape", [(4200, 1040, 1111, 16, 5, "random"), (4200, 1040, 1111, 27, 5, "runs"), (4200, 1111, 1040, 64, 3, "random"),
                                   (4200, 1040, 1040, 128, 3, "runs"), (1300, 4100, 4099, 8, 70, "random")], ids=str)
def test_long_batches(shape):
    """The kernels' tiles of 64 (ranks beyond 64: 32) rows, which only calls of many rows and columns take."""
    test_forward_and_backward(shape, BF)
    test_forward_and_backward(shape, FP)


@pytest.mark.parametrize("pad", [1, 8])
@pytest.mark.parametrize("T", [37, 600])
def test_rows_apart_in_place_and_without_scales(T, pad):
    import applied_ai_amd as A

    c = make(T, 72, 120, 16, 3, "random", pad=pad)
    c["scales"] = torch.ones(3)
    d = on_gpu(c)
    plan = A.lora_plan(d["ids"], 3)
    want, h64, tol, _ = forward64(c)
    y = d["y"]
    wide = y.as_strided((T - 1, y.stride(0) - 120), (y.stride(0), 1), y.storage_offset() + 120)
    behind = wide.clone()
    before = y.clone()
    got = A.lora_add(y, d["x"], d["a"], d["b"], plan, out=y)
    assert got is y
    near(y, want, tol, "in place")
    none = (c["ids"] < 0).cuda()
    assert torch.equal(y[none].view(torch.int16), before[none].view(torch.int16))  # rows without an adapter keep their bits
    assert torch.equal(wide.contiguous().view(torch.int16), behind.view(torch.int16))  # and nothing is written between the rows
    gx = d["gx"].clone()
    got = A.lora_backward(d["go"], d["x"], d["a"], d["b"], plan, grad_x=gx, out=gx)
    assert got[0] is gx
    for g, (v, t) in zip(got, backward64(c, h64)):
        near(g, v, t, "in place")


def test_plan_groups_rows_in_order():
    import applied_ai_amd as A

    for T, L in ((1, 1), (7, 3), (300, 65), (64, 767), (5, 0)):
        g = torch.Generator().manual_seed(T)
        ids = torch.randint(-2, L + 2, (T,), generator=g, dtype=torch.int32)
        plan = A.lora_plan(ids.cuda(), L)
        key = torch.where((ids < 0) | (ids >= L), torch.full_like(ids, L), ids).long()
        assert torch.equal(plan.perm.cpu().long(), torch.argsort(key, stable=True))
        assert plan.offsets.cpu().tolist() == [0] + torch.bincount(key, minlength=L + 1).cumsum(0).tolist()


def test_rows_without_an_adapter_touch_nothing():
    """Infinities and NaN in rows that name no adapter stay in their rows."""
    import applied_ai_amd as A

    for T in (40, 540):
        c = make(T, 64, 72, 16, 3, "random", seed=5)
        off = c["ids"] < 0
        assert off.any()
        for n in ("x", "go"):
            c[n][off] = float("nan")
            c[n][off.nonzero()[0]] = float("inf")
        clean = dict(c, x=torch.where(off[:, None], torch.zeros_like(c["x"]), c["x"]), go=torch.where(off[:, None], torch.zeros_like(c["go"]), c["go"]))
        d = on_gpu(c)
        plan = A.lora_plan(d["ids"], 3)
        out, h = A.lora_add(d["y"], d["x"], d["a"], d["b"], plan, d["scales"], return_h=True)
        want, h64, tol, th = forward64(clean)
        near(out, want, tol, "out")
        near(h, h64, th, "h")
        for g, (v, t), what in zip(A.lora_backward(d["go"], d["x"], d["a"], d["b"], plan, d["scales"], h=h, grad_x=d["gx"]), backward64(clean, h64),
                                   ("grad_x", "grad_a", "grad_b")):
            near(g, v, t, what)


def test_half_precision_rows_of_every_magnitude():
    """fp16: h far beyond the type's range and far below its smallest value (scaled rows, scaled ranks)."""
    import applied_ai_amd as A

    c = make(48, 128, 64, 8, 2, "random", FP, seed=3)
    c["x"] = (c["x"].float() * torch.logspace(-3, 3.5, 48)[:, None]).to(FP)
    c["a"] = (c["a"].float() * torch.logspace(-2, 1.5, 8)[None, :, None]).to(FP)
    c["b"] = (c["b"].float() * 0.01).to(FP)
    d = on_gpu(c)
    plan = A.lora_plan(d["ids"], 2)
    out, h = A.lora_add(d["y"], d["x"], d["a"], d["b"], plan, d["scales"], return_h=True)
    want, h64, tol, th = forward64(c)
    assert h64.abs().max() > 65504 and want.abs().max() < 60000
    near(h, h64, th, "h")
    # what a row's two parts lose is relative to its largest rank: 2^-22 of it
    row = c["scales"].double()[c["ids"].clamp(min=0).long()][:, None] * h64.abs().max(1).values[:, None] * 2.0 ** -22
    near(out, want, tol + row * torch.where(c["ids"][:, None] >= 0, c["b"].double().abs().sum(2)[c["ids"].clamp(min=0).long()], torch.zeros(())), "out")


def test_empty_calls():
    import applied_ai_amd as A

    c = make(0, 64, 48, 8, 2, "random")
    d = on_gpu(c)
    plan = A.lora_plan(d["ids"], 2)
    assert plan.offsets.cpu().tolist() == [0, 0, 0, 0]
    out, h = A.lora_add(d["y"], d["x"], d["a"], d["b"], plan, d["scales"], return_h=True)
    assert out.shape == (0, 48) and h.shape == (0, 8)
    gx, ga, gb = A.lora_backward(d["go"], d["x"], d["a"], d["b"], plan, d["scales"], h=h)
    assert gx.shape == (0, 64) and not ga.any() and not gb.any()
    c = make(9, 64, 48, 8, 0, "none")  # no adapters at all: everything passes through
    d = on_gpu(c)
    plan = A.lora_plan(d["ids"], 0)
    out = A.lora_add(d["y"], d["x"], d["a"], d["b"], plan)
    assert torch.equal(out, d["y"])
    gx, ga, gb = A.lora_backward(d["go"], d["x"], d["a"], d["b"], plan, grad_x=d["gx"])
    assert torch.equal(gx, d["gx"]) and ga.numel() == 0 and gb.numel() == 0


def test_same_inputs_give_the_same_bits():
    import applied_ai_amd as A

    c = make(1300, 136, 200, 16, 2, "runs", seed=9)
    d = on_gpu(c)
    plan = A.lora_plan(d["ids"], 2)
    first = A.lora_backward(d["go"], d["x"], d["a"], d["b"], plan, d["scales"])
    for _ in range(3):
        again = A.lora_backward(d["go"], d["x"], d["a"], d["b"], plan, d["scales"])
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_gradient_against_differences():
    """The directional derivative of sum(go * out) along random directions of x, a and b: the sum is quadratic along each of
    them alone, so central differences are exact but for rounding; computed in 64 bits, compared with the kernels' gradients."""
    import applied_ai_amd as A

    c = make(24, 40, 32, 8, 2, "random", seed=1)
    d = on_gpu(c)
    plan = A.lora_plan(d["ids"], 2)
    grads = A.lora_backward(d["go"], d["x"], d["a"], d["b"], plan, d["scales"])
    g = torch.Generator().manual_seed(4)
    for name, grad, tol in zip(("x", "a", "b"), grads, (t for _, t in backward64(c, forward64(c)[1], with_base=False))):
        way = torch.randn(c[name].shape, generator=g).double()
        side = []
        for sign in (1, -1):
            moved = dict(c, **{name: c[name].double() + sign * 0.5 * way})
            side.append((c["go"].double() * forward64(moved)[0]).sum())
        assert abs((side[0] - side[1]) - (grad.double().cpu() * way).sum()) <= (tol * way.abs()).sum() + 1e-9


def test_refusals():
    import applied_ai_amd as A

    c = make(6, 16, 24, 4, 2, "random")
    d = on_gpu(c)
    plan = A.lora_plan(d["ids"], 2)
    args = dict(y=d["y"], x=d["x"], a=d["a"], b=d["b"], plan=plan)
    with pytest.raises(ValueError):
        A.lora_add(**dict(args, x=d["x"].half()))
    with pytest.raises(ValueError):
        A.lora_add(**dict(args, b=d["b"][:, :, :3]))
    with pytest.raises(ValueError):
        A.lora_add(**dict(args, plan=A.lora_plan(d["ids"], 3)))
    with pytest.raises(ValueError):
        A.lora_add(**dict(args, scales=torch.ones(3).cuda()))
    with pytest.raises(ValueError):
        A.lora_add(**dict(args, out=torch.empty(6, 23, dtype=BF).cuda()))
    with pytest.raises(ValueError):
        A.lora_backward(d["go"], d["x"], d["a"], d["b"], plan, h=torch.zeros(6, 5).cuda())
    with pytest.raises(RuntimeError):  # a rank beyond what the kernels cover
        A.lora_add(d["y"], d["x"], torch.zeros(2, 129, 16, dtype=BF).cuda(), torch.zeros(2, 24, 129, dtype=BF).cuda(), plan)
    with pytest.raises(ValueError):
        A.lora_plan(d["ids"].long(), 2)
