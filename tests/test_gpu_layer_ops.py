"""The norms, the gate, the adapters and the expert layer together, as a layer uses them; captured into graphs; on another stream;
on tensors of more than 2^31 elements."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def inputs(T=48, d=256, n=128, E=8, k=2, L=3, R=8, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    c = dict(y0=r(T, d).to(BF), stream=r(T, d) * 2, post=(1 + 0.1 * r(d)).to(BF), gate=r(d).to(BF), pre=(1 + 0.1 * r(d)).to(BF), router=(r(E, d) / d ** 0.5).float(),
             w1=(r(E, 2 * n, d) / d ** 0.5).to(BF), w2=(r(E, d, n) / n ** 0.5).to(BF), shared=(r(d, d) / d ** 0.5).to(BF), a=(r(L, R, d) / d ** 0.5).to(BF),
             b=(r(L, d, R) * 0.3).to(BF), scales=torch.rand(L, generator=g) + 0.5, ids=torch.randint(-1, L, (T,), generator=g, dtype=torch.int32),
             post2=(1 + 0.1 * r(d)).to(BF), pre2=(1 + 0.1 * r(d)).to(BF), row_gate=torch.rand(T, 1, generator=g).to(BF), gz=(r(T, d) * 0.2).to(BF), gh=r(T, d) * 0.2)
    return c, dict(k=k, L=L, E=E)


def layer(A, c, p):
    """Forward through one layer: the norms behind the block before it, the router, the experts, a shared projection with adapters,
    the norms behind them. Then the gradients of everything but the experts back to the layer's input."""
    h1, z1 = A.block_norm(c["y0"], c["stream"], c["post"], c["gate"], c["pre"])
    logits = z1.float() @ c["router"].T
    weights, ids = A.route_gate(logits, p["k"])
    experts = A.fused_moe(z1, c["w1"], c["w2"], weights, ids)
    d = z1.shape[1]
    m = torch.full((1,), z1.shape[0], dtype=torch.int32, device=z1.device)
    y = A.grouped_gemm(z1, c["shared"].reshape(d, d), m)
    plan = A.lora_plan(c["ids"], p["L"])
    y, hl = A.lora_add(y, z1, c["a"], c["b"], plan, c["scales"], out=y, return_h=True)
    y2 = y + experts
    h2, z2 = A.block_norm(y2, h1, c["post2"], c["row_gate"], c["pre2"], 1.0, 0.5)
    gy2, gh1, gpost2, grow, gpre2 = A.block_norm_backward(c["gh"], c["gz"], y2, h2, c["post2"], c["row_gate"], c["pre2"], 1.0, 0.5)
    gz1, gshared = A.grouped_gemm_backward(gy2, z1, c["shared"].reshape(d, d), m)
    gz1, ga, gb = A.lora_backward(gy2, z1, c["a"], c["b"], plan, c["scales"], h=hl, grad_x=gz1, out=gz1)
    gw = torch.ones_like(weights)
    glogits = A.route_gate_backward(gw * weights, logits, ids)
    gz1 = gz1 + (glogits @ c["router"]).to(BF)
    gy0, gstream, gpost, ggate, gpre = A.block_norm_backward(gh1, gz1, c["y0"], h1, c["post"], c["gate"], c["pre"])
    return dict(h1=h1, z1=z1, weights=weights, ids=ids, h2=h2, z2=z2, ga=ga, gb=gb, gshared=gshared, gy0=gy0, gstream=gstream, gpost=gpost, ggate=ggate, gpre=gpre,
                gpost2=gpost2, grow=grow, gpre2=gpre2, glogits=glogits)


def layer64(c, p, ids):
    """The same in 64 bits with automatic differentiation, the choice of experts given (a near tie may fall the other way)."""
    w = {k: v.double().requires_grad_() if v.is_floating_point() else v for k, v in c.items()}

    def norm(v, g):
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6) * g

    h1 = w["stream"] + norm(w["y0"], w["post"]) * w["gate"]
    z1 = norm(h1, w["pre"])
    logits = z1 @ w["router"].T
    weights = torch.softmax(logits.gather(1, ids), 1)
    zd = z1.detach()
    out = []
    for t in range(z1.shape[0]):
        rows = []
        for e in ids[t].tolist():
            v = zd[t] @ w["w1"][e].T
            n = v.shape[0] // 2
            rows.append((torch.nn.functional.silu(v[:n]) * v[n:]) @ w["w2"][e].T)
        out.append((weights[t].detach()[:, None] * torch.stack(rows)).sum(0))
    y = z1 @ w["shared"].T
    who, has = c["ids"].clamp(min=0).long(), (c["ids"] >= 0).double()[:, None]
    hl = (w["a"][who] @ z1[:, :, None])[:, :, 0]
    y = y + has * w["scales"][who][:, None] * (w["b"][who] @ hl[:, :, None])[:, :, 0]
    y2 = y + torch.stack(out).detach()
    h2 = h1 + 0.5 * norm(y2, w["post2"]) * w["row_gate"]
    z2 = norm(h2, w["pre2"])
    # the gate's own gradient enters as that of sum weights^2 / 2
    total = (h2 * w["gh"].detach()).sum() + (z2 * w["gz"].detach()).sum() + (weights * weights).sum() / 2
    total.backward()
    return dict(h1=h1, z1=z1, weights=weights, h2=h2, z2=z2, ga=w["a"].grad, gb=w["b"].grad, gshared=w["shared"].grad, gy0=w["y0"].grad, gstream=w["stream"].grad,
                gpost=w["post"].grad, ggate=w["gate"].grad, gpre=w["pre"].grad, gpost2=w["post2"].grad, grow=w["row_gate"].grad, gpre2=w["pre2"].grad)


def test_a_layer_forward_and_back():
    """Each operator is held to its own tolerance elsewhere; here the chain, by norms. A result passes through at most ten roundings
    to bf16 (2^-8 of their own norm at most), each of which the following stages (norms, products of matrices of norm about 2)
    carry on with a factor of at most 2."""
    import applied_ai_amd as A

    c, p = inputs()
    got = layer(A, {k: v.cuda() for k, v in c.items()}, p)
    want = layer64(c, p, got["ids"].cpu().long())
    for k, v in want.items():
        off = float((got[k].double().cpu() - v.detach()).norm() / v.detach().norm())
        assert off <= 10 * 2 * 2.0 ** -8, (k, off)


def test_graph_replays_of_two_captures():
    """Two captures of the layer, replayed in turn with new inputs, give what the eager calls give, bit for bit."""
    import applied_ai_amd as A

    p = None
    state, graphs, outs = [], [], []
    for i, T in enumerate((16, 200)):
        c, p = inputs(T=T, seed=i)
        state.append({k: v.cuda() for k, v in c.items()})
    for s in state:
        layer(A, s, p)  # outside the capture first
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for s in state:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            with torch.cuda.graph(g, stream=side):
                outs.append(layer(A, s, p))
        graphs.append(g)
    for rep in range(3):
        for i, s in enumerate(state):
            c, _ = inputs(T=s["y0"].shape[0], seed=10 * rep + i + 5)
            for k, v in c.items():
                s[k].copy_(v)
        torch.cuda.synchronize()
        for g in graphs if rep % 2 else graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for s, o in zip(state, outs):
            want = layer(A, s, p)
            torch.cuda.synchronize()
            for k in o:
                assert torch.equal(o[k], want[k]), (rep, k)


def test_another_stream():
    import applied_ai_amd as A

    c, p = inputs(T=100, seed=3)
    d = {k: v.cuda() for k, v in c.items()}
    want = layer(A, d, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(A, d, p)
    torch.cuda.current_stream().wait_stream(side)
    for k in want:
        assert torch.equal(got[k], want[k]), k


def test_long_tensors_adapters():
    """More than 2^31 elements of y: rows at both ends and in between against the definition."""
    import applied_ai_amd as A

    T, K, N, R, L = 140000, 64, 16384, 8, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=BF)  # noqa: E731
    x, y, a, b = r(T, K), r(T, N), r(L, R, K) * 0.1, r(L, N, R) * 0.3
    ids = torch.randint(-1, L, (T,), generator=g, device="cuda", dtype=torch.int32)
    assert y.numel() > 2 ** 31
    plan = A.lora_plan(ids, L)
    out, h = A.lora_add(y, x, a, b, plan, return_h=True)
    rows = torch.tensor([0, 1, 63, 64, T // 2, 131072, T - 65, T - 2, T - 1], device="cuda")
    who = ids[rows].clamp(min=0).long()
    hw = (a.double()[who] @ x[rows].double()[:, :, None])[:, :, 0] * (ids[rows] >= 0)[:, None]
    part = (b.double()[who] @ hw[:, :, None])[:, :, 0]
    want = y[rows].double() + part
    # half a step of bf16; h off by 2^-17 of itself and 66 * 2^-23 of at most 64 * 16 * 0.5, against eight b of at most 1.5
    assert bool(((out[rows].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -17 * 4 + 66 * 2.0 ** -23 * 512) * 8 * 1.5).all())
    assert bool((h[rows].double() - hw).abs().max() <= 66 * 2.0 ** -23 * 512)
    del out
    gx, ga, gb = A.lora_backward(y, x, a, b, plan, h=h)
    # gradients of the first adapter, from its rows
    mine = (ids == 0).nonzero()[:, 0]
    u = torch.cat([part.float() @ b[0].float() for part in y[mine].split(8192)])
    want = u.T @ x[mine].float()
    assert float((ga[0].float() - want).norm() / want.norm()) <= 2.0 ** -8  # a rounding to bf16, and fp32 sums on both sides
    t = int(mine[-1])
    assert float((gx[t].float() - u[-1] @ a[0].float()).norm() / gx[t].float().norm()) <= 2.0 ** -8


def test_long_tensors_norms():
    import applied_ai_amd as A

    T, d = 270000, 8192
    g = torch.Generator(device="cuda").manual_seed(2)
    y = torch.randn(T, d, generator=g, device="cuda", dtype=BF)
    assert y.numel() > 2 ** 31
    w = 1 + 0.1 * torch.randn(d, generator=g, device="cuda")
    h, z = A.block_norm(y, y, w, None, w)
    gy, gres, gpost, _, gpre = A.block_norm_backward(None, y, y, h, w, None, w)
    rows = torch.tensor([0, 1, T // 2, 262144, T - 2, T - 1], device="cuda")
    v = y[rows].double()

    def norm(v):
        return v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6) * w.double()

    # half a step of bf16, and (d + 64) * 2^-23 < 2^-9 of terms that are below 8 in magnitude here
    want, fp32 = v + norm(v), 2.0 ** -9 * 8
    assert bool(((h[rows].double() - want).abs() <= 2.0 ** -8 * want.abs() + fp32).all())
    assert bool(((z[rows].double() - norm(want)).abs() <= 2.0 ** -8 * norm(want).abs() + fp32).all())
    hs = h[rows].double().requires_grad_()
    (norm(hs) * v).sum().backward()
    assert bool(((gres[rows].double() - hs.grad).abs() <= 2.0 ** -8 * hs.grad.abs() + fp32).all())
    assert bool(gy.isfinite().all()) and bool(gpost.isfinite().all()) and bool(gpre.isfinite().all())


def test_storage_that_begins_at_any_element():
    """Contiguous tensors whose first element lies 2 bytes (fp32: 4) past an aligned address: the same bits as aligned ones."""
    import applied_ai_amd as A

    def off_by_one(t):
        raw = torch.zeros(t.numel() + 9, dtype=t.dtype, device=t.device)
        v = raw[1:1 + t.numel()].view(t.shape)
        v.copy_(t)
        return v

    g = torch.Generator().manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    T, K, N, R, L = 40, 136, 72, 16, 3
    x, y, a, b, go, gx = (v.to(BF).cuda() for v in (r(T, K), r(T, N), r(L, R, K), r(L, N, R), r(T, N), r(T, K)))
    s, ids = torch.rand(L, generator=g).cuda(), torch.randint(-1, L, (T,), generator=g, dtype=torch.int32).cuda()
    plan = A.lora_plan(ids, L)
    want = A.lora_add(y, x, a, b, plan, s, return_h=True)
    got = A.lora_add(*(off_by_one(v) for v in (y, x, a, b)), A.LoraPlan(off_by_one(plan.perm), off_by_one(plan.offsets)), off_by_one(s), return_h=True)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    back = A.lora_backward(go, x, a, b, plan, s, h=want[1], grad_x=gx)
    got = A.lora_backward(off_by_one(go), off_by_one(x), off_by_one(a), off_by_one(b), plan, s, h=off_by_one(want[1]), grad_x=off_by_one(gx))
    assert all(torch.equal(p, q) for p, q in zip(back, got))
    st, w, gate, gh, gz = r(T, K).cuda(), r(K).cuda(), r(K).cuda(), r(T, K).cuda(), r(T, K).to(BF).cuda()
    want = A.block_norm(x, st, w, gate, w)
    got = A.block_norm(*(off_by_one(v) for v in (x, st, w, gate, w)))
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    back = A.block_norm_backward(gh, gz, x, want[0], w, gate, w)
    got = A.block_norm_backward(*(off_by_one(v) for v in (gh, gz, x, want[0], w, gate, w)))
    assert all(torch.equal(p, q) for p, q in zip(back, got))
    logits = r(T, 20).to(BF).cuda()
    weights, chosen = A.route_gate(logits, 3)
    got = A.route_gate(off_by_one(logits), 3)
    assert torch.equal(weights, got[0]) and torch.equal(chosen, got[1])
    assert torch.equal(A.route_gate_backward(weights, logits, chosen), A.route_gate_backward(off_by_one(weights), off_by_one(logits), off_by_one(chosen)))


def test_nothing_is_written_beside_the_results():
    """In-place results in the middle of a larger buffer leave what is around them."""
    import applied_ai_amd as A

    for T, N in ((5, 33), (600, 264)):
        g = torch.Generator().manual_seed(T)
        r = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()  # noqa: E731
        raw = torch.full(((T + 4) * (N + 5),), 7.0, dtype=BF, device="cuda")
        wide = raw.view(T + 4, N + 5)
        y = wide[2:T + 2, 3:N + 3]
        y.copy_(r(T, N))
        ids = torch.randint(-1, 2, (T,), generator=g, dtype=torch.int32).cuda()
        A.lora_add(y, r(T, 48), r(2, 12, 48), r(2, N, 12), A.lora_plan(ids, 2), out=y)
        around = wide.clone()
        around[2:T + 2, 3:N + 3] = 7.0
        assert bool((around == 7.0).all())
