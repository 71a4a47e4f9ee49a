"""Random calls of the adapters, the norms and the gate on the emulated library, with EMU_GUARD=end or start every tensor
against an inaccessible page (tests/emu/harness.py), compared with numpy; plans with entries that name no row among them, of
which nothing is asked but that no access leaves a tensor. Run by tests/test_layer_ops_host.py in child processes.

usage: fuzz_layer_ops.py SEED CASES [wide]
wide: the adapters' kernels on tiles of 64 (32) rows first, which only large calls take."""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import harness as H  # noqa: E402

P = H.P


def data(rng, shape, fp16, scale=1.0):
    b = H.to16((rng.standard_normal(shape) * scale).astype(np.float32), fp16)
    return H.G(b), H.from16(b, fp16).astype(np.float64)


def work(nbytes):
    raw = H._full(max(int(nbytes), 256) // 256 * 256 + 512, 0xFF, np.uint8)
    off = (-raw.ctypes.data) % 256 if H.GUARD != "end" else (raw.size - nbytes) // 256 * 256 + (-raw.ctypes.data) % 256 - (256 if raw.ctypes.data % 256 else 0)
    off = max(off, (-raw.ctypes.data) % 256)
    assert off + nbytes <= raw.size and (raw.ctypes.data + off) % 256 == 0
    return raw.ctypes.data + off


def near(got, want, fp16, what, terms=0.0):
    """terms: magnitudes of fp32 terms whose difference the result is (up to 64 roundings of 2^-24 each)."""
    got = got if got.dtype == np.float32 else H.from16(got, fp16)
    scale = np.sqrt(np.mean(want * want)) + 1e-6 if want.size else 1.0
    assert np.all(np.abs(got - want) <= 0.02 * scale + 0.02 * np.abs(want) + 2.0 ** -18 * terms), what


def size(rng, hi):
    v = int(np.exp(rng.uniform(0, np.log(hi))))
    return max(1, v // 8 * 8) if rng.random() < 0.5 else v


def c_lora(rng, shape=None):
    L, fp16 = H.lib(), bool(rng.integers(2))
    T = int(rng.choice([1, 2, 15, 16, 17, 40, 511, 512, 600, 1030])) if rng.random() < 0.7 else size(rng, 700)
    K, N, R, n = size(rng, 300), size(rng, 300), int(rng.choice([1, 4, 8, 12, 16, 17, 33, 64, 128])), int(rng.choice([0, 1, 2, 5, 63, 64, 70]))
    corrupt = rng.random() < 0.2
    if shape:
        (T, K, N, R, n), corrupt = shape, False
    what = ("lora", T, K, N, R, n, fp16, corrupt)
    print(what, flush=True)
    ids = rng.integers(-1, max(n, 1), T).astype(np.int32)
    perm, off = H._full(T, -7, dtype=np.int32), H._full(n + 2, -7, dtype=np.int32)
    scratch = H._full(T + n + 1, -7, dtype=np.int32)
    H.ok(L.moe_gg_lora_plan(P(ids), T, n, P(perm), P(off), P(scratch), None))
    if corrupt:
        perm[...] = rng.integers(-5, T + 5, T)
        off[...] = rng.integers(-3, T + 4, n + 2)
        if rng.random() < 0.5:
            off.sort()
    (x, xf), (a, af), (b, bf), (y, yf), (g, gf), (gi, gif) = (data(rng, s, fp16, f) for s, f in (((T, K), 1), ((n, R, K), K ** -0.5), ((n, N, R), 0.3), ((T, N), 1),
                                                                                          ((T, N), 0.3), ((T, K), 0.3)))
    s = H.G(rng.uniform(0.5, 2, n).astype(np.float32))
    dt = H.FP16 if fp16 else H.BF16
    out, h = H._full((T, N), H.NAN16, np.uint16), H._full((T, R), np.nan, np.float32)
    nb = L.moe_gg_lora_add_workspace(T, n, K, N, R)
    H.ok(L.moe_gg_lora_add(P(y), N, P(x), K, P(a), P(b), P(s), P(perm), P(off), n, T, K, N, R, P(out), N, P(h), dt, work(nb), nb, None))
    gx, ga, gb = H._full((T, K), H.NAN16, np.uint16), H._full((n, R, K), H.NAN16, np.uint16), H._full((n, N, R), H.NAN16, np.uint16)
    keep = rng.random() < 0.5
    nb = L.moe_gg_lora_backward_workspace(T, n, K, N, R, int(keep))
    H.ok(L.moe_gg_lora_backward(P(g), N, P(x), K, P(a), P(b), P(s), P(perm), P(off), n, T, K, N, R, P(h) if keep else None, P(gi), K, P(gx), K, P(ga), P(gb), dt,
                                work(nb), nb, None))
    if corrupt:
        return
    hw, ow, gxw, gaw, gbw = np.zeros((T, R)), yf.copy(), gif.copy(), np.zeros((n, R, K)), np.zeros((n, N, R))
    for e in range(n):
        r = np.nonzero(ids == e)[0]
        hw[r] = xf[r] @ af[e].T
        ow[r] += s[e] * hw[r] @ bf[e].T
        u = s[e] * gf[r] @ bf[e]
        gxw[r] += u @ af[e]
        gaw[e], gbw[e] = u.T @ xf[r], s[e] * gf[r].T @ hw[r]
    for got, want, name in ((h, hw, "h"), (out, ow, "out"), (gx, gxw, "gx"), (ga, gaw, "ga"), (gb, gbw, "gb")):
        near(got, want, fp16, what + (name,))


def c_norm(rng):
    L, fp16, wide, wide_w = H.lib(), bool(rng.integers(2)), bool(rng.integers(2)), bool(rng.integers(2))
    T, d = int(rng.choice([1, 2, 5, 33, 130, 700])), size(rng, 3000)
    T = T if d * T < 40000 else 2
    kind, post, pre = int(rng.integers(3)), bool(rng.integers(2)), bool(rng.integers(2))
    what = ("norm", T, d, fp16, wide, wide_w, kind, post, pre)
    print(what, flush=True)
    dt, ds, dw = H.FP16 if fp16 else H.BF16, H.FP32 if wide else (H.FP16 if fp16 else H.BF16), H.FP32 if wide_w else (H.FP16 if fp16 else H.BF16)

    def either(shape, as32, scale=1.0):
        if as32:
            v = (rng.standard_normal(shape) * scale).astype(np.float32)
            return H.G(v), v.astype(np.float64)
        return data(rng, shape, fp16, scale)

    (y, yf), (gz, gzf) = data(rng, (T, d), fp16, 2), data(rng, (T, d), fp16, 0.3)
    (res, rf), (gh, ghf) = either((T, d), wide, 3), either((T, d), wide, 0.3)
    wp, wpf = either((d,), wide_w) if post else (None, np.ones(d))
    wn, wnf = either((d,), wide_w) if pre else (None, None)
    gt, gtf = either((d,), wide_w) if kind == 1 else either((T,), wide_w) if kind == 2 else (None, np.ones(1))
    gtf = gtf[:, None] if kind == 2 else gtf

    def out(shape, as32):
        return H._full(shape, np.nan, np.float32) if as32 else H._full(shape, H.NAN16, np.uint16)

    h, z = out((T, d), wide), out((T, d), False) if pre else None
    H.ok(L.moe_gg_block_norm(P(y), d, P(res), d, P(wp), P(gt), kind, P(wn), 0.9, 0.5, 1e-6, P(h), P(z), T, d, dt, ds, dw, None))
    ry = 1 / np.sqrt((yf * yf).mean(1, keepdims=True) + 1e-6) if post else 1.0
    n = yf * ry * wpf
    hw = 0.9 * rf + 0.5 * gtf * n
    near(h, hw, fp16, what + ("h",))
    if pre:
        rh = 1 / np.sqrt((hw * hw).mean(1, keepdims=True) + 1e-6)
        near(z, hw * rh * wnf, fp16, what + ("z",))
    gy, gr = out((T, d), False), out((T, d), wide)
    gpost, gpre = out((d,), wide_w) if post else None, out((d,), wide_w) if pre else None
    ggate = out((d,), wide_w) if kind == 1 else out((T,), wide_w) if kind == 2 else None
    nb = L.moe_gg_block_norm_backward_workspace(T, d)
    H.ok(L.moe_gg_block_norm_backward(P(gh), d, P(gz) if pre else None, d, P(y), d, P(h), d, P(wp), P(gt), kind, P(wn), 0.9, 0.5, 1e-6, P(gy), P(gr), P(gpost), P(ggate),
                                      P(gpre), T, d, dt, ds, dw, work(nb), nb, None))
    hs = h.astype(np.float64) if wide else H.from16(h, fp16).astype(np.float64)
    tot = ghf.copy()
    if pre:
        rh = 1 / np.sqrt((hs * hs).mean(1, keepdims=True) + 1e-6)
        g = gzf * wnf
        tot += rh * (g - hs * rh * (g * hs * rh).mean(1, keepdims=True))
        near(gpre, (gzf * hs * rh).sum(0), fp16, what + ("gpre",))
    near(gr, 0.9 * tot, fp16, what + ("gres",))
    bt = 0.5 * tot
    g = bt * gtf * wpf
    yn = yf * ry
    # for a width of 1 the normed row does not depend on y: the two terms of the gradient cancel but for eps
    near(gy, ry * (g - yn * (g * yn).mean(1, keepdims=True)) if post else g, fp16, what + ("gy",),
         ry * (abs(g) + abs(yn) * abs(g * yn).mean(1, keepdims=True)))
    if post:
        near(gpost, (bt * gtf * yf * ry).sum(0), fp16, what + ("gpost",))
    if kind:
        near(ggate, (bt * n).sum(0 if kind == 1 else 1), fp16, what + ("ggate",))


def c_gate(rng):
    L = H.lib()
    T, E = int(rng.integers(1, 60)), int(rng.choice([1, 3, 8, 9, 16, 31, 64, 65, 128, 200, 256, 300, 768]))
    k = int(rng.integers(1, min(E, 64) + 1))
    score, renorm, dt = int(rng.integers(2)), int(rng.integers(2)), int(rng.integers(3))
    print(("gate", T, E, k, score, renorm, dt), flush=True)
    v = rng.standard_normal((T, E)).astype(np.float32) * 2
    raw = v if dt == 2 else H.to16(v, dt == 1)
    v = v.astype(np.float64) if dt == 2 else H.from16(raw, dt == 1).astype(np.float64)
    w, ids = H._full((T, k), np.nan, np.float32), H._full((T, k), -7, np.int32)
    H.ok(L.moe_gg_route_gate(P(raw), dt, T, E, k, score, renorm, 1.5, P(w), P(ids), None))
    want = np.argsort(-v, axis=1, kind="stable")[:, :k]
    assert (ids == want).all()
    p = 1 / (1 + np.exp(-v)) if score else np.exp(v - v.max(1, keepdims=True)) / np.exp(v - v.max(1, keepdims=True)).sum(1, keepdims=True)
    of = np.take_along_axis(p, want, 1)
    assert np.allclose(w, 1.5 * of / (of.sum(1, keepdims=True) if renorm else 1), rtol=1e-4, atol=0)
    g = H._full((T, E), np.nan, np.float32) if dt == 2 else H._full((T, E), H.NAN16, np.uint16)
    gw = rng.standard_normal((T, k)).astype(np.float32)
    if rng.random() < 0.3:
        ids[...] = rng.integers(-3, E + 3, ids.shape)
    H.ok(L.moe_gg_route_gate_backward(P(gw), P(raw), dt, P(ids), T, E, k, score, renorm, 1.5, P(g), None))
    assert np.isfinite(g if dt == 2 else H.from16(g, dt == 1)).all()


def main(seed, cases, wide=False):
    rng = np.random.default_rng(seed)
    for shape in ((1090, 4099, 40, 16, 3), (1090, 24, 4100, 20, 2), (1090, 4096, 17, 36, 2), (1090, 2056, 2050, 72, 2)) if wide else ():
        c_lora(rng, shape)
        H.release()
    for _ in range(cases):
        (c_lora, c_norm, c_gate)[int(rng.integers(3))](rng)
        H.release()
    print("done", cases)


if __name__ == "__main__":
    main(int(sys.argv[1]), int(sys.argv[2]), "wide" in sys.argv[3:])
