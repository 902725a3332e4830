"""The norms and the recurrence over tensors of more than 2^32 bytes, and the
feed-forward block over the largest it takes, in pieces, against float64 on the GPU.

Bounds are counts of roundings (2^-24) of the sums of the terms' absolute values,
as at small sizes: norms 24 and, for gradients, 64 (sums over a million rows are in
chains of about 1000 and 64 more, whose roundings grow as their root: 128);
recurrence: 8 of each step's terms, carried on by the gates as the state is (a step
checked on its own results would not do: a run of tokens starts from a state that was
worked out beside the written one, and the two differ by the roundings of all earlier
terms, which do not cancel where the terms do);
feed-forward: sqrt(K) + 8 for K terms.
"""
import math

import pytest
import torch   # ahead of the engine, which then shares its HIP runtime

from tests.test_gpu_long_tensors import filled, view

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


def pieces(n, by=50_000):
    return [slice(i, min(i + by, n)) for i in range(0, n, by)]


def test_residual_norm_over_a_long_tensor(eng):
    M, C = 1_050_001, 1025
    assert M * C * 4 > 2 ** 32
    print("residual_norm over", M, "rows", flush=True)
    x, b, dn = filled(eng, (M, C), 1, True), filled(eng, (M, C), 2, True), filled(eng, (M, C), 3)
    gate, post, pre = (filled(eng, (C,), 4 + i, True) for i in range(3))
    h, n = eng.residual_norm(x, b, gate, post, pre, 0.5)
    h.grad = dn
    n.backward(dn)
    eng.sync_gpu()
    X, B, DN, H, N, DX, DB = (view(t) for t in (x, b, dn, h, n, x.grad, b.grad))
    g, p, q = (view(t).double() for t in (gate, post, pre))
    sums = {k: [torch.zeros(C, dtype=torch.float64, device="cuda") for _ in range(2)] for k in ("gate", "post", "pre")}

    def ok(got, want, size, count):
        assert ((got - want).abs() <= count * EPS * size).all()
    for s in pieces(M):
        xs, bs, dn_s = X[s].double(), B[s].double(), DN[s].double()
        r1 = torch.rsqrt((bs * bs).mean(1, keepdim=True) + 1e-6)
        u = bs * r1 * p
        hs, size = 0.5 * xs + g * u, 0.5 * xs.abs() + (g * u).abs()
        ok(H[s], hs, size, 24)
        r2 = torch.rsqrt((hs * hs).mean(1, keepdim=True) + 1e-6)
        rel = 1 + (hs.abs() * size).mean(1, keepdim=True) * r2 * r2
        ok(N[s], hs * r2 * q, (size + hs.abs() * rel) * r2 * q.abs(), 24)
        w = q * dn_s
        t = dn_s + r2 * (w - hs * r2 * r2 * (w * hs).mean(1, keepdim=True))
        T = dn_s.abs() + r2 * rel * (w.abs() + size * r2 * r2 * (w.abs() * size).mean(1, keepdim=True))
        ok(DX[s], 0.5 * t, 0.5 * T, 64)
        du, DU = g * t, g.abs() * T
        v, V = p * du, p.abs() * DU
        ok(DB[s], r1 * (v - bs * r1 * r1 * (v * bs).mean(1, keepdim=True)),
           r1 * (V + bs.abs() * r1 * r1 * (V * bs.abs()).mean(1, keepdim=True)), 64)
        for k, a, c in (("gate", t * u, T * u.abs()), ("post", du * bs * r1, DU * bs.abs() * r1),
                        ("pre", dn_s * hs * r2, dn_s.abs() * size * r2 * rel)):
            sums[k][0] += a.sum(0)
            sums[k][1] += c.sum(0)
    for k, t in (("gate", gate), ("post", post), ("pre", pre)):
        ok(view(t.grad).view(-1), *sums[k], 128)
    eng.end_batch()
    torch.cuda.empty_cache()


def linear(f, v, start):
    """h_t = f_t h_(t-1) + v_t along the first dimension, by doubling."""
    f, v = f.clone(), v.clone()
    v[0] += f[0] * start
    d = 1
    while d < len(v):
        v[d:] += f[d:] * v[:-d].clone()
        f[d:] *= f[:-d].clone()
        d *= 2
    return v


def after(first, rows):
    return torch.cat([first[None], rows[:-1]])


def test_gated_scan_over_a_long_tensor(eng):
    S, C = 1_050_001, 1030
    assert S * C * 4 > 2 ** 32
    print("gated_scan over", S, "tokens", flush=True)
    x, z, dy = filled(eng, (1, S, C), 1, True), filled(eng, (1, S, C), 2, True), filled(eng, (1, S, C), 3)
    y, last = eng.gated_scan(x, z, return_state=True)
    y.backward(dy)
    eng.sync_gpu()
    X, Z, DY, Y, DX, DZ = (view(t)[0] for t in (x, z, dy, y, x.grad, z.grad))
    assert torch.equal(view(last)[0], Y[-1])
    every = pieces(S, 20_000)
    # the state ahead of each piece, and its bound
    h = e = torch.zeros(C, dtype=torch.float64, device="cuda")
    ahead = []
    for s in every:
        ahead.append((h, e))
        f, kx = torch.sigmoid(Z[s].double()), torch.sigmoid(-Z[s].double()) * X[s].double()
        ys = linear(f, kx, h)
        es = linear(f, 8 * EPS * ((f * after(h, ys)).abs() + kx.abs()), e)
        assert ((Y[s] - ys).abs() <= es).all(), s
        h, e = ys[-1], es[-1]
    back = eb = torch.zeros(C, dtype=torch.float64, device="cuda")   # what later tokens hand to the piece's last one
    for s, (h, e) in zip(every[::-1], ahead[::-1]):
        xs, ds = X[s].double(), DY[s].double()
        f, k = torch.sigmoid(Z[s].double()), torch.sigmoid(-Z[s].double())
        ys = linear(f, k * xs, h)
        es = linear(f, 8 * EPS * ((f * after(h, ys)).abs() + (k * xs).abs()), e)
        before, e_before = after(h, ys), after(e, es)
        # d_t = dy_t + f_(t+1) d_(t+1): in reverse, with each token's gate that of the token behind it
        fr, dr = f.flip(0), ds.flip(0)
        gates = after(torch.ones_like(back), fr)
        d = linear(gates, dr, back)
        came = gates * after(back, d)
        ed = linear(gates, EPS * (dr.abs() + came.abs()) + gates * 8 * EPS * after(back, d).abs(), eb)
        back, eb = fr[-1] * d[-1], fr[-1] * (ed[-1] + 8 * EPS * d[-1].abs())
        d, ed = d.flip(0), ed.flip(0)
        assert ((DX[s] - k * d).abs() <= k * (ed + 8 * EPS * d.abs())).all(), s
        tol = f * k * (ed * (before - xs).abs() + d.abs() * (e_before + 12 * EPS * (before.abs() + xs.abs())))
        assert ((DZ[s] - d * (before - xs) * f * k).abs() <= tol).all(), s
    eng.end_batch()
    torch.cuda.empty_cache()


def test_gated_mlp_at_its_largest(eng):
    M, C, F = 520_728, 64, 1031   # just below the 2^29 values a tensor may have; all of them together have more
    assert 2 ** 29 - F < M * F < 2 ** 29 and 3 * M * F * 4 > 2 ** 32
    print("gated_mlp over", M, "rows", flush=True)
    x, dy = filled(eng, (M, C), 1, True), filled(eng, (M, C), 2)
    W = [filled(eng, s, 3 + i, True) for i, s in enumerate(((C, F), (C, F), (F, C)))]
    y = eng.gated_mlp(x, *W)
    y.backward(dy)
    eng.sync_gpu()
    X, DY, Y, DX = (view(t) for t in (x, dy, y, x.grad))
    wg, wu, wd = (view(t).double() for t in W)
    sums = [[torch.zeros(s, dtype=torch.float64, device="cuda") for _ in range(2)] for s in ((C, F), (C, F), (F, C))]

    def k(n):
        return (math.sqrt(n) + 8) * EPS
    for s in pieces(M, 20_000):
        xs, ds = X[s].double(), DY[s].double()
        ax, ad = xs.abs(), ds.abs()
        g, u = xs @ wg, xs @ wu
        eg, eu = k(C) * (ax @ wg.abs()), k(C) * (ax @ wu.abs())
        p = torch.sigmoid(g)
        a, da = g * p, p + g * p * (1 - p)
        ea, eda = 1.13 * eg + 16 * EPS * a.abs(), 1.13 * eg + 16 * EPS * (1 + g.abs())
        m = a * u
        em = ea * u.abs() + a.abs() * eu + ea * eu + EPS * m.abs()
        assert ((Y[s] - m @ wd).abs() <= em @ wd.abs() + k(F) * (m.abs() @ wd.abs())).all(), s
        dm, edm = ds @ wd.t(), k(C) * (ad @ wd.abs().t())
        dg, du = dm * u * da, dm * a
        edg = edm * (u * da).abs() + (dm.abs() + edm) * (eu * da.abs() + (u.abs() + eu) * eda) + 3 * EPS * dg.abs()
        edu = edm * a.abs() + (dm.abs() + edm) * ea + 2 * EPS * du.abs()
        tol = edg @ wg.abs().t() + edu @ wu.abs().t() + k(2 * F) * (dg.abs() @ wg.abs().t() + du.abs() @ wu.abs().t())
        assert ((DX[s] - (dg @ wg.t() + du @ wu.t())).abs() <= tol).all(), s
        for i, (l, v, ev) in enumerate(((xs, dg, edg), (xs, du, edu), (m, ds, None))):
            sums[i][0] += l.t() @ v
            sums[i][1] += (l.abs().t() @ ev if ev is not None else em.t() @ ad) + k(M) * (l.abs().t() @ v.abs())
    for t, (want, tol) in zip(W, sums):
        assert ((view(t.grad) - want).abs() <= tol).all()
    eng.end_batch()
    torch.cuda.empty_cache()
