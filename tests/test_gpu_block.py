"""The norms around a residual stream, the gated feed-forward block and the
gated recurrence, with their gradients, against plain float64 implementations.

Every bound is element by element: the reference is worked out a second time
with the absolute values of all terms, which gives for each result the sum of
what was added up to it, and a result may be off by a count of roundings (eps =
2^-24, fp32's half step) of that sum:
  norms: a row's sum of squares is added up over at most 16 values a thread and
    a tree of 10, and its root halves the error: 16; a product or two and a sum
    each around it: 24 for the forward, and twice for the gradients, which go
    through both norms and a row's mean more: 64.  Sums over rows: chains of at
    most 64 rows beside that, whose roundings grow as their root: 64 too.
  recurrence: a step adds a rounding to f, 1 - f and x's product each, and the
    gates have at most 4 of their own: 8 of the step's terms, carried on by f as
    the state is.
  feed-forward: a dot product of K terms in chains: sqrt(K) + 8 of the sum of
    its terms' absolute values; the activations' slopes are at most 1.13.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from tests.helpers import rng

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


def dev(eng, a, grad=False):
    return eng.Tensor(np.array(a, np.float32), requires_grad=grad, track=False)


def within(name, got, ref, bound):
    """|got - ref| <= bound everywhere."""
    got = np.asarray(got, np.float64)
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert np.isfinite(got).all(), name
    bad = np.abs(got - ref) - bound - 1e-37
    i = np.unravel_index(np.argmax(bad), bad.shape)
    assert bad[i] <= 0, f"{name}{i}: {got[i]!r} for {ref[i]!r}, {abs(got[i] - ref[i]):.3g} off, {np.broadcast_to(bound, ref.shape)[i]:.3g} allowed"


# -------------------------------------------------------------------- norms
def norm64(x, b, gate, post, pre, scale, eps, dh, dn):
    """Results and gradients {name: (value, sum of the terms' absolute values)} of rows (M, C)."""
    M, C = x.shape
    A = np.abs
    G = np.ones((1, C)) if gate is None else gate.reshape(-1, C)
    R = G.shape[0]
    g = np.repeat(G, M // R, 0)
    r1 = 1 / np.sqrt((b * b).mean(1, keepdims=True) + eps) if post is not None else np.ones((M, 1))
    u = b * r1 * (post if post is not None else 1.0)
    h = scale * x + g * u
    H = A(scale * x) + A(g * u)
    out = {"h": (h, H)}
    r2 = 1 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    # what an error of h does to r2: at most mean(|h| H) r2^2 of it
    rel = 1 + (A(h) * H).mean(1, keepdims=True) * r2 * r2
    if pre is not None:
        out["n"] = (h * r2 * pre, (H + A(h) * rel) * r2 * A(pre))
    t, T = (np.zeros_like(x),) * 2 if dh is None else (dh, A(dh))
    if dn is not None:
        w = pre * dn
        t = t + r2 * (w - h * r2 * r2 * (w * h).mean(1, keepdims=True))
        T = T + r2 * rel * (A(w) + H * r2 * r2 * (A(w) * H).mean(1, keepdims=True))
        out["dpre"] = ((dn * h * r2).sum(0), (A(dn) * H * r2 * rel).sum(0))
    out["dx"] = (scale * t, A(scale) * T)
    tu, TU = t * u, T * A(u)
    out["dgate"] = (tu.reshape(R, M // R, C).sum(1), TU.reshape(R, M // R, C).sum(1))
    du, DU = g * t, A(g) * T
    if post is not None:
        out["dpost"] = ((du * b * r1).sum(0), (DU * A(b) * r1).sum(0))
        w, W = post * du, A(post) * DU
        du = r1 * (w - b * r1 * r1 * (w * b).mean(1, keepdims=True))
        DU = r1 * (W + A(b) * r1 * r1 * (W * A(b)).mean(1, keepdims=True))
    out["dblock"] = (du, DU)
    return out


def check_norm(eng, batch, seq, width, gate, post, pre, scale, r, grads="hn", sizes=None, eps=1e-6):
    """grads: which of the results have gradients."""
    M = batch * seq
    shape = (batch, seq, width)
    a = {"x": 3 * r.standard_normal(shape), "block": r.standard_normal(shape)}
    if gate:
        a["gate"] = r.standard_normal({"channel": (width,), "sequence": (batch, width), "token": shape}[gate])
    if post:
        a["post"] = 1 + 0.3 * r.standard_normal(width)
    if pre:
        a["pre"] = 1 + 0.3 * r.standard_normal(width)
    if sizes is not None:  # rows of very different size
        f = sizes(r, M).reshape(batch, seq, 1)
        a["x"], a["block"] = a["x"] * f, a["block"] * f
    a = {k: v.astype(np.float32) for k, v in a.items()}
    dh, dn = (r.standard_normal(shape).astype(np.float32) for _ in range(2))
    T = {k: dev(eng, v, True) for k, v in a.items()}
    got = eng.residual_norm(T["x"], T["block"], T.get("gate"), T.get("post"), T.get("pre"), scale, eps)
    h, n = got if pre else (got, None)
    use_h, use_n = "h" in grads or not pre, "n" in grads and bool(pre)
    if use_n:
        if use_h:
            h.grad = dev(eng, dh)
        n.backward(dev(eng, dn))
    else:
        h.backward(dev(eng, dh))

    def rows(k):
        return a[k].astype(np.float64).reshape(-1, width) if k in a else None
    ref = norm64(rows("x"), rows("block"), rows("gate"), a["post"].astype(np.float64) if post else None,
                 a["pre"].astype(np.float64) if pre else None, scale, eps,
                 dh.astype(np.float64).reshape(M, width) if use_h else None,
                 dn.astype(np.float64).reshape(M, width) if use_n else None)

    def match(name, t, count):
        v, s = ref[name]
        within(name, t.sync().reshape(v.shape), v, count * EPS * s)
    match("h", h, 24)
    if pre:
        match("n", n, 24)
    for k, t in T.items():
        if k == "pre" and not use_n:
            assert t.grad is None
            continue
        assert tuple(t.grad.shape) == tuple(t.shape)
        match("d" + k, t.grad, 64)
    eng.end_batch()


@pytest.mark.parametrize("width", [1, 3, 4, 5, 31, 64, 255, 256, 257, 512, 771, 1024, 1030, 2048, 4096, 4099, 8192, 16384])
@pytest.mark.parametrize("gate,post,pre", [(None, 0, 1), ("channel", 1, 1), ("sequence", 1, 0), ("token", 0, 1), ("token", 1, 1)])
def test_residual_norm(eng, width, gate, post, pre):
    print("residual_norm", width, gate, post, pre, flush=True)
    check_norm(eng, 3, 5, width, gate, post, pre, 0.75, rng(width))


@pytest.mark.parametrize("batch,seq,width,gate", [
    (1, 1, 2048, "channel"), (1, 1, 7, "token"), (8, 1, 300, "sequence"), (2, 1501, 64, "channel"), (700, 3, 96, "sequence"),
    (2, 2100, 40, "sequence"), (5, 601, 130, "token"), (1, 3000, 520, None), (1100, 2, 16, "sequence"), (2, 700, 2052, "channel")])
def test_residual_norm_over_many_rows(eng, batch, seq, width, gate):
    """Rows in several workgroups, whole gate rows in one, pieces that do not come out even."""
    print("residual_norm rows", batch, seq, width, gate, flush=True)
    check_norm(eng, batch, seq, width, gate, 1, 1, 1.0, rng(batch + seq))


@pytest.mark.parametrize("grads", ["h", "n"])
def test_residual_norm_with_one_gradient(eng, grads):
    check_norm(eng, 2, 9, 100, "channel", 1, 1, 0.5, rng(8), grads=grads)


def test_residual_norm_of_rows_of_all_sizes(eng):
    check_norm(eng, 2, 40, 260, "channel", 1, 1, 1.0, rng(9), sizes=lambda r, m: 10.0 ** r.uniform(-12, 12, m))


def test_residual_norm_of_zeros(eng):
    """A row of zeros has the factor 1 / sqrt(eps) and stays zeros."""
    z = np.zeros((4, 64))
    x, b, g = dev(eng, z, True), dev(eng, z, True), dev(eng, np.ones(64), True)
    h, n = eng.residual_norm(x, b, post=g, pre=g)
    n.backward(dev(eng, np.ones((4, 64))))
    assert not h.sync().any() and not n.sync().any() and not g.grad.sync().any()
    # d n / d h = 1 / sqrt(eps), d h / d block likewise
    assert np.allclose(x.grad.sync(), 1e3, rtol=1e-6) and np.allclose(b.grad.sync(), 1e6, rtol=1e-6)
    eng.end_batch()


@pytest.mark.parametrize("rows,width", [(1, 1), (1, 64), (7, 33), (300, 512), (1000, 771), (5, 5000)])
def test_rms_norm(eng, rows, width):
    r = rng(rows + width)
    x, gain, dy = (r.standard_normal(s).astype(np.float32) for s in ((rows, width), width, (rows, width)))
    xt, gt = dev(eng, x, True), dev(eng, gain, True)
    y = eng.rms_norm(xt, gt, eps=1e-5)
    y.backward(dev(eng, dy))
    ref = norm64(x.astype(np.float64), np.zeros((rows, width)), None, None, gain.astype(np.float64), 1.0, 1e-5, None,
                 dy.astype(np.float64))
    for name, t, c in (("n", y, 24), ("dx", xt.grad, 64), ("dpre", gt.grad, 64)):
        v, s = ref[name]
        within(name, t.sync(), v, c * EPS * s)
    eng.end_batch()


def test_norm_gradients_against_differences(eng):
    """Along a random direction of all operands, central differences in float64
    of the formula: what the steps' products leave is below 1e-6 of the slope's
    terms."""
    r = rng(77)
    shape, step = (2, 3, 20), 1e-4
    a = {"x": r.standard_normal(shape), "block": r.standard_normal(shape), "gate": r.standard_normal((2, 20)),
         "post": 1 + r.random(20), "pre": 1 + r.random(20)}
    a = {k: v.astype(np.float32) for k, v in a.items()}
    dh, dn = (r.standard_normal(shape).astype(np.float32) for _ in range(2))
    T = {k: dev(eng, v, True) for k, v in a.items()}
    h, n = eng.residual_norm(T["x"], T["block"], T["gate"], T["post"], T["pre"], 0.5, 1e-3)
    h.grad = dev(eng, dh)
    n.backward(dev(eng, dn))
    way = {k: r.standard_normal(v.shape) for k, v in a.items()}

    def value(s):
        b = {k: v.astype(np.float64) + s * way[k] for k, v in a.items()}
        f = norm64(b["x"].reshape(6, 20), b["block"].reshape(6, 20), b["gate"], b["post"], b["pre"], 0.5, 1e-3, None, None)
        return (f["h"][0] * dh.reshape(6, 20)).sum() + (f["n"][0] * dn.reshape(6, 20)).sum()
    slope = (value(step) - value(-step)) / (2 * step)
    terms = {k: T[k].grad.sync().astype(np.float64) * way[k] for k in a}
    assert abs(sum(t.sum() for t in terms.values()) - slope) <= 1e-6 * sum(np.abs(t).sum() for t in terms.values())
    eng.end_batch()


def test_residual_norm_operands_that_need_no_gradient(eng):
    r = rng(12)
    for need in ("x", "block", "gate", "post", "pre"):
        T = {k: dev(eng, r.standard_normal(s), k == need) for k, s in
             (("x", (6, 40)), ("block", (6, 40)), ("gate", (40,)), ("post", (40,)), ("pre", (40,)))}
        h, n = eng.residual_norm(T["x"], T["block"], T["gate"], T["post"], T["pre"])
        assert n.requires_grad and h.requires_grad == (need != "pre")
        n.backward(dev(eng, np.ones((6, 40))))
        assert all((t.grad is not None) == (k == need) for k, t in T.items())
        eng.end_batch()
    h, n = eng.residual_norm(*(dev(eng, r.standard_normal((6, 40))) for _ in range(2)), pre=dev(eng, np.ones(40)))
    assert not h.requires_grad and not n.requires_grad


def test_the_same_tensor_twice(eng):
    """x as its own block and its own gate: three gradients for one leaf."""
    x0 = rng(4).standard_normal((5, 24)).astype(np.float32)
    x = dev(eng, x0, True)
    eng.residual_norm(x, x, gate=x).backward(dev(eng, np.ones((5, 24))))
    x64 = x0.astype(np.float64)
    within("dx", x.grad.sync(), 1 + 2 * x64, 16 * EPS * (1 + 2 * np.abs(x64)))
    eng.end_batch()


def test_norm_refusals(eng):
    x, g = dev(eng, np.zeros((4, 6))), dev(eng, np.zeros(6))
    for bad in (lambda: eng.rms_norm(x, dev(eng, np.zeros(5))), lambda: eng.rms_norm(x, dev(eng, np.zeros((6, 1)))),
                lambda: eng.residual_norm(x, dev(eng, np.zeros((6, 4)))), lambda: eng.residual_norm(x, x, pre=x),
                lambda: eng.residual_norm(x, x, post=dev(eng, np.zeros(7))),
                lambda: eng.residual_norm(x, x, gate=dev(eng, np.zeros((3, 6)))),
                lambda: eng.residual_norm(x, x, gate=dev(eng, np.zeros((4, 3))))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="16384"):
        eng.rms_norm(dev(eng, np.zeros((1, 16385))), dev(eng, np.zeros(16385)))
    lib, b, st, n = eng.lib, x.gpu_buf, ctypes.c_void_p(), ctypes.c_void_p()
    assert not lib.RmsNorm(b, g.gpu_buf, 5, 6, 1e-6, None)
    assert not lib.RmsNorm(b, g.gpu_buf, 0, 6, 1e-6, None)
    assert not lib.RmsNorm(b, None, 4, 6, 1e-6, None)
    assert not lib.ResidualNorm(b, None, None, None, None, 4, 6, 0, 1.0, 1e-6, None, None)
    assert not lib.ResidualNorm(b, b, g.gpu_buf, None, None, 4, 6, 0, 1.0, 1e-6, None, None)
    assert not lib.ResidualNorm(b, b, None, None, g.gpu_buf, 4, 6, 0, 1.0, 1e-6, None, None)
    assert not lib.ResidualNorm(b, b, None, None, None, 4, 6, 0, 1.0, 1e-6, ctypes.byref(n), ctypes.byref(st))
    assert not n.value and not st.value
    got = ctypes.c_void_p(1)
    lib.ResidualNormBackward(None, None, b, b, None, None, None, None, 4, 6, 0, 1.0, ctypes.byref(got), None, None, None, None)
    assert got.value is None
    lib.ResidualNormBackward(None, b, b, b, None, None, g.gpu_buf, g.gpu_buf, 4, 6, 0, 1.0, ctypes.byref(got), None, None, None, None)
    assert got.value is None and "stats" in eng.last_error()
    lib.ClearLastError()


# ------------------------------------------------------------- feed-forward
def act64(g, act):
    """act(g), its derivative."""
    if act == "relu":
        return np.maximum(g, 0), (g > 0) * 1.0
    t = torch.tensor(g, requires_grad=True)
    y = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid}[act](t)
    y.sum().backward()
    return y.detach().numpy(), t.grad.numpy()


def mlp64(x, wg, wu, wd, act, dy):
    """Results and gradients {name: (value, bound)}."""
    A = np.abs
    C, F = wg.shape
    M, O = x.shape[0], wd.shape[1]

    def k(n):
        return (math.sqrt(n) + 8) * EPS
    g, u = x @ wg, x @ wu
    eg, eu = k(C) * (A(x) @ A(wg)), k(C) * (A(x) @ A(wu))
    a, da = act64(g, act)
    # slopes of the activations and of their derivatives are at most 1.13; a step at relu's corner
    ea = 1.13 * eg + 16 * EPS * (A(a) + A(g) * (act == "gelu"))
    eda = (np.where(A(g) <= eg, 1.0, 0.0) if act == "relu" else 1.13 * eg + 16 * EPS * (1 + A(g)))
    m = a * u
    em = ea * A(u) + A(a) * eu + ea * eu + EPS * A(m)
    out = {"y": (m @ wd, em @ A(wd) + k(F) * (A(m) @ A(wd)))}
    dm = dy @ wd.T
    edm = k(O) * (A(dy) @ A(wd).T)
    dg, du = dm * u * da, dm * a
    edg = edm * A(u * da) + (A(dm) + edm) * (eu * A(da) + (A(u) + eu) * eda) + 3 * EPS * A(dg)
    edu = edm * A(a) + (A(dm) + edm) * ea + 2 * EPS * A(du)
    out["dwd"] = (m.T @ dy, em.T @ A(dy) + k(M) * (A(m).T @ A(dy)))
    out["dwg"] = (x.T @ dg, A(x).T @ edg + k(M) * (A(x).T @ A(dg)))
    out["dwu"] = (x.T @ du, A(x).T @ edu + k(M) * (A(x).T @ A(du)))
    out["dx"] = (dg @ wg.T + du @ wu.T,
                 edg @ A(wg).T + edu @ A(wu).T + k(2 * F) * (A(dg) @ A(wg).T + A(du) @ A(wu).T))
    return out


def check_mlp(eng, rows, width, hidden, out, act, r, need=("x", "wg", "wu", "wd"), change=None):
    a = {"x": r.standard_normal((rows, width)), "wg": r.standard_normal((width, hidden)) / math.sqrt(width),
         "wu": r.standard_normal((width, hidden)) / math.sqrt(width), "wd": r.standard_normal((hidden, out)) / math.sqrt(hidden),
         "dy": r.standard_normal((rows, out))}
    if change:
        change(a)
    a = {k: v.astype(np.float32) for k, v in a.items()}
    T = {k: dev(eng, a[k], k in need) for k in ("x", "wg", "wu", "wd")}
    y = eng.gated_mlp(T["x"], T["wg"], T["wu"], T["wd"], act)
    ref = mlp64(*(a[k].astype(np.float64) for k in ("x", "wg", "wu", "wd")), act, a["dy"].astype(np.float64))
    within("y", y.sync(), *ref["y"])
    if need:
        y.backward(dev(eng, a["dy"]))
    for k, t in T.items():
        assert (t.grad is not None) == (k in need), k
        if k in need:
            within("d" + k, t.grad.sync(), *ref["d" + k])
    eng.end_batch()


MLP_SIZES = [(1, 1, 1, 1), (1, 64, 100, 64), (2, 7, 5, 3), (8, 128, 344, 128), (16, 130, 77, 61), (17, 64, 64, 64), (33, 100, 257, 40),
             (77, 96, 192, 96), (154, 63, 130, 65), (200, 256, 512, 256), (257, 129, 513, 127), (1000, 64, 96, 48)]


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("size", MLP_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_gated_mlp(eng, size, act):
    print("gated_mlp", size, act, flush=True)
    check_mlp(eng, *size, act, rng(sum(size)))


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 15, 16, 24, 32, 40])
def test_gated_mlp_of_a_few_tokens(eng, rows):
    """Without gradients, as a program that answers calls it."""
    check_mlp(eng, rows, 1024, 1416, 1024, "silu", rng(rows), need=())


@pytest.mark.parametrize("size", [(700, 512, 1400, 512), (1024, 640, 1024, 384), (1500, 400, 1100, 404)], ids=lambda s: "x".join(map(str, s)))
def test_gated_mlp_of_large_calls(eng, size):
    print("gated_mlp", size, flush=True)
    check_mlp(eng, *size, "silu", rng(sum(size)))


@pytest.mark.parametrize("need", [("x",), ("wg",), ("wu",), ("wd",), ("x", "wd")])
@pytest.mark.parametrize("size", [(40, 48, 80, 56), (900, 512, 768, 512)], ids=lambda s: "x".join(map(str, s)))
def test_gated_mlp_gradients_asked_for(eng, size, need):
    check_mlp(eng, *size, "gelu", rng(3), need=need)


@pytest.mark.parametrize("rows", [6, 120, 1024])
def test_gated_mlp_of_rows_and_columns_of_all_sizes(eng, rows):
    """Tokens, gradients and weights whose sizes lie 2^30 and more apart."""
    r = rng(rows)

    def change(a):
        a["x"] *= 2.0 ** r.integers(-15, 3, (rows, 1))
        a["dy"] *= 2.0 ** r.integers(-20, 20, (rows, 1))
        a["wu"] *= 2.0 ** r.integers(-15, 15, (1, a["wu"].shape[1]))
        a["wd"] *= 2.0 ** r.integers(-15, 15, (1, a["wd"].shape[1]))
    check_mlp(eng, rows, 512, 640, 384, "silu", r, change=change)


@pytest.mark.parametrize("rows", [5, 130, 1024])
def test_gated_mlp_of_zeros(eng, rows):
    """Rows, columns and whole operands of zeros."""
    def change(a):
        a["x"][::2] = 0
        a["wg"][:, 3:9] = 0
        a["wd"][:, ::5] = 0
        a["dy"][1:4] = 0
    check_mlp(eng, rows, 384, 512, 256, "gelu", rng(rows), change=change)

    def all_zero(a):
        a["wu"][:] = 0
    check_mlp(eng, rows, 384, 512, 256, "gelu", rng(rows), change=all_zero)


@pytest.mark.parametrize("rows", [4, 200, 1024])
def test_gated_mlp_keeps_what_is_not_finite_in_its_row(eng, rows):
    """A token that holds a NaN, an infinity or one value of 1e15: other tokens' results stay as they are."""
    r = rng(rows)
    w = [dev(eng, r.standard_normal(s) / 16) for s in ((384, 512), (384, 512), (512, 384))]
    x = r.standard_normal((rows, 384)).astype(np.float32)
    want = eng.gated_mlp(dev(eng, x), *w).sync().copy()
    x[1, 7], x[2, 9], x[3, 11] = np.nan, np.inf, 1e15
    got = eng.gated_mlp(dev(eng, x), *w).sync()
    assert not np.isfinite(got[1:3]).any() and np.array_equal(got[0], want[0]) and np.array_equal(got[4:], want[4:])
    ref = mlp64(x[3:4].astype(np.float64), *(t.sync().astype(np.float64) for t in w), "silu", np.zeros((1, 384)))["y"]
    within("y", got[3:4], *ref)
    eng.end_batch()


def test_gated_mlp_in_three_dimensions(eng):
    r = rng(6)
    x, wg, wu, wd = (r.standard_normal(s).astype(np.float32) for s in ((2, 9, 32), (32, 48), (32, 48), (48, 20)))
    t = [dev(eng, v, True) for v in (x, wg, wu, wd)]
    y = eng.gated_mlp(*t)
    assert tuple(y.shape) == (2, 9, 20)
    y.backward(dev(eng, np.ones((2, 9, 20))))
    flat = [dev(eng, v, True) for v in (x.reshape(18, 32), wg, wu, wd)]
    z = eng.gated_mlp(*flat)
    z.backward(dev(eng, np.ones((18, 20))))
    assert np.array_equal(y.sync().reshape(18, 20), z.sync())
    assert all(np.array_equal(a.grad.sync().ravel(), b.grad.sync().ravel()) for a, b in zip(t, flat))
    eng.end_batch()


def test_gated_mlp_refusals(eng):
    def z(*s):
        return dev(eng, np.zeros(s))
    x, w, v = z(4, 6), z(6, 8), z(8, 6)
    for bad in (lambda: eng.gated_mlp(x, w, w, v, "tanh"), lambda: eng.gated_mlp(x, w, z(6, 7), v),
                lambda: eng.gated_mlp(x, z(5, 8), z(5, 8), v), lambda: eng.gated_mlp(x, w, w, z(7, 6)),
                lambda: eng.gated_mlp(x, w, w, z(8)), lambda: eng.gated_mlp(x, z(48), z(48), v)):
        with pytest.raises(ValueError):
            bad()
    lib, b = eng.lib, [t.gpu_buf for t in (x, w, w, v)]
    assert not lib.GatedMlpForward(*b, 4, 6, 8, 6, 4, None)
    assert not lib.GatedMlpForward(*b, 5, 6, 8, 6, 0, None)
    assert not lib.GatedMlpForward(*b, 4, 6, 9, 6, 0, None)
    assert not lib.GatedMlpForward(*b, 4, 6, 8, 7, 0, None)
    assert not lib.GatedMlpForward(*b, 0, 6, 8, 6, 0, None)
    assert not lib.GatedMlpForward(*b, 1 << 20, 6, 1 << 12, 6, 0, None)
    assert not lib.GatedMlpForward(b[0], None, b[2], b[3], 4, 6, 8, 6, 0, None)
    got = ctypes.c_void_p(1)
    lib.GatedMlpBackward(b[0], *b, b[0], 4, 6, 8, 6, 0, ctypes.byref(got), None, None, None)
    assert got.value is None and "saved" in eng.last_error()
    lib.ClearLastError()


# --------------------------------------------------------------- recurrence
def scan64(x, z, state, lens, dy):
    """Results and gradients {name: (value, bound)}, token by token."""
    B, S, C = x.shape
    A = np.abs
    with np.errstate(over="ignore"):
        f, k = 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))
    h = np.zeros((B, C)) if state is None else state.copy()
    e = np.zeros((B, C))
    y, before, eb, ey = (np.zeros_like(x) for _ in range(4))
    for t in range(S):
        live = (t < lens)[:, None]
        before[:, t], eb[:, t] = h, e
        n = f[:, t] * h + np.where(live, k[:, t] * x[:, t], 0)
        ne = f[:, t] * e + 8 * EPS * (A(f[:, t] * h) + np.where(live, A(k[:, t] * x[:, t]), 0))
        h, e = np.where(live, n, h), np.where(live, ne, e)
        y[:, t], ey[:, t] = np.where(live, h, 0), e
    out = {"y": (y, ey), "last": (h, e)}
    D, eD = np.zeros_like(x), np.zeros_like(x)
    back, e = np.zeros((B, C)), np.zeros((B, C))
    for t in reversed(range(S)):
        live = (t < lens)[:, None]
        d = np.where(live, dy[:, t] + back, 0)
        D[:, t], eD[:, t] = d, np.where(live, e + EPS * (A(dy[:, t]) + A(back)), 0)
        back, e = np.where(live, f[:, t] * d, back), np.where(live, f[:, t] * (eD[:, t] + 8 * EPS * A(d)), e)
    xs = np.where((np.arange(S)[None] < lens[:, None])[..., None], x, 0)
    out["dx"] = (k * D, k * (eD + 8 * EPS * A(D)))
    out["dz"] = (D * (before - xs) * f * k,
                 f * k * (eD * A(before - xs) + A(D) * (eb + 12 * EPS * (A(before) + A(xs)))))
    out["dstate"] = (back, e)
    return out


def check_scan(eng, B, S, C, with_state, lens, r, z=None, need=("x", "z", "state")):
    x, dy, state = (r.standard_normal(s).astype(np.float32) for s in ((B, S, C), (B, S, C), (B, C)))
    z = (2 + 1.5 * r.standard_normal((B, S, C)) if z is None else z).astype(np.float32)
    n = np.full(B, S) if lens is None else np.clip(np.nan_to_num(np.asarray(lens, np.float64)), 0, S).astype(int)
    pad = np.arange(S)[None] >= n[:, None]
    dirty = [v.copy() for v in (x, z, dy)]
    for v in dirty:
        v[pad] = np.nan  # nothing past the lengths may be read into a result
    T = {"x": dev(eng, dirty[0], "x" in need), "z": dev(eng, dirty[1], "z" in need)}
    if with_state:
        T["state"] = dev(eng, state, "state" in need)
    y, last = eng.gated_scan(T["x"], T["z"], T.get("state"), None if lens is None else dev(eng, lens), return_state=True)
    ref = scan64(*(v.astype(np.float64) for v in (x, z)), state.astype(np.float64) if with_state else None, n, dy.astype(np.float64))
    within("y", y.sync(), *ref["y"])
    within("last", last.sync(), *ref["last"])
    assert not y.sync()[pad].any() and not last.requires_grad
    if any(t.requires_grad for t in T.values()):
        y.backward(dev(eng, dirty[2]))
    for k, t in T.items():
        assert (t.grad is not None) == (k in need), k
        if k in need:
            v, b = ref["d" + k]
            within("d" + k, t.grad.sync(), v, b)
            if k != "state":
                assert not t.grad.sync()[pad].any()
    eng.end_batch()


@pytest.mark.parametrize("with_state", [False, True])
@pytest.mark.parametrize("B,S,C", [(1, 1, 1), (8, 1, 300), (2, 2, 64), (1, 7, 65), (3, 16, 130), (2, 17, 20), (1, 31, 64), (1, 64, 3), (2, 100, 96),
                                   (1, 127, 40), (1, 255, 33), (1, 257, 200), (2, 512, 64), (1, 513, 70), (3, 1000, 65), (1, 2049, 130), (1, 5000, 12)])
def test_gated_scan(eng, B, S, C, with_state):
    print("gated_scan", B, S, C, with_state, flush=True)
    check_scan(eng, B, S, C, with_state, None, rng(B + S + C))


@pytest.mark.parametrize("S,C,lens", [(40000, 3, None), (33000, 64, None), (20000, 7, [20000, 16385]), (50000, 2, [8192, 49999])])
def test_gated_scan_of_long_sequences(eng, S, C, lens):
    """Over more than the 64 workgroups from one state to the next."""
    print("gated_scan long", S, C, lens, flush=True)
    check_scan(eng, 2, S, C, True, lens, rng(S))


@pytest.mark.parametrize("S,lens", [(1, [0, 1, 1]), (9, [9, 0, 4]), (40, [1, 40, 33]), (300, [300, 17, 0]), (600, [256, 257, 600]), (1500, [1, 1024, 1030]),
                                    (30, [99, -4, float("nan")]), (700, [0, 0, 0])])
def test_gated_scan_of_lengths(eng, S, lens):
    print("gated_scan lengths", S, lens, flush=True)
    for with_state in (False, True):
        check_scan(eng, 3, S, 70, with_state, lens, rng(S))


@pytest.mark.parametrize("S", [5, 400, 3000])
def test_gated_scan_of_gates_at_their_ends(eng, S):
    """Gates of 0 and 1 to the last bit: a reset and a token that is passed over."""
    r = rng(S)
    z = r.choice([-np.inf, np.inf, -200.0, 200.0, -90.0, 30.0, 0.0], (2, S, 70), p=[0.02, 0.3, 0.02, 0.3, 0.02, 0.3, 0.04])
    check_scan(eng, 2, S, 70, True, None, r, z=z)


@pytest.mark.parametrize("need", [("x",), ("z",), ("state",)])
def test_gated_scan_gradients_asked_for(eng, need):
    check_scan(eng, 2, 600, 40, True, None, rng(1), need=need)


def test_gated_scan_goes_on_from_its_state(eng):
    """A sequence in pieces of 1 to 700 tokens, each from the state before."""
    r = rng(2)
    x, z = (r.standard_normal((2, 1200, 70)).astype(np.float32) for _ in range(2))
    ref = scan64(x.astype(np.float64), z.astype(np.float64), None, np.full(2, 1200), np.zeros((2, 1200, 70)))["y"]
    state, got, at = None, [], 0
    for n in (1, 1, 5, 700, 1, 492):
        y, state = eng.gated_scan(dev(eng, x[:, at:at + n]), dev(eng, z[:, at:at + n]), state, return_state=True)
        got.append(y.sync().copy())
        at += n
        del y
        eng.end_batch()  # leaves the state alone
    within("y", np.concatenate(got, 1), *ref)
    eng.end_batch()


def test_gated_scan_gradients_against_differences(eng):
    r = rng(5)
    x, z, s, dy = (r.standard_normal(v).astype(np.float32) for v in ((1, 40, 6), (1, 40, 6), (1, 6), (1, 40, 6)))
    T = [dev(eng, v, True) for v in (x, z, s)]
    eng.gated_scan(*T).backward(dev(eng, dy))
    way = [r.standard_normal(v.shape) for v in (x, z, s)]

    def value(t):
        a = [v.astype(np.float64) + t * w for v, w in zip((x, z, s), way)]
        return (scan64(*a, np.full(1, 40), np.zeros((1, 40, 6)))["y"][0] * dy).sum()
    slope = (value(1e-4) - value(-1e-4)) / 2e-4
    terms = [t.grad.sync().astype(np.float64) * w for t, w in zip(T, way)]
    assert abs(sum(t.sum() for t in terms) - slope) <= 1e-6 * sum(np.abs(t).sum() for t in terms)
    eng.end_batch()


def test_gated_scan_refusals(eng):
    def z(*s):
        return dev(eng, np.zeros(s))
    x = z(2, 5, 4)
    for bad in (lambda: eng.gated_scan(x, z(2, 5, 3)), lambda: eng.gated_scan(z(2, 5), z(2, 5)),
                lambda: eng.gated_scan(x, x, z(2, 5)), lambda: eng.gated_scan(x, x, lengths=z(3))):
        with pytest.raises(ValueError):
            bad()
    lib, b = eng.lib, x.gpu_buf
    assert not lib.GatedScanForward(b, b, None, None, 2, 5, 5, None)
    assert not lib.GatedScanForward(b, b, None, None, 0, 5, 4, None)
    assert not lib.GatedScanForward(b, None, None, None, 2, 5, 4, None)
    few = z(7)
    assert not lib.GatedScanForward(b, b, few.gpu_buf, None, 2, 5, 4, None)
    got = ctypes.c_void_p(1)
    lib.GatedScanBackward(b, few.gpu_buf, b, b, None, None, 2, 5, 4, ctypes.byref(got), None, None)
    assert got.value is None and "out" in eng.last_error()
    lib.ClearLastError()


# ------------------------------------------------------------------ together
WIDTH, HIDDEN, HEADS = 48, 80, 4


def block_params(r, classes):
    def w(*s):
        return (r.standard_normal(s) / math.sqrt(s[0])).astype(np.float32)
    P = {n: w(WIDTH, WIDTH) for n in ("wx", "wz", "wo", "wq", "wk", "wv", "wp")}
    P.update(g_in=w(WIDTH, HIDDEN), g_up=w(WIDTH, HIDDEN), g_down=w(HIDDEN, WIDTH), head=w(WIDTH, classes))
    for n in ("n0", "post1", "n1", "post2", "n2", "n3"):
        P[n] = (1 + 0.2 * r.standard_normal(WIDTH)).astype(np.float32)
    P["gate"] = (0.5 * r.standard_normal(WIDTH)).astype(np.float32)
    return P


def block(eng, P, x, table, B, S):
    """A recurrence, attention and a feed-forward block in one residual stream; logits."""
    def tokens(t, w):
        return eng.matmul(t, P[w])
    n = eng.rms_norm(x, P["n0"])
    y = eng.gated_scan(eng.reshape(tokens(n, "wx"), (B, S, WIDTH)), eng.reshape(tokens(n, "wz"), (B, S, WIDTH)))
    h, n = eng.residual_norm(x, tokens(eng.reshape(y, (B * S, WIDTH)), "wo"), P["gate"], P["post1"], P["n1"])
    q, k, v = (eng.reshape(tokens(n, w), (B, S, HEADS, WIDTH // HEADS)) for w in ("wq", "wk", "wv"))
    o = eng.attention(eng.rotary(q, table), eng.rotary(k, table), v, causal=True)
    h, n = eng.residual_norm(h, tokens(eng.reshape(o, (B * S, WIDTH)), "wp"), None, P["post2"], P["n2"])
    h, n = eng.residual_norm(h, eng.gated_mlp(n, P["g_in"], P["g_up"], P["g_down"]), pre=P["n3"], scale=0.5)
    return tokens(n, "head")


def block64(P, x, table, B, S):
    def norm(t, g):
        return t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * g
    n = norm(x, P["n0"])
    X, F = (n @ P["wx"]).view(B, S, -1), torch.sigmoid(n @ P["wz"]).view(B, S, -1)
    ys, s = [], torch.zeros(B, WIDTH, dtype=torch.float64)
    for t in range(S):
        s = F[:, t] * s + (1 - F[:, t]) * X[:, t]
        ys.append(s)
    h = x + P["gate"] * norm(torch.stack(ys, 1).reshape(B * S, -1) @ P["wo"], P["post1"])
    n = norm(h, P["n1"])
    q, k, v = ((n @ P[w]).view(B, S, HEADS, -1) for w in ("wq", "wk", "wv"))
    c, s = table[:S, None, :, 0], table[:S, None, :, 1]

    def spin(t):
        a, b = t.chunk(2, -1)
        return torch.cat([a * c - b * s, a * s + b * c], -1)
    sc = torch.matmul(spin(q).transpose(1, 2), spin(k).permute(0, 2, 3, 1).contiguous()) * (WIDTH // HEADS) ** -0.5
    sc = sc.masked_fill(torch.ones(S, S).triu(1).bool(), -math.inf)
    o = torch.matmul(sc.softmax(-1), v.transpose(1, 2).contiguous()).transpose(1, 2).reshape(B * S, -1)
    h = h + norm(o @ P["wp"], P["post2"])
    n = norm(h, P["n2"])
    h = 0.5 * h + (torch.nn.functional.silu(n @ P["g_in"]) * (n @ P["g_up"])) @ P["g_down"]
    return norm(h, P["n3"]) @ P["head"]


def test_block_gradients(eng):
    """All of them together in one residual stream, against float64 autograd: every
    gradient's error, 2-norm over 2-norm, is below 2^-24 times the root of the terms
    of the longest product (80) times 16 operations in a row, times 4."""
    B, S, classes = 2, 70, 11
    r = rng(60)
    P0 = block_params(r, classes)
    x, labels = r.standard_normal((B * S, WIDTH)).astype(np.float32), r.integers(0, classes, B * S)
    P = {n: dev(eng, a, True) for n, a in P0.items()}
    table = eng.rotary_table(S, WIDTH // HEADS)
    xt = dev(eng, x, True)
    loss = eng.softmax_ce(block(eng, P, xt, table, B, S), dev(eng, labels))
    loss.backward()
    R = {n: torch.tensor(a, dtype=torch.float64, requires_grad=True) for n, a in P0.items()}
    x64 = torch.tensor(x, dtype=torch.float64, requires_grad=True)
    ref = torch.nn.functional.cross_entropy(block64(R, x64, torch.tensor(np.asarray(table.sync(), np.float64)), B, S),
                                            torch.as_tensor(labels))
    ref.backward()
    tol = EPS * math.sqrt(80) * 16 * 4
    assert abs(float(loss.sync()[0]) - float(ref.detach())) <= tol * float(ref.detach())
    for n, t in (*P.items(), ("x", xt)):
        want = (R[n] if n != "x" else x64).grad.numpy()
        e = float(np.linalg.norm(t.grad.sync().astype(np.float64) - want) / np.linalg.norm(want))
        print(n, "%.2g of %.2g" % (e, tol), flush=True)
        assert e <= tol, n
    eng.end_batch()


def test_block_recorded(eng):
    """A recorded training step of it, replayed between other work of the same
    operators at larger sizes (which share the engine's workspace), trains as eager
    steps do, to the last bit."""
    B, S, classes = 2, 700, 11
    r = rng(61)
    P0 = block_params(r, classes)
    data = [(r.standard_normal((B * S, WIDTH)).astype(np.float32), r.integers(0, classes, B * S).astype(np.float32)) for _ in range(4)]
    table = eng.rotary_table(S, WIDTH // HEADS)

    def fresh():
        P = {n: dev(eng, a, True) for n, a in P0.items()}
        return P, eng.AdamW(list(P.values()), lr=0.01)
    P, opt = fresh()
    losses = []
    for x, y in data:
        opt.zero_grad()
        loss = eng.softmax_ce(block(eng, P, dev(eng, x), table, B, S), dev(eng, y))
        loss.backward()
        opt.step(clip=1.0)
        losses.append(float(loss.sync()[0]))
        eng.end_batch()
    want = {n: t.sync().copy() for n, t in P.items()}
    P, opt = fresh()
    graph = eng.ComputeGraph()
    graph.trace(lambda x: block(eng, P, x, table, B, S), opt, *data[0], list(P.values()), clip=1.0)
    for i, (x, y) in enumerate(data[1:]):
        graph.replay(x, y)
        n = 900 + 500 * i
        a = [dev(eng, r.standard_normal(s), True) for s in ((n, 512), (512, 640), (512, 640), (640, 512), (512,))]
        h, m = eng.residual_norm(a[0], eng.gated_mlp(*a[:4]), a[4], a[4], a[4])
        m.backward(a[0])
        big = dev(eng, r.standard_normal((1, 2 * n, 256)), True)
        eng.gated_scan(big, big).backward(big)
        assert graph.read_loss() == losses[i + 1], i
        eng.end_batch()
    for n, t in P.items():
        assert np.array_equal(t.sync(), want[n]), n
    graph.release()
    eng.end_batch()


def test_runs_are_alike(eng):
    """The same call twice gives the same bits."""
    r = rng(70)
    a = [r.standard_normal(s).astype(np.float32) for s in ((3, 901, 200), (200, 300), (200, 300), (300, 200), (200,))]

    def once():
        T = [dev(eng, v, True) for v in a]
        y = eng.gated_scan(T[0], T[0])
        h, n = eng.residual_norm(y, eng.gated_mlp(y, *T[1:4]), T[4], T[4], T[4])
        n.backward(dev(eng, a[0]))
        got = [n.sync().copy()] + [t.grad.sync().copy() for t in T]
        eng.end_batch()
        return got
    first = once()
    for _ in range(2):
        assert all(np.array_equal(p, q) for p, q in zip(first, once()))


def test_streaming_accesses_change_nothing(eng):
    """The kernels' nontemporal forms, taken above a size, at small sizes."""
    r = rng(71)
    a = [r.standard_normal(s).astype(np.float32) for s in ((2, 600, 203), (203, 2000), (203, 2000), (2000, 203), (203,))]

    def once():
        T = [dev(eng, v, True) for v in a]
        y = eng.gated_scan(T[0], T[0])
        h, n = eng.residual_norm(y, eng.gated_mlp(y, *T[1:4]), T[4], T[4], T[4])
        n.backward(dev(eng, a[0]))
        got = [n.sync().copy()] + [t.grad.sync().copy() for t in T]
        eng.end_batch()
        return got
    want = once()
    eng.lib.SetStreamingThreshold(0.0)
    try:
        got = once()
    finally:
        eng.lib.SetStreamingThreshold(-1.0)
    assert all(np.array_equal(p, q) for p, q in zip(got, want))


def test_layers(eng):
    """RMSNorm and GatedMLP as layers: a model lists their parameters, and trains them."""
    np.random.seed(3)

    class Net(eng.Model):
        def __init__(self):
            super().__init__()
            self.norm, self.mlp = eng.RMSNorm(24), eng.GatedMLP(24, 40, act="gelu")
            self.head = eng.Linear(24, 5)

        def forward(self, x):
            return self.head(eng.add(x, self.mlp(self.norm(x))))
    net = Net()
    params = net.parameters()
    assert [tuple(p.shape) for p in params] == [(24, 5), (5,), (24, 40), (24, 40), (40, 24), (24,)]
    loss = eng.softmax_ce(net(dev(eng, rng(1).standard_normal((6, 24)))), dev(eng, np.arange(6) % 5))
    loss.backward()
    before = [p.sync().copy() for p in params]
    eng.Muon(params, lr=0.01).step()
    assert all(p.grad is not None and not np.array_equal(p.sync(), b) for p, b in zip(params, before))
    eng.end_batch()


@pytest.mark.parametrize("rows", [1, 4, 7, 16])
@pytest.mark.parametrize("size", [(2053, 5000, 131), (131, 9000, 300), (4100, 300, 2100)], ids=lambda s: "x".join(map(str, s)))
def test_gated_mlp_of_few_tokens_and_many_weights(eng, size, rows):
    """Shares of the depth of one and of several steps, the last one not whole."""
    print("gated_mlp few", rows, size, flush=True)
    check_mlp(eng, rows, *size, "gelu", rng(rows + size[0]))


@pytest.mark.parametrize("rows", [1, 12, 40])
def test_gated_mlp_of_a_weight_that_is_infinite(eng, rows):
    """The last ones of their columns, where the depth ends inside a step: the
    results that it makes infinite are that, the other outputs as before."""
    r = rng(rows)
    x, wg, wu, wd = (r.standard_normal(s).astype(np.float32) for s in ((rows, 300), (300, 37), (300, 37), (37, 90)))
    t = [dev(eng, v) for v in (np.abs(x), np.abs(wg), np.abs(wu), wd)]
    want = eng.gated_mlp(*t).sync().copy()
    down = wd.copy()
    down[36, 5] = np.inf
    got = eng.gated_mlp(*t[:3], dev(eng, down)).sync()
    assert (got[:, 5] == np.inf).all()
    assert np.array_equal(np.delete(got, 5, 1), np.delete(want, 5, 1))
    up = np.abs(wu)
    up[299, 36] = np.inf
    got = eng.gated_mlp(*t[:2], dev(eng, up), t[3]).sync()
    assert (got == np.where(wd[36] < 0, -np.inf, np.inf)).all()
    eng.end_batch()


def test_gated_scan_refuses_what_no_launch_holds(eng):
    four = dev(eng, np.zeros(4))
    lib, b = eng.lib, four.gpu_buf
    for sizes in ((255, 1 << 24, 1), (1, 1 << 30, 3), (2, 1 << 29, 2)):
        assert not lib.GatedScanForward(b, b, None, None, *sizes, None) and "2^30" in eng.last_error(), sizes
        lib.ClearLastError()


@pytest.mark.parametrize("size", [(400, 512, 2048, 512), (33, 300, 4100, 70), (20, 2000, 37, 2000), (3000, 1, 1, 1), (5001, 3, 2, 5), (18, 1030, 515, 33),
                                  (70, 520, 1500, 519), (600, 40, 90, 1)], ids=lambda s: "x".join(map(str, s)))
def test_gated_mlp_of_shared_depths(eng, size):
    """Products whose depths waves and workgroups share in all numbers, and a call whose directions are worked out on different paths."""
    print("gated_mlp", size, flush=True)
    check_mlp(eng, *size, "silu", rng(sum(size)))


@pytest.mark.parametrize("size", [(20, 12, 16, 10), (150, 40, 70, 36), (700, 512, 1400, 512)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_gated_mlp_gradients_against_differences(eng, act, size):
    """Along a random direction of all operands, central differences in float64 of
    the formula: off by what the gradients may be off by, and by step^2 = 1e-8
    times third derivatives, which are sums of the slope's own terms: 1e-6 of those."""
    M, C, F, O = size
    r = rng(M)
    a = {"x": r.standard_normal((M, C)), "wg": r.standard_normal((C, F)) / math.sqrt(C), "wu": r.standard_normal((C, F)) / math.sqrt(C),
         "wd": r.standard_normal((F, O)) / math.sqrt(F)}
    a = {k: v.astype(np.float32) for k, v in a.items()}
    dy = r.standard_normal((M, O)).astype(np.float32)
    T = {k: dev(eng, v, True) for k, v in a.items()}
    eng.gated_mlp(*T.values(), act).backward(dev(eng, dy))
    way = {k: r.standard_normal(v.shape) / math.sqrt(v.size) for k, v in a.items()}

    def value(s):
        x, wg, wu, wd = (a[k].astype(np.float64) + s * way[k] for k in a)
        return (((act64(x @ wg, act)[0] * (x @ wu)) @ wd) * dy).sum()
    slope = (value(1e-4) - value(-1e-4)) / 2e-4
    ref = mlp64(*(v.astype(np.float64) for v in a.values()), act, dy.astype(np.float64))
    terms = {k: T[k].grad.sync().astype(np.float64) * way[k] for k in a}
    bound = sum((ref["d" + k][1] * np.abs(way[k])).sum() + 1e-6 * np.abs(terms[k]).sum() for k in a)
    assert abs(sum(t.sum() for t in terms.values()) - slope) <= bound
    eng.end_batch()


def test_the_same_operand_in_two_places(eng):
    """One matrix as gate and upward weights, one tensor as tokens and gates: the gradients of both places are added up."""
    r = rng(8)
    x, w, v, dy = (r.standard_normal(s).astype(np.float32) for s in ((40, 24), (24, 30), (30, 24), (40, 24)))
    t = [dev(eng, a, True) for a in (x, w, v)]
    eng.gated_mlp(t[0], t[1], t[1], t[2]).backward(dev(eng, dy))
    ref = mlp64(*(a.astype(np.float64) for a in (x, w, w, v)), "silu", dy.astype(np.float64))
    (g, eg), (u, eu) = ref["dwg"], ref["dwu"]
    within("dw", t[1].grad.sync(), g + u, eg + eu + EPS * np.abs(g + u))
    x, dy = r.standard_normal((2, 50, 30)).astype(np.float32), r.standard_normal((2, 50, 30)).astype(np.float32)
    t = dev(eng, x, True)
    eng.gated_scan(t, t).backward(dev(eng, dy))
    ref = scan64(x.astype(np.float64), x.astype(np.float64), None, np.full(2, 50), dy.astype(np.float64))
    (a, ea), (b, eb) = ref["dx"], ref["dz"]
    within("dx", t.grad.sync(), a + b, ea + eb + EPS * np.abs(a + b))
    eng.end_batch()


@pytest.mark.parametrize("width", [3, 64, 771, 2048, 9001])
def test_norms_keep_what_is_not_finite_in_its_row(eng, width):
    r = rng(width)
    x, b, dh, dn = (r.standard_normal((9, width)).astype(np.float32) for _ in range(4))
    gate, post, pre = (r.standard_normal(width).astype(np.float32) for _ in range(3))

    def run():
        T = [dev(eng, v, True) for v in (x, b)]
        h, n = eng.residual_norm(*T, *(dev(eng, v) for v in (gate, post, pre)))
        h.grad = dev(eng, dh)
        n.backward(dev(eng, dn))
        out = [t.sync().copy() for t in (h, n, T[0].grad, T[1].grad)]
        eng.end_batch()
        return out
    want = run()
    x[1, 0], b[4, width - 1], dn[7, 1] = np.nan, np.inf, np.nan
    got = run()
    keep = [0, 2, 3, 5, 6, 8]
    assert all(np.array_equal(g[keep], w[keep]) for g, w in zip(got, want))
    assert np.isnan(got[1][1]).all() and np.isnan(got[2][7]).all()


@pytest.mark.parametrize("rows", [6, 40, 600, 1400, 2300])
def test_gated_mlp_recorded(eng, rows):
    """A recorded step through each of the block's paths, replayed with a product of
    another size between the replays, trains as eager steps do, to the last bit."""
    C, F, classes = 512, 1024, 7
    r = rng(rows)
    P0 = {n: (r.standard_normal(s) / math.sqrt(s[0])).astype(np.float32)
          for n, s in (("wg", (C, F)), ("wu", (C, F)), ("wd", (F, C)), ("head", (C, classes)))}
    P0["gain"] = np.ones(C, np.float32)
    data = [(r.standard_normal((rows, C)).astype(np.float32), r.integers(0, classes, rows).astype(np.float32)) for _ in range(4)]

    def model(P, x):
        return eng.matmul(eng.residual_norm(x, eng.gated_mlp(x, P["wg"], P["wu"], P["wd"]), pre=P["gain"])[1], P["head"])

    def fresh():
        P = {n: dev(eng, a, True) for n, a in P0.items()}
        return P, eng.AdamW(list(P.values()), lr=0.01)
    P, opt = fresh()
    losses = []
    for x, y in data:
        opt.zero_grad()
        loss = eng.softmax_ce(model(P, dev(eng, x)), dev(eng, y))
        loss.backward()
        opt.step(clip=1.0)
        losses.append(float(loss.sync()[0]))
        eng.end_batch()
    want = {n: t.sync().copy() for n, t in P.items()}
    P, opt = fresh()
    graph = eng.ComputeGraph()
    graph.trace(lambda x: model(P, x), opt, *data[0], list(P.values()), clip=1.0)
    for i, (x, y) in enumerate(data[1:]):
        graph.replay(x, y)
        a = [dev(eng, r.standard_normal(s), True) for s in ((rows + 300, 400), (400, 500), (400, 500), (500, 400))]
        eng.gated_mlp(*a).backward(a[0])
        assert graph.read_loss() == losses[i + 1], i
        eng.end_batch()
    for n, t in P.items():
        assert np.array_equal(t.sync(), want[n]), n
    graph.release()
    eng.end_batch()


@pytest.mark.parametrize("size,need", [((60, 1501, 5003, 1499), ("x", "wg", "wu", "wd")), ((64, 300, 9000, 3800), ()), ((64, 40, 9000, 3801), ("x", "wd"))],
                         ids=lambda s: "x".join(map(str, s)))
def test_gated_mlp_of_some_tokens_and_many_weights(eng, size, need):
    """Tiles of 64 x 64, of one wave and of several."""
    print("gated_mlp some", size, flush=True)
    check_mlp(eng, *size, "silu", rng(size[0]), need=need)
