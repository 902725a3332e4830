"""Rotary positions, attention with its gradients, and the orthogonalised
update, against plain float64 implementations (torch on the CPU).

Tolerances (eps = 2^-24, fp32's half step; errors are max |difference| over
max |result|, unless a test says otherwise):
  rotary: two products and a sum, on a table rounded to fp32: 4 eps of the
    pair's length, which is at most sqrt(2) max |x|.
  attention: a score of up to s_max carries the roundings of a dot product of D
    terms, sqrt(D) eps s_max at the usual spread, and the exponential turns an
    absolute error of a score into a relative one of P; the sum over T keys
    adds sqrt(T) eps.  tol = 8 eps (sqrt(D) s_max + sqrt(T) + 4); the gradients
    go through P, dP and another product: 4 tol.
  orthogonalised update: each step rounds its products to 4 * 2^-23 of |X|, and
    the remaining steps grow a perturbation by 3.4445 each: at most 3.4445^5 = 485
    of |X_0| = 1 in all, against |X_5| >= 0.67 sqrt(rank) (the quintic's image
    of a singular value that has arrived): 485 * 4 * 2^-23 / (0.67 sqrt(rank)),
    2-norm over 2-norm.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from tests.helpers import rel2, rng

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


def rel_max(got, ref):
    top = np.abs(ref).max()
    return float(np.abs(np.asarray(got, np.float64) - ref).max() / (top if top else 1.0))


def dev(eng, a, grad=False):
    return eng.Tensor(np.array(a, np.float32), requires_grad=grad, track=False)


# ------------------------------------------------------------------- rotary
def turned(x, table, pos, interleaved, sign=1.0):
    """x (B, S, H, D) float64, table (P, pairs, 2), pos (B, S) ints, -1: a row of zeros."""
    pairs = table.shape[1]
    rows = np.concatenate([table, np.zeros_like(table[:1])])[pos][:, :, None]
    c, s = rows[..., 0], sign * rows[..., 1]
    y = x.copy()
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape,rot,scattered", [
    ((1, 1, 1, 2), 2, False), ((2, 1, 5, 64), 64, True), ((3, 17, 4, 64), 32, False), ((2, 9, 7, 80), 60, True),
    ((1, 33, 3, 50), 50, False), ((2, 5, 1, 7), 4, True), ((2, 300, 9, 128), 96, False), ((1, 70, 6, 20), 8, True)])
def test_rotary(eng, shape, rot, scattered, interleaved):
    print("rotary", shape, rot, scattered, interleaved, flush=True)
    r = rng(sum(shape) + rot)
    x, dy = (r.standard_normal(shape).astype(np.float32) for _ in range(2))
    rows = 500
    t = eng.rotary_table(rows, rot)
    pos = r.integers(0, rows, shape[:2]) if scattered else np.tile(np.arange(shape[1]), (shape[0], 1))
    p = dev(eng, pos) if scattered else None
    xt = dev(eng, x, True)
    y = eng.rotary(xt, t, p, interleaved)
    y.backward(dev(eng, dy))
    f = 10000.0 ** (-np.arange(0, rot, 2) / rot)
    ang = np.arange(rows)[:, None] * f
    table = np.stack([np.cos(ang), np.sin(ang)], -1)
    tol = 4 * EPS * math.sqrt(2)
    assert rel_max(y.sync(), turned(x.astype(np.float64), table, pos, interleaved)) <= tol
    assert rel_max(xt.grad.sync(), turned(dy.astype(np.float64), table, pos, interleaved, -1.0)) <= tol
    eng.end_batch()


@pytest.mark.parametrize("interleaved", [False, True])
def test_streaming_accesses_change_nothing(eng, interleaved):
    """The kernels' nontemporal forms, taken above a size, at small sizes."""
    r = rng(3)
    x = dev(eng, r.standard_normal((3, 40, 6, 96)))
    q, k, v = (dev(eng, r.standard_normal(s)) for s in ((2, 1, 4, 64), (2, 500, 2, 64), (2, 500, 2, 64)))
    t = eng.rotary_table(40, 72)

    def both():
        return eng.rotary(x, t, None, interleaved).sync().copy(), eng.attention(q, k, v).sync().copy()
    want = both()
    eng.lib.SetStreamingThreshold(0.0)
    try:
        got = both()
    finally:
        eng.lib.SetStreamingThreshold(-1.0)
    assert all(np.array_equal(a, b) for a, b in zip(got, want))
    eng.end_batch()


def test_rotary_outside_the_table_reads_zeros(eng):
    r = rng(1)
    x = r.standard_normal((1, 6, 2, 16)).astype(np.float32)
    t = eng.rotary_table(10, 8)
    y = eng.rotary(dev(eng, x), t, dev(eng, [[0, 10, -1, np.nan, 1e9, 9]])).sync()
    assert np.array_equal(y[0, 1:5, :, :8], np.zeros((4, 2, 8), np.float32))
    assert np.array_equal(y[..., 8:], x[..., 8:])
    assert np.array_equal(y[0, 0], x[0, 0])
    eng.end_batch()


def test_rotary_table_of_long_contexts(eng):
    """A stretched table: slow pairs at position * 1 / factor, fast ones as they were."""
    t = eng.rotary_table(20000, 64, factor=4.0, original=4096).sync()
    plain = eng.rotary_table(20000, 64).sync()
    f = 10000.0 ** (-np.arange(0, 64, 2) / 64)
    turns = 4096 * f / (2 * np.pi)
    keep = np.clip((turns - 1) / 31, 0, 1)
    ang = np.arange(20000)[:, None] * (keep * f + (1 - keep) * f / 4)
    assert np.abs(t[..., 0] - np.cos(ang)).max() <= 2 * EPS and np.abs(t[..., 1] - np.sin(ang)).max() <= 2 * EPS
    assert np.array_equal(t[:, turns > 32], plain[:, turns > 32])
    straight = eng.rotary_table(100, 8, factor=2.0).sync()
    assert np.array_equal(straight[::2], eng.rotary_table(50, 8).sync())


def test_rotary_refusals(eng):
    x, t = dev(eng, np.zeros((2, 4, 3, 8))), eng.rotary_table(4, 8)
    for bad in (lambda: eng.rotary(dev(eng, np.zeros((2, 4, 8))), t),
                lambda: eng.rotary(x, dev(eng, np.zeros((4, 8)))),
                lambda: eng.rotary(x, eng.rotary_table(3, 8)),
                lambda: eng.rotary(x, t, dev(eng, np.zeros((4, 2)))),
                lambda: eng.rotary_table(0, 8), lambda: eng.rotary_table(4, 7)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="even number"):
        eng.rotary(x, eng.rotary_table(4, 10))
    lib = eng.lib
    assert not lib.RotaryApply(x.gpu_buf, t.gpu_buf, None, 2, 4, 3, 9, 8, 0)
    assert not lib.RotaryApply(x.gpu_buf, t.gpu_buf, None, 2, 4, 3, 8, 7, 0)
    assert not lib.RotaryApply(x.gpu_buf, None, None, 2, 4, 3, 8, 8, 0)
    assert not lib.RotaryApply(x.gpu_buf, t.gpu_buf, t.gpu_buf, 50000, 50000, 3, 8, 8, 0)
    assert not lib.RotaryApply(x.gpu_buf, t.gpu_buf, None, 0, 4, 3, 8, 8, 0)
    lib.ClearLastError()


# ---------------------------------------------------------------- attention
def attend64(q, k, v, causal, scale, lengths):
    """Plain attention in float64 torch with autograd; empty rows are zeros."""
    B, S, H, D = q.shape
    T, G = k.shape[1], k.shape[2]
    kr, vr = k.repeat_interleave(H // G, 2), v.repeat_interleave(H // G, 2)
    s = torch.matmul(q.permute(0, 2, 1, 3), kr.permute(0, 2, 3, 1)) * scale
    j = torch.arange(T)
    ok = torch.ones(B, 1, S, T, dtype=torch.bool)
    if causal:
        ok = ok & (j <= torch.arange(S)[:, None] + T - S)
    if lengths is not None:
        ok = ok & (j < torch.as_tensor(lengths)[:, None, None, None])
    s = s.masked_fill(~ok, -math.inf)
    p = torch.softmax(s, -1)
    p = torch.where(ok.any(-1, keepdim=True), p, torch.zeros_like(p))
    return torch.matmul(p, vr.permute(0, 2, 1, 3)).permute(0, 2, 1, 3), float(s.detach()[ok.expand_as(s)].abs().max()) if ok.any() else 0.0


CASES = [  # B, S, T, H, G, D, causal, lengths
    (1, 1, 1, 1, 1, 1, False, None),
    (2, 1, 37, 4, 2, 64, False, [37, 5]),
    (1, 2, 3, 2, 1, 3, True, None),
    (2, 33, 33, 3, 3, 32, True, None),
    (2, 64, 64, 2, 2, 64, False, None),
    (1, 65, 65, 4, 1, 64, True, None),
    (3, 50, 129, 6, 2, 40, True, [129, 1, 0]),      # an empty sequence
    (2, 100, 31, 2, 2, 48, True, None),             # rows before the first key see none
    (1, 100, 260, 8, 2, 128, True, None),
    (2, 77, 200, 2, 1, 80, False, [200, 64]),
    (1, 130, 130, 2, 2, 50, True, None),            # dims that are no multiple of 4
    (1, 40, 96, 3, 1, 33, False, [95]),
    (1, 35, 70, 2, 1, 256, True, None),
    (1, 20, 90, 2, 2, 200, False, [33]),
    (1, 300, 300, 1, 1, 96, True, None),
    (5, 16, 16, 12, 4, 16, True, [16, 15, 1, 0, 7]),
    (1, 60, 700, 1, 1, 32, True, None),             # keys split over workgroups in dQ
    (2, 700, 60, 2, 1, 64, False, [60, 0]),         # rows split in dK, dV
]


def attention_inputs(case, seed):
    B, S, T, H, G, D, _, lengths = case
    r = rng(seed)
    q, dy = (r.standard_normal((B, S, H, D)).astype(np.float32) for _ in range(2))
    k, v = (r.standard_normal((B, T, G, D)).astype(np.float32) for _ in range(2))
    return q, k, v, dy


def attention_tol(case, s_max):
    return 8 * EPS * (math.sqrt(case[5]) * s_max + math.sqrt(case[2]) + 4)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:6])) + ("c" if c[6] else "") + ("l" if c[7] else ""))
def test_attention(eng, case):
    print("attention", case, flush=True)
    B, S, T, H, G, D, causal, lengths = case
    q, k, v, dy = attention_inputs(case, 100 + S + T + D)
    # memory past a sequence's length may hold anything
    kd, vd = k.copy(), v.copy()
    for b, n in enumerate(lengths or []):
        kd[b, n:], vd[b, n:] = np.nan, np.inf
    qt, kt, vt = dev(eng, q, True), dev(eng, kd, True), dev(eng, vd, True)
    lt = dev(eng, lengths) if lengths is not None else None
    out = eng.attention(qt, kt, vt, causal=causal, lengths=lt)
    out.backward(dev(eng, dy))
    ref = [torch.tensor(a, dtype=torch.float64, requires_grad=True) for a in (q, k, v)]
    o, s_max = attend64(*ref, causal, D ** -0.5, lengths)
    o.backward(torch.tensor(dy, dtype=torch.float64))
    tol = attention_tol(case, s_max)
    errs = [rel_max(out.sync(), o.detach().numpy())] + [rel_max(t.grad.sync(), r.grad.numpy())
                                                        for t, r in zip((qt, kt, vt), ref)]
    print(["%.2g" % e for e in errs], "tol %.2g" % tol, flush=True)
    assert errs[0] <= tol and max(errs[1:]) <= 4 * tol
    # without gradients: the same values from the evaluating call
    again = eng.attention(dev(eng, q), dev(eng, kd), dev(eng, vd), causal=causal, lengths=lt)
    assert np.array_equal(again.sync(), out.data)
    eng.end_batch()


@pytest.mark.parametrize("case", [(8, 1, 5000, 8, 2, 64, False, [5000, 4999, 1, 0, 31, 32, 33, 2500]),
                                  (1, 3, 2100, 4, 1, 128, True, None), (1, 200, 3000, 1, 1, 32, True, [2950])],
                         ids=["tokens", "chunk", "rows"])
def test_attention_few_rows_over_many_keys(eng, case):
    """Few rows: the keys are split over workgroups and joined."""
    print("attention split", case, flush=True)
    test_attention(eng, case)


def test_attention_scale_and_large_scores(eng):
    """Scores of hundreds: the maximum is taken off before the exponential;
    negative scales are scales too."""
    case = (1, 40, 70, 2, 1, 64, True, None)
    q, k, v, dy = attention_inputs(case, 5)
    for scale in (4.0, -0.5):
        qt, kt, vt = (dev(eng, a, True) for a in (q, k, v))
        out = eng.attention(qt, kt, vt, causal=True, scale=scale)
        out.backward(dev(eng, dy))
        ref = [torch.tensor(a, dtype=torch.float64, requires_grad=True) for a in (q, k, v)]
        o, s_max = attend64(*ref, True, scale, None)
        o.backward(torch.tensor(dy, dtype=torch.float64))
        tol = attention_tol(case, s_max)
        assert rel_max(out.sync(), o.detach().numpy()) <= tol
        for t, r in zip((qt, kt, vt), ref):
            assert rel_max(t.grad.sync(), r.grad.numpy()) <= 4 * tol
    eng.end_batch()


def test_attention_gradients_against_differences(eng):
    """d/dh of sum(out * dy) along random directions, by central differences of
    the kernel's own forward: a step of h = 2^-6 leaves h^2 / 6 of the third
    derivative (of the order of the sum's terms, for inputs of unit spread) and
    the forward's error over h."""
    case = (2, 21, 45, 4, 2, 24, True, [45, 30])
    q, k, v, dy = attention_inputs(case, 6)
    lt = dev(eng, case[7])
    ts = [dev(eng, a, True) for a in (q, k, v)]
    eng.attention(*ts, causal=True, lengths=lt).backward(dev(eng, dy))
    grads = [t.grad.sync().astype(np.float64) for t in ts]
    r, h = rng(7), 2.0 ** -6

    def value(parts):
        o = eng.attention(*[dev(eng, p) for p in parts], causal=True, lengths=lt).sync()
        return float((o.astype(np.float64) * dy).sum())
    for i in range(3):
        way = r.standard_normal(grads[i].shape)
        way /= np.abs(way).max()
        parts = [q, k, v]
        ends = []
        for s in (h, -h):
            p = list(parts)
            p[i] = (parts[i] + s * way).astype(np.float32)
            ends.append(value(p))
        slope = (ends[0] - ends[1]) / (2 * h)
        size = math.sqrt(float((grads[i] ** 2).sum()) * float((way ** 2).sum()))
        assert abs(slope - float((grads[i] * way).sum())) <= (h * h + 8 * EPS * 40 / h) * size
    eng.end_batch()


def test_attention_only_wanted_gradients(eng):
    case = (1, 20, 20, 2, 1, 32, True, None)
    q, k, v, dy = attention_inputs(case, 8)
    every = [dev(eng, a, True) for a in (q, k, v)]
    eng.attention(*every, causal=True).backward(dev(eng, dy))
    whole = [t.grad.sync().copy() for t in every]
    for i in range(3):
        ts = [dev(eng, a, j == i) for j, a in enumerate((q, k, v))]
        eng.attention(*ts, causal=True).backward(dev(eng, dy))
        for j, t in enumerate(ts):
            assert (t.grad is None) == (j != i)
        assert np.array_equal(ts[i].grad.sync(), whole[i])
    # one tensor as query, key and vector: its three gradients add up
    x = dev(eng, q[:, :, :1], True)
    eng.attention(x, x, x).backward(dev(eng, dy[:, :, :1]))
    r = torch.tensor(q[:, :, :1], dtype=torch.float64, requires_grad=True)
    o, s_max = attend64(r, r, r, False, 32 ** -0.5, None)
    o.backward(torch.tensor(dy[:, :, :1], dtype=torch.float64))
    assert rel_max(x.grad.sync(), r.grad.numpy()) <= 12 * attention_tol(case, s_max)
    eng.end_batch()


def test_attention_not_finite_inputs_stay_in_their_sequence(eng):
    case = (3, 40, 40, 2, 2, 32, True, None)
    q, k, v, _ = attention_inputs(case, 9)
    clean = eng.attention(dev(eng, q), dev(eng, k), dev(eng, v), causal=True).sync().copy()
    q[1, 7], k[1, 3], v[1, 2] = np.nan, np.inf, np.nan
    out = eng.attention(dev(eng, q), dev(eng, k), dev(eng, v), causal=True).sync()
    assert np.array_equal(out[[0, 2]], clean[[0, 2]]) and np.isnan(out[1, 7]).all()
    eng.end_batch()


def test_attention_refusals(eng):
    z = lambda *s: dev(eng, np.zeros(s))  # noqa: E731
    q, k = z(2, 3, 4, 8), z(2, 5, 2, 8)
    for bad in ((z(2, 3, 32), k, k), (q, z(1, 5, 2, 8), z(1, 5, 2, 8)), (q, z(2, 5, 3, 8), z(2, 5, 3, 8)),
                (q, z(2, 5, 2, 16), z(2, 5, 2, 16)), (q, k, z(2, 6, 2, 8))):
        with pytest.raises(ValueError):
            eng.attention(*bad)
    with pytest.raises(ValueError):
        eng.attention(q, k, k, lengths=z(3))
    with pytest.raises(RuntimeError, match="256"):
        eng.attention(z(1, 1, 1, 257), z(1, 1, 1, 257), z(1, 1, 1, 257))
    lib, st = eng.lib, ctypes.c_void_p()
    args = [q.gpu_buf, k.gpu_buf, k.gpu_buf, None]
    for dims in ((2, 3, 6, 4, 2, 8), (2, 4, 5, 4, 2, 8), (2, 3, 5, 4, 3, 8), (0, 3, 5, 4, 2, 8), (2, 3, 0, 4, 2, 8),
                 (65535, 65535, 65535, 4, 2, 8), (1 << 22, 1, 1, 1, 1, 1)):
        assert not lib.AttentionForward(*args, *dims, 0, 1.0, ctypes.byref(st)) and not st.value
        assert eng.last_error()
    assert not lib.AttentionForward(q.gpu_buf, None, k.gpu_buf, None, 2, 3, 5, 4, 2, 8, 0, 1.0, None)
    out = [ctypes.c_void_p() for _ in range(3)]
    lib.AttentionBackward(q.gpu_buf, q.gpu_buf, *args[:3], None, z(5).gpu_buf, 2, 3, 5, 4, 2, 8, 0, 1.0, 1, 1, 1,
                          *[ctypes.byref(p) for p in out])
    assert not any(p.value for p in out) and "stats" in eng.last_error()
    lib.ClearLastError()


# --------------------------------------------------------------------- Muon
def orthogonalised64(d, steps):
    x = d.T if d.shape[0] > d.shape[1] else d
    x = x / (np.linalg.norm(x) + 1e-7)
    for _ in range(steps):
        a = x @ x.T
        x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
    return x.T if d.shape[0] > d.shape[1] else x


def muon_tol(rank):
    return 485 * 4 * 2.0 ** -23 / (0.67 * math.sqrt(rank))


def test_muon_orthogonalises(eng):
    """Weights of zero, a step of one: w = -X, for matrices of every kind in one call."""
    r = rng(20)
    shapes = [(1, 1), (1, 300), (300, 1), (6, 25), (120, 84), (128, 128), (129, 127), (257, 400), (400, 130), (64, 2000),
              (2000, 96), (33, 2, 3, 3), (512, 512), (7, 1), (16, 1, 3, 3)]
    gs = [r.standard_normal(s).astype(np.float32) * 10.0 ** r.integers(-3, 2) for s in shapes]
    ranks = [min(s[0], int(np.prod(s[1:]))) for s in shapes]
    gs[8] = (r.standard_normal((400, 2)) @ r.standard_normal((2, 130))).astype(np.float32)     # rank 2
    ranks[8] = 2
    rows = np.logspace(0, -5, 257)[:, None]                                                   # rows of very different size
    gs[7] = (r.standard_normal((257, 400)) * rows).astype(np.float32)
    ranks[7] = 8
    ws = [dev(eng, np.zeros(s), True) for s in shapes]
    opt = eng.Muon(ws, lr=1.0, momentum=0.0, nesterov=False, rms=1.0)
    for w, g in zip(ws, gs):
        w.grad = dev(eng, g)
    opt.step(clip=1e30)
    for s, w, g, rank in zip(shapes, ws, gs, ranks):
        rw, cl = s[0], int(np.prod(s[1:]))
        want = -orthogonalised64(g.reshape(rw, cl).astype(np.float64), 5).reshape(s) * math.sqrt(max(rw, cl))
        e = rel2(w.sync(), want)
        print(s, "%.2g of %.2g" % (e, muon_tol(rank)), flush=True)
        assert np.isfinite(w.data).all() and e <= muon_tol(rank), s


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("steps", [1, 3, 5])
def test_muon_steps(eng, nesterov, steps):
    """Three updates with momentum, decay and clipping; vectors by AdamW."""
    r = rng(21)
    shapes = [(40, 70), (9, 4, 3, 3), (50,), (1,)]
    w0 = [r.standard_normal(s).astype(np.float32) for s in shapes]
    ws = [dev(eng, w, True) for w in w0]
    ref = [dev(eng, w, True) for w in w0[2:]]
    opt = eng.Muon(ws, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, steps=steps)
    adam = eng.AdamW(ref, lr=0.02, weight_decay=0.0)
    want, mom = [w.astype(np.float64) for w in w0[:2]], [np.zeros(s) for s in shapes[:2]]
    for _ in range(3):
        gs = [r.standard_normal(s).astype(np.float32) for s in shapes]
        for w, g in zip(ws, gs):
            w.grad = dev(eng, g)
        for w, g in zip(ref, gs[2:]):
            w.grad = dev(eng, g)
        opt.step(clip=0.8)
        adam.step(clip=0.8)
        for i in range(2):
            g = np.clip(gs[i].astype(np.float64), np.float32(-0.8), np.float32(0.8))
            mom[i] = 0.9 * mom[i] + g
            d = g + 0.9 * mom[i] if nesterov else mom[i]
            rw = shapes[i][0]
            x = orthogonalised64(d.reshape(rw, -1), steps).reshape(shapes[i])
            want[i] = want[i] * (1 - 0.02 * 0.1) - 0.02 * 0.2 * math.sqrt(max(rw, d.size // rw)) * x
    assert opt.t == 3
    for i in range(2):
        # three updates, each of 2-norm 0.004 sqrt(rows cols) or less, and six fp32 roundings of w
        tol = 3 * 0.0044 * muon_tol(9) * math.sqrt(want[i].size) / np.linalg.norm(want[i]) + 12 * EPS
        assert rel2(ws[i].sync(), want[i]) <= tol
        assert rel2(opt.m[i].sync(), mom[i]) <= 8 * EPS
    for w, a in zip(ws[2:], ref):
        assert np.array_equal(w.sync(), a.sync())


def test_muon_zero_and_absent_gradients(eng):
    r = rng(22)
    w0 = [r.standard_normal((20, 30)).astype(np.float32) for _ in range(3)]
    ws = [dev(eng, w, True) for w in w0]
    opt = eng.Muon(ws, lr=0.1)
    ws[0].grad = dev(eng, np.zeros((20, 30)))
    ws[2].grad = dev(eng, np.full((20, 30), np.nan))
    opt.step()
    assert np.array_equal(ws[0].sync(), w0[0]) and np.array_equal(ws[1].sync(), w0[1])
    assert np.isnan(ws[2].sync()).all()


def test_muon_more_matrices_than_a_launch_holds(eng):
    r = rng(23)
    ws = [dev(eng, np.zeros((5 + i % 7, 9)), True) for i in range(95)]
    gs = [r.standard_normal(w.shape).astype(np.float32) for w in ws]
    opt = eng.Muon(ws, lr=1.0, momentum=0.0, rms=1.0)
    for w, g in zip(ws, gs):
        w.grad = dev(eng, g)
    opt.step(clip=1e30)
    for w, g in zip(ws, gs):
        want = -orthogonalised64(g.astype(np.float64), 5) * math.sqrt(max(g.shape))
        assert rel2(w.sync(), want) <= muon_tol(5)


def test_muon_refusals(eng):
    with pytest.raises(ValueError):
        eng.Muon([], steps=0)
    with pytest.raises(ValueError):
        eng.Muon([], steps=21)
    w = dev(eng, np.zeros((4, 4)), True)
    lib = eng.lib
    one = lambda t, v: (t * 1)(v)  # noqa: E731
    h, u, f = ctypes.c_void_p, ctypes.c_uint, ctypes.c_float
    P = lambda: one(h, w.gpu_buf)  # noqa: E731
    assert not lib.MuonBatch(P(), P(), P(), one(u, 5), one(u, 4), one(f, 1.0), 1, 0.9, 1, 0.0, 1.0, 5)
    assert "does not fit" in eng.last_error()
    assert not lib.MuonBatch(P(), P(), P(), one(u, 0), one(u, 4), one(f, 1.0), 1, 0.9, 1, 0.0, 1.0, 5)
    assert not lib.MuonBatch(P(), P(), P(), one(u, 4), one(u, 4), one(f, 1.0), 1, 0.9, 1, 0.0, 1.0, 21)
    assert not lib.MuonBatch(P(), P(), one(h, None), one(u, 4), one(u, 4), one(f, 1.0), 1, 0.9, 1, 0.0, 1.0, 5)
    w.grad = dev(eng, np.ones((4, 4)))
    with pytest.raises(RuntimeError, match="another one"):
        eng.Muon([w, w]).step()
    wide = eng.Tensor.empty((1, 4200000), requires_grad=True, track=False)
    wide.grad = wide
    with pytest.raises(RuntimeError, match="4 million"):
        eng.Muon([wide]).step()
    w.grad = None
    lib.ClearLastError()
    eng.Muon([w]).step()        # no gradients: nothing to do
    assert np.array_equal(w.sync(), np.zeros((4, 4), np.float32))


# ----------------------------------------------------------- all of them together
def block_data(r, B, S, C, classes):
    shapes = {"wq": (C, C), "wk": (C, C // 2), "wv": (C, C // 2), "wo": (C, C), "head": (C, classes), "bias": (classes,)}
    P = {n: (r.standard_normal(s) / math.sqrt(s[0])).astype(np.float32) for n, s in shapes.items()}
    return P, r.standard_normal((B * S, C)).astype(np.float32), r.integers(0, classes, B * S)


def block_forward(eng, P, x, table, B, S, H, D):
    q = eng.rotary(eng.reshape(eng.matmul(x, P["wq"]), (B, S, H, D)), table)
    k = eng.rotary(eng.reshape(eng.matmul(x, P["wk"]), (B, S, H // 2, D)), table)
    v = eng.reshape(eng.matmul(x, P["wv"]), (B, S, H // 2, D))
    o = eng.reshape(eng.attention(q, k, v, causal=True), (B * S, H * D))
    return eng.add_bias(eng.matmul(eng.add(x, eng.matmul(o, P["wo"])), P["head"]), P["bias"])


def test_block_trains(eng):
    """Projections, rotary positions, causal attention over shared key heads,
    residual, loss, gradients and the update, against float64 autograd."""
    B, S, H, D, classes = 2, 45, 4, 16, 11
    r = rng(30)
    P0, x, y = block_data(r, B, S, H * D, classes)
    P = {n: dev(eng, a, True) for n, a in P0.items()}
    table = eng.rotary_table(S, D)
    loss = eng.softmax_ce(block_forward(eng, P, dev(eng, x), table, B, S, H, D), dev(eng, y))
    loss.backward()
    R = {n: torch.tensor(a, dtype=torch.float64, requires_grad=True) for n, a in P0.items()}
    xt = torch.tensor(x, dtype=torch.float64)
    tb = torch.tensor(np.asarray(table.sync(), np.float64))

    def spin(t):
        c, s = tb[:, None, :, 0], tb[:, None, :, 1]
        a, b = t[..., :D // 2], t[..., D // 2:]
        return torch.cat([a * c - b * s, a * s + b * c], -1)
    q, k = spin((xt @ R["wq"]).view(B, S, H, D)), spin((xt @ R["wk"]).view(B, S, H // 2, D))
    o, s_max = attend64(q, k, (xt @ R["wv"]).view(B, S, H // 2, D), True, D ** -0.5, None)
    z = (xt + o.reshape(B * S, H * D) @ R["wo"]) @ R["head"] + R["bias"]
    ref = torch.nn.functional.cross_entropy(z, torch.as_tensor(y))
    ref.backward()
    # the products around attention add sqrt(C) eps each
    tol = 4 * attention_tol((B, S, S, H, H // 2, D), s_max) + 16 * EPS * math.sqrt(H * D)
    assert abs(float(loss.sync()[0]) - float(ref.detach())) <= tol * float(ref.detach())
    for n in P:
        e = rel_max(P[n].grad.sync(), R[n].grad.numpy())
        print(n, "%.2g of %.2g" % (e, tol), flush=True)
        assert e <= tol, n
    opt = eng.Muon(list(P.values()), lr=0.01)
    opt.step()
    for n in ("wq", "wk", "head"):
        g = R[n].grad.numpy()
        want = P0[n] - 0.01 * 0.2 * math.sqrt(max(g.shape)) * orthogonalised64(g, 5)
        # a gradient off by tol of its largest value is off by that of |d| or
        # less, which the update grows by up to 485
        assert rel2(P[n].sync(), want) <= 0.002 * math.sqrt(max(g.shape)) * 485 * tol / np.linalg.norm(want) * math.sqrt(g.size)
    eng.end_batch()


def test_block_recorded(eng):
    """The same step recorded and replayed, with eager work between the
    replays, trains exactly as the eager steps do."""
    B, S, H, D, classes = 2, 40, 4, 16, 7
    r = rng(31)
    P0, _, _ = block_data(r, B, S, H * D, classes)
    data = [(r.standard_normal((B * S, H * D)).astype(np.float32), r.integers(0, classes, B * S).astype(np.float32))
            for _ in range(4)]
    table = eng.rotary_table(S, D)

    def fresh():
        P = {n: dev(eng, a, True) for n, a in P0.items()}
        return P, eng.Muon(list(P.values()), lr=0.01)
    P, opt = fresh()
    losses = []
    for x, y in data:
        opt.zero_grad()
        loss = eng.softmax_ce(block_forward(eng, P, dev(eng, x), table, B, S, H, D), dev(eng, y))
        loss.backward()
        opt.step(clip=1.0)
        losses.append(float(loss.sync()[0]))
        eng.end_batch()
    want = {n: t.sync().copy() for n, t in P.items()}
    P, opt = fresh()
    graph = eng.ComputeGraph()
    graph.trace(lambda x: block_forward(eng, P, x, table, B, S, H, D), opt, *data[0], list(P.values()), clip=1.0)
    other = eng.Muon([dev(eng, np.ones((300, 200)), True)], lr=0.1)
    for i, (x, y) in enumerate(data[1:]):
        graph.replay(x, y)
        # eager work over the same workspace between the replays
        other.params[0].grad = dev(eng, r.standard_normal((300, 200)))
        other.step()
        eng.attention(dev(eng, np.ones((1, 1, 2, 8))), dev(eng, np.ones((1, 900, 1, 8))), dev(eng, np.ones((1, 900, 1, 8)))).sync()
        assert graph.read_loss() == losses[i + 1]
    assert opt.t == len(data)
    for n, t in P.items():
        assert np.array_equal(t.sync(), want[n]), n
    graph.release()
    eng.end_batch()


def test_results_repeat_bit_for_bit(eng):
    case = (2, 150, 150, 6, 2, 64, True, [150, 90])
    q, k, v, dy = attention_inputs(case, 40)
    seen = []
    for _ in range(3):
        ts = [dev(eng, a, True) for a in (q, k, v)]
        out = eng.attention(*ts, causal=True, lengths=dev(eng, case[7]))
        out.backward(dev(eng, dy))
        w = dev(eng, np.zeros((200, 900)), True)
        w.grad = dev(eng, rng(41).standard_normal((200, 900)))
        eng.Muon([w]).step()
        seen.append([out.sync().copy(), w.sync().copy()] + [t.grad.sync().copy() for t in ts])
        eng.end_batch()
    for s in seen[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(s, seen[0]))


def test_reshape(eng):
    r = rng(50)
    x = r.standard_normal((6, 8)).astype(np.float32)
    t = dev(eng, x, True)
    y = eng.reshape(t, (2, 3, 8))
    eng.relu(y).backward(dev(eng, np.ones((2, 3, 8))))
    assert y.shape == (2, 3, 8) and np.array_equal(t.grad.sync(), (x > 0).astype(np.float32))
    for bad in ((6, 7), (0, 48), (-1, 8)):
        with pytest.raises(ValueError):
            eng.reshape(t, bad)
    eng.end_batch()


# ------------------------------------------------- large calls, on fp16 parts
LARGE = [  # operations times keys from 1e12 on (the last one's backward alone)
    (1, 1024, 1024, 8, 8, 64, True, None),
    (2, 700, 700, 12, 4, 40, False, [700, 333]),
    (1, 1100, 1300, 4, 2, 128, True, None),
    (3, 515, 777, 6, 3, 96, True, [777, 0, 261]),
    (1, 1500, 1500, 8, 1, 30, True, None),
    (1, 33, 9000, 8, 8, 128, True, [8999]),
    (2, 1300, 400, 8, 2, 100, False, None),
    (1, 2000, 1024, 4, 4, 80, True, None),          # 976 rows see nothing
    (1, 1200, 1200, 1, 1, 64, True, None),          # one head: both split
    (2, 400, 1500, 1, 1, 128, True, [1500, 700]),
]


@pytest.mark.parametrize("case", LARGE, ids=lambda c: "x".join(map(str, c[:6])) + ("c" if c[6] else "") + ("l" if c[7] else ""))
def test_attention_large(eng, case):
    test_attention(eng, case)


def test_attention_large_scores(eng):
    """Scores of hundreds on parts: the maximum moves by more than its slack."""
    case = (1, 1024, 1024, 8, 8, 64, True, None)
    q, k, v, dy = attention_inputs(case, 63)
    k *= np.linspace(0.2, 4, 1024, dtype=np.float32)[None, :, None, None]  # later keys score higher
    ts = [dev(eng, a, True) for a in (q, k, v)]
    out = eng.attention(*ts, causal=True, scale=1.0)
    out.backward(dev(eng, dy))
    ref = [torch.tensor(a, dtype=torch.float64, requires_grad=True) for a in (q, k, v)]
    o, s_max = attend64(*ref, True, 1.0, None)
    o.backward(torch.tensor(dy, dtype=torch.float64))
    tol = attention_tol(case, s_max)
    assert s_max > 100 and rel_max(out.sync(), o.detach().numpy()) <= tol
    for t, r in zip(ts, ref):
        assert rel_max(t.grad.sync(), r.grad.numpy()) <= 4 * tol
    eng.end_batch()


@pytest.mark.parametrize("change", ["rows", "tiles", "tiny", "huge", "grads"])
def test_attention_large_of_uneven_sizes(eng, change):
    """Vectors of very different sizes: between the tiles of a call (the parts
    of each tile have an exponent of their own) and within one (those problems
    run on fp32)."""
    case = (2, 1024, 1024, 4, 4, 64, True, None)
    q, k, v, dy = attention_inputs(case, 60)
    r = rng(61)
    if change == "tiles":            # values and gradients grow and shrink along the sequence
        v *= np.exp2(np.round(10 * np.sin(np.arange(1024) / 90)))[None, :, None, None].astype(np.float32)
        dy *= np.exp2(np.round(10 * np.cos(np.arange(1024) / 70)))[None, :, None, None].astype(np.float32)
    elif change == "rows":           # one head of a sequence has vectors 2^20 apart side by side
        v[1, :, 2] *= np.exp2(r.choice([-20, 0], 1024))[:, None].astype(np.float32)
    elif change == "tiny":
        v *= np.float32(2.0 ** -40)
    elif change == "huge":
        v *= np.float32(2.0 ** 40)
    else:                            # gradients as a mean over many tokens gives them, some of them zero
        dy *= np.float32(2.0 ** -45)
        dy[:, ::3] = 0
    ts = [dev(eng, a, True) for a in (q, k, v)]
    out = eng.attention(*ts, causal=True)
    out.backward(dev(eng, dy))
    ref = [torch.tensor(a, dtype=torch.float64, requires_grad=True) for a in (q, k, v)]
    o, s_max = attend64(*ref, True, 64 ** -0.5, None)
    o.backward(torch.tensor(dy, dtype=torch.float64))
    tol = attention_tol(case, s_max)
    # tol is relative to a result's largest value where all terms are of one
    # size; here each value gets the sum of its terms' sizes instead
    qa, ka, va, ya = (torch.tensor(a, dtype=torch.float64).permute(0, 2, 1, 3) for a in (q, k, v, dy))
    p = torch.softmax((qa @ ka.transpose(2, 3) / 8).masked_fill(~torch.ones(1024, 1024, dtype=torch.bool).tril(), -math.inf), -1)
    big = lambda t: t.abs().amax(-1, keepdim=True)  # noqa: E731
    dp = ya.abs() @ va.abs().transpose(2, 3)
    ds = p * (dp + (p * dp).sum(-1, keepdim=True)) / 8
    size = [p @ big(va), ds @ big(ka), ds.transpose(2, 3) @ big(qa), p.transpose(2, 3) @ big(ya)]
    for i, (got, want, z) in enumerate(zip([out.sync()] + [t.grad.sync() for t in ts],
                                           [o.detach()] + [t.grad for t in ref], size)):
        z = z.permute(0, 2, 1, 3).numpy()
        e = np.abs(got - want.numpy()).max(-1, keepdims=True)
        print(change, "%.2g of the terms' size, tol %.2g" % ((e[z > 0] / z[z > 0]).max(), (4 if i else 1) * tol), flush=True)
        assert (e <= (4 if i else 1) * tol * z).all()
    eng.end_batch()


def test_attention_large_not_finite(eng):
    case = (2, 1024, 1024, 4, 4, 64, True, None)
    q, k, v, _ = attention_inputs(case, 62)
    clean = eng.attention(dev(eng, q), dev(eng, k), dev(eng, v), causal=True).sync().copy()
    v[1, 500, 3] = np.inf
    q[0, 9, 1] = np.nan
    out = eng.attention(dev(eng, q), dev(eng, k), dev(eng, v), causal=True).sync()
    assert np.array_equal(out[0, :, [0, 2, 3]], clean[0, :, [0, 2, 3]]) and np.array_equal(out[1, :, :3], clean[1, :, :3])
    assert np.isnan(out[0, 9, 1]).all() and np.array_equal(np.isnan(out[0, :, 1]).any(-1).nonzero()[0], [9])
    # dim by dim: an infinite value is in every later sum
    assert not np.isfinite(out[1, 500:, 3]).any() and np.isfinite(out[1, :480, 3]).all()
    eng.end_batch()


@pytest.mark.parametrize("apart", [2.0 ** 6, 2.0 ** 24])
@pytest.mark.parametrize("change", ["values", "gradients"])
def test_attention_large_ignored_vectors(eng, change, apart):
    """Large values that no row gives any weight, and large gradients of rows
    that give a key none, cost the others nothing.  Each result is off by
    attention_tol of its own terms' sizes."""
    case = (1, 1024, 1024, 8, 8, 64, False, None)
    q, k, v, dy = attention_inputs(case, 64)
    first = np.arange(1024) < 512
    q[..., 0] = 8
    if change == "values":           # scores of -60 for the first half
        k[..., 0] = np.where(first, -60, 0)[None, :, None]
        v[:, first] *= np.float32(apart)
    else:                            # 40 for a row's own half, -40 for the other
        q[:, ~first, :, 0] = -8
        k[..., 0] = np.where(first, 40, -40)[None, :, None]
        dy[:, first] *= np.float32(apart)
    ts = [dev(eng, a, True) for a in (q, k, v)]
    out = eng.attention(*ts)
    out.backward(dev(eng, dy))
    ref = [torch.tensor(a, dtype=torch.float64, requires_grad=True) for a in (q, k, v)]
    o, s_max = attend64(*ref, False, 64 ** -0.5, None)
    o.backward(torch.tensor(dy, dtype=torch.float64))
    tol = attention_tol(case, s_max)
    qa, ka, va, ya = (torch.tensor(a, dtype=torch.float64).permute(0, 2, 1, 3) for a in (q, k, v, dy))
    p = torch.softmax(qa @ ka.transpose(2, 3) / 8, -1)
    big = lambda t: t.abs().amax(-1, keepdim=True)  # noqa: E731
    dp = ya.abs() @ va.abs().transpose(2, 3)
    ds = p * (dp + (p * dp).sum(-1, keepdim=True)) / 8
    size = [p @ big(va), ds @ big(ka), ds.transpose(2, 3) @ big(qa), p.transpose(2, 3) @ big(ya)]
    # keys to which no row gives 2^-60 of its weight have results of no size
    for i, (got, want, z) in enumerate(zip([out.sync()] + [t.grad.sync() for t in ts],
                                           [o.detach()] + [t.grad for t in ref], size)):
        z = z.permute(0, 2, 1, 3).numpy()
        z = np.maximum(z, z.max() * 2.0 ** -60)
        e = np.abs(got - want.numpy()).max(-1, keepdims=True)
        print(change, "%.2g of the terms' size, tol %.2g" % ((e / z).max(), (4 if i else 1) * tol), flush=True)
        assert (e <= (4 if i else 1) * tol * z).all()
    eng.end_batch()


def test_muon_gradient_that_is_written(eng):
    a, b = (dev(eng, np.ones((6, 5)), True) for _ in range(2))
    opt = eng.Muon([a, b])
    a.grad, b.grad = dev(eng, np.ones((6, 5))), opt.m[0]
    with pytest.raises(RuntimeError, match="gradient is a parameter or momentum"):
        opt.step()
    assert np.array_equal(a.sync(), np.ones((6, 5), np.float32))
    b.grad = a.grad                  # one gradient for two parameters is fine
    opt.step()
    assert np.array_equal(a.sync(), b.sync()) and np.isfinite(a.sync()).all()


def test_muon_takes_any_iterable(eng):
    w, bias = dev(eng, np.ones((4, 3)), True), dev(eng, np.ones(3), True)
    opt = eng.Muon(p for p in (w, bias))
    w.grad, bias.grad = dev(eng, np.ones((4, 3))), dev(eng, np.ones(3))
    opt.step()
    assert opt.params == [w, bias] and (w.sync() != 1).all() and (bias.sync() != 1).all()


SPLIT = [  # splits joined and summed: by 4 values and by one, few rows and many
    (1, 61, 701, 1, 1, 33, False, None),
    (1, 701, 61, 1, 1, 33, True, None),
    (1, 1100, 300, 1, 1, 33, False, [299]),
    (1, 1100, 300, 1, 1, 40, True, None),
    (1, 3, 2100, 4, 2, 7, True, None),
    # and where the blocks alone would fill the chip
    (1, 2048, 2048, 16, 4, 128, True, None),
    (1, 1100, 1100, 32, 32, 128, False, [1077]),
]


@pytest.mark.parametrize("case", SPLIT, ids=lambda c: "x".join(map(str, c[:6])) + ("c" if c[6] else "") + ("l" if c[7] else ""))
def test_attention_split(eng, case):
    test_attention(eng, case)


@pytest.mark.parametrize("shape", [(2050, 2050), (3000, 5000), (4097, 1), (1, 4095)])
def test_muon_of_many_values(eng, shape):
    """Sums of the norm over more than 4096 values each, and ragged ends: one step
    of zero weights.  Its products are off by 4 * 2^-23 of |X_0| = 1, grown by
    3.4445 at most, and the update is rounded."""
    g = rng(70).standard_normal(shape).astype(np.float32)
    w = dev(eng, np.zeros(shape), True)
    w.grad = dev(eng, g)
    eng.Muon([w], lr=1.0, momentum=0.0, nesterov=False, steps=1, rms=1.0).step(clip=1e30)
    x = orthogonalised64(g.astype(np.float64), 1)
    assert rel2(w.sync(), -x * math.sqrt(max(shape))) <= 3.4445 * 4 * 2.0 ** -23 / np.linalg.norm(x) + 4 * EPS
