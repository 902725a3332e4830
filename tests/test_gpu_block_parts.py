"""The gated feed-forward block's large calls, whose products are worked out on
fp16 parts, against float64.  Every test here asks which path its calls took.

Bounds are those of tests/test_gpu_block.py, element by element: sqrt(K) + 8
roundings (2^-24) of the sum of a product's K terms' absolute values.  On parts a
value is off by 2^-23 of itself at most, and of a product of two the smaller
parts' is dropped, 2^-22: 8 roundings of the term in the worst case, of either
sign; a common exponent may add 4, or sqrt(K) / 4, before a result is worked out
on fp32 instead; and sums are rounded once for every 16 terms, twice: sqrt(K) / 2
at most.  From K = 64 on that is within sqrt(K) + 8.
"""
import contextlib
import ctypes
import math

import numpy as np
import pytest

from tests.helpers import rng
from tests.test_gpu_block import act64, check_mlp, dev, mlp64, within

pytestmark = pytest.mark.gpu

BELOW, ABOVE = (1400, 512, 1024, 512), (2300, 512, 1024, 512)   # weights split in one pass, or in two
ODD = (1301, 515, 1001, 533)


def calls(eng, family):
    n = ctypes.c_uint64()
    return n.value if eng.lib.GetProfile(family, ctypes.byref(n), None, None, None) else 0


@contextlib.contextmanager
def on_parts(eng, directions=2):
    """The calls inside, `directions` of them, run on parts, and no other."""
    eng.lib.SetProfiling(1)
    eng.lib.ResetProfile()
    try:
        yield
        assert (calls(eng, b"mlp_parts"), calls(eng, b"mlp")) == (directions, 0)
    finally:
        eng.lib.SetProfiling(0)
        eng.lib.ResetProfile()


def check(eng, size, act, seed, change=None, need=("x", "wg", "wu", "wd")):
    print("gated_mlp on parts", size, act, seed, flush=True)
    with on_parts(eng, 2 if need else 1):
        check_mlp(eng, *size, act, rng(seed), change=change, need=need)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("size", [BELOW, ABOVE, ODD], ids=lambda s: "x".join(map(str, s)))
def test_sizes_and_activations(eng, size, act):
    check(eng, size, act, sum(size))


@pytest.mark.parametrize("need", [("x",), ("wg",), ("wu",), ("wd",), ("wg", "wd"), ()])
def test_gradients_asked_for(eng, need):
    check(eng, ODD, "gelu", 3, need=need)


@pytest.mark.parametrize("size", [(150, 2100, 12001, 2047), (40000, 128, 260, 130), (700, 129, 8200, 130)], ids=lambda s: "x".join(map(str, s)))
def test_shapes(eng, size):
    """Few rows over large weights, many rows over small ones, a depth in many splits."""
    check(eng, size, "silu", size[0])


@pytest.mark.parametrize("size", [BELOW, ABOVE], ids=lambda s: "x".join(map(str, s)))
def test_rows_and_columns_of_all_sizes(eng, size):
    r = rng(7)

    def change(a):
        a["x"] *= 2.0 ** r.integers(-15, 3, (size[0], 1))
        a["dy"] *= 2.0 ** r.integers(-20, 20, (size[0], 1))
        a["wu"] *= 2.0 ** r.integers(-15, 15, (1, size[2]))
        a["wd"] *= 2.0 ** r.integers(-15, 15, (1, size[3]))
    check(eng, size, "silu", 8, change)


@pytest.mark.parametrize("size", [BELOW, ABOVE], ids=lambda s: "x".join(map(str, s)))
def test_zeros(eng, size):
    def change(a):
        a["x"][::2] = 0
        a["wg"][:, 3:9] = 0
        a["wd"][:, ::5] = 0
        a["dy"][1:4] = 0
        a["wu"][:, 256:512] = 0
        a["x"][:, 128:384] = 0
    check(eng, size, "gelu", 9, change)

    def half(a):
        a["dy"][:size[0] // 2] = 0
        a["wd"][:300] = 0
    check(eng, size, "relu", 10, half)

    def none(a):
        a["wu"][:] = 0
    check(eng, size, "gelu", 11, none)


@pytest.mark.parametrize("k", [18, 24, 30, 40, 50])
@pytest.mark.parametrize("size", [BELOW, ABOVE], ids=lambda s: "x".join(map(str, s)))
def test_large_tokens_without_gradients(eng, size, k):
    """Tokens of any size that the loss passes over (padded ones, say) have no part in the weights'
    gradients."""
    for tokens in ([7], [5, 700, 701, 1200], range(300, 900)):
        def change(a):
            a["x"][list(tokens)] *= 2.0 ** k
            a["dy"][list(tokens)] = 0
        check(eng, size, "silu", k, change)


@pytest.mark.parametrize("k", [20, 40])
def test_large_tokens_with_small_gradients(eng, k):
    def change(a):
        a["x"][3::50] *= 2.0 ** k
        a["dy"][3::50] *= 2.0 ** (-3 * k)
        a["x"][4::50] *= 2.0 ** -k
        a["dy"][4::50] *= 2.0 ** k
    check(eng, BELOW, "silu", k, change)


@pytest.mark.parametrize("k", [8, 12, 15, 30, 50])
def test_scales_along_the_hidden_axis(eng, k):
    """Upward weights' columns and downward weights' rows whose scales cancel."""
    r = rng(k)
    s = 2.0 ** r.integers(-k, k + 1, BELOW[2])

    def change(a):
        a["wu"] *= s
        a["wd"] /= s[:, None]
    check(eng, BELOW, "silu", k, change)


@pytest.mark.parametrize("k", [12, 20, 40])
@pytest.mark.parametrize("size", [BELOW, ABOVE, ODD], ids=lambda s: "x".join(map(str, s)))
def test_scales_along_the_width(eng, size, k):
    """Features and weights whose scales cancel, and likewise dy's and the downward weights' columns."""
    r = rng(k)
    s, t = (2.0 ** r.integers(-k, k + 1, n) for n in (size[1], size[3]))

    def change(a):
        a["x"] *= s
        a["wg"] /= s[:, None]
        a["wu"] /= s[:, None]
        a["wd"] *= t
        a["dy"] /= t
    check(eng, size, "gelu", k, change)


def beside_zeros(r, size, k, tokens):
    """Inputs of which each of `tokens` has one feature 2^k times the others, an even one, that odd hidden
    units do not see; the first half of the outputs sees none but those."""
    M, C, F, O = size
    x, dy = r.standard_normal((M, C)), r.standard_normal((M, O))
    wg, wu, wd = r.standard_normal((C, F)) / 16, r.standard_normal((C, F)) / 16, r.standard_normal((F, O)) / 16
    for t in tokens:
        x[t, 2 * (t % (C // 2))] *= 2.0 ** k
    wg[::2, 1::2] = wu[::2, 1::2] = 0
    wd[::2, :O // 2] = 0
    dy[:, O // 2:] = 0
    return [v.astype(np.float32) for v in (x, wg, wu, wd, dy)]


@pytest.mark.parametrize("k", [16, 22, 28, 34, 50])
@pytest.mark.parametrize("size", [BELOW, ABOVE], ids=lambda s: "x".join(map(str, s)))
def test_large_features_that_meet_zeros(eng, size, k):
    a = beside_zeros(rng(k), size, k, range(size[0]))
    with on_parts(eng):
        T = [dev(eng, v, True) for v in a[:4]]
        y = eng.gated_mlp(*T)
        y.backward(dev(eng, a[4]))
        ref = mlp64(*(v.astype(np.float64) for v in a[:4]), "silu", a[4].astype(np.float64))
        within("y", y.sync(), *ref["y"])
        for n, t in zip(("dx", "dwg", "dwu", "dwd"), T):
            within(n, t.grad.sync(), *ref[n])
    eng.end_batch()


@pytest.mark.parametrize("act", ["silu", "relu"])
@pytest.mark.parametrize("k,keep", [(4, 1.0), (12, 1.0), (0, 0.02), (8, 0.3), (12, 0.05)])
@pytest.mark.parametrize("size", [BELOW, ABOVE, ODD], ids=lambda s: "x".join(map(str, s)))
def test_values_of_all_sizes_and_zeros(eng, size, k, keep, act):
    """Every value of every operand 2^-k to 2^k times itself, or zero."""
    r = rng(size[0] + k)

    def change(a):
        for v in a.values():
            v *= np.exp2(r.integers(-k, k + 1, v.shape)) * (r.random(v.shape) < keep)
    check(eng, size, act, k, change)


@pytest.mark.parametrize("k", [0, 30])
def test_blocks_of_zeros(eng, k):
    """Weights, tokens and gradients that are zeros in whole blocks, beside blocks 2^k times the others."""
    def change(a):
        a["wd"][:512, :128] = 0
        a["wd"][512:, 128:256] *= 2.0 ** k
        a["wg"][:256, 640:] = 0
        a["x"][100:700, :256] *= 2.0 ** -k
        a["dy"][600:, :300] = 0
        a["dy"][::2, 300:] = 0
        a["wu"][:, 700:] *= 2.0 ** -k
    check(eng, BELOW, "silu", k, change)
    check(eng, ABOVE, "gelu", k, change)


def test_rows_that_need_fp32_leave_the_others_alone(eng):
    """A forward's other rows keep their bits, kept and returned, beside rows that parts do not hold."""
    size = BELOW
    plain = beside_zeros(rng(1), size, 0, ())
    mixed = beside_zeros(rng(1), size, 45, (0, 130, 131, 1399))
    got = []
    for a in (plain, mixed):
        with on_parts(eng, 1):
            T = [dev(eng, v, True) for v in a[:4]]
            y = eng.gated_mlp(*T)
            kept = np.empty(2 * size[0] * size[2], np.float32)
            eng.lib.ReadBuffer(y._ctx.kept, kept.ctypes.data_as(ctypes.POINTER(ctypes.c_float)))
            got.append((y.sync().copy(), kept.reshape(2, size[0], size[2])))
    keep = np.setdiff1d(np.arange(size[0]), (0, 130, 131, 1399))
    assert np.array_equal(got[0][0][keep], got[1][0][keep]) and np.array_equal(got[0][1][:, keep], got[1][1][:, keep])
    ref = mlp64(*(v.astype(np.float64) for v in mixed[:4]), "silu", mixed[4].astype(np.float64))["y"]
    within("y", got[1][0], *ref)
    eng.end_batch()


@pytest.mark.parametrize("size", [BELOW, ABOVE], ids=lambda s: "x".join(map(str, s)))
def test_what_is_not_finite_stays_in_its_row(eng, size):
    """A token that holds a NaN, an infinity or one value of 1e15: other tokens' results stay as they are."""
    r = rng(5)
    M, C, F, O = size
    w = [dev(eng, r.standard_normal(s) / 16) for s in ((C, F), (C, F), (F, O))]
    x = r.standard_normal((M, C)).astype(np.float32)
    with on_parts(eng):
        want = eng.gated_mlp(dev(eng, x), *w).sync().copy()
        x[1, 7], x[2, 9], x[3, 11] = np.nan, np.inf, 1e15
        got = eng.gated_mlp(dev(eng, x), *w).sync()
    assert not np.isfinite(got[1:3]).any() and np.array_equal(got[0], want[0]) and np.array_equal(got[4:], want[4:])
    ref = mlp64(x[3:4].astype(np.float64), *(t.sync().astype(np.float64) for t in w), "silu", np.zeros((1, O)))["y"]
    within("y", got[3:4], *ref)
    eng.end_batch()


def train(eng, a, act="silu"):
    T = [dev(eng, v, True) for v in a[:4]]
    y = eng.gated_mlp(*T, act)
    y.backward(dev(eng, a[4]))
    got = [y.sync().copy()] + [t.grad.sync().copy() for t in T]
    eng.end_batch()
    return got


@pytest.mark.parametrize("k", [0, 45])
@pytest.mark.parametrize("size", [BELOW, ABOVE, ODD], ids=lambda s: "x".join(map(str, s)))
def test_runs_are_alike(eng, size, k):
    a = beside_zeros(rng(k), size, k, range(0, size[0], 9))
    with on_parts(eng):
        first = train(eng, a)
    for _ in range(3):
        assert all(np.array_equal(p, q) for p, q in zip(first, train(eng, a)))


@pytest.mark.parametrize("size", [BELOW, ABOVE, ODD], ids=lambda s: "x".join(map(str, s)))
def test_streaming_accesses_change_nothing(eng, size):
    a = beside_zeros(rng(2), size, 0, ())
    with on_parts(eng):
        want = train(eng, a)
    eng.lib.SetStreamingThreshold(0.0)
    try:
        got = train(eng, a)
    finally:
        eng.lib.SetStreamingThreshold(-1.0)
    assert all(np.array_equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_gradients_against_differences(eng, act):
    """Along a random direction of all operands: see the test of the same name in tests/test_gpu_block.py."""
    M, C, F, O = BELOW
    r = rng(12)
    a = {"x": r.standard_normal((M, C)), "wg": r.standard_normal((C, F)) / math.sqrt(C), "wu": r.standard_normal((C, F)) / math.sqrt(C),
         "wd": r.standard_normal((F, O)) / math.sqrt(F)}
    a = {k: v.astype(np.float32) for k, v in a.items()}
    dy = r.standard_normal((M, O)).astype(np.float32)
    with on_parts(eng):
        got = dict(zip(("y", *a), train(eng, [*a.values(), dy], act)))
    way = {k: r.standard_normal(v.shape) / math.sqrt(v.size) for k, v in a.items()}

    def value(s):
        x, wg, wu, wd = (a[k].astype(np.float64) + s * way[k] for k in a)
        return (((act64(x @ wg, act)[0] * (x @ wu)) @ wd) * dy).sum()
    slope = (value(1e-4) - value(-1e-4)) / 2e-4
    ref = mlp64(*(v.astype(np.float64) for v in a.values()), act, dy.astype(np.float64))
    terms = {k: got[k].astype(np.float64) * way[k] for k in a}
    bound = sum((ref["d" + k][1] * np.abs(way[k])).sum() + 1e-6 * np.abs(terms[k]).sum() for k in a)
    assert abs(sum(t.sum() for t in terms.values()) - slope) <= bound


def test_recorded_steps_that_need_fp32(eng):
    """Steps recorded over weights whose scales along the hidden axis cancel, and whose batches hold tokens that
    parts do not suit, replayed with a product of another size in between, train as eager steps do, to the last bit."""
    rows, C, F, classes = 1400, 512, 1024, 7
    r = rng(60)
    s = 2.0 ** r.integers(-40, 41, F)
    P0 = {n: (r.standard_normal(z) / math.sqrt(z[0])).astype(np.float32) for n, z in (("wg", (C, F)), ("wu", (C, F)), ("wd", (F, C)), ("head", (C, classes)))}
    P0["wu"] = (P0["wu"] * s).astype(np.float32)
    P0["wd"] = (P0["wd"] / s[:, None]).astype(np.float32)
    data = []
    for i in range(4):
        x = r.standard_normal((rows, C)).astype(np.float32)
        if i % 2:
            x[i::9, 4] *= 2.0 ** 30
        data.append((x, r.integers(0, classes, rows).astype(np.float32)))

    def model(P, x):
        return eng.matmul(eng.gated_mlp(x, P["wg"], P["wu"], P["wd"]), P["head"])

    def fresh():
        P = {n: dev(eng, a, True) for n, a in P0.items()}
        return P, eng.SGD(list(P.values()), lr=1e-6)
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
        a = [dev(eng, r.standard_normal(z), True) for z in ((rows + 300, 400), (400, 500), (400, 500), (500, 400))]
        eng.gated_mlp(*a).backward(a[0])
        assert graph.read_loss() == losses[i + 1], i
        eng.end_batch()
    for n, t in P.items():
        assert np.array_equal(t.sync(), want[n]), n
    graph.release()
    eng.end_batch()
