"""Calls of the block's operators that their documentation allows or refuses."""
import numpy as np
import pytest

from tests.helpers import rng
from tests.test_gpu_block import EPS, dev, norm64, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,gate,spread", [
    ((3, 5, 8), (8,), (1, 1, 8)), ((3, 5, 8), (1, 8), (1, 1, 8)), ((3, 5, 8), (1, 1, 8), (1, 1, 8)), ((3, 5, 8), (3, 8), (3, 1, 8)),
    ((3, 5, 8), (3, 1, 8), (3, 1, 8)), ((3, 5, 8), (3, 5, 8), (3, 5, 8)), ((3, 5, 8), (15, 8), (3, 5, 8)), ((1, 5, 8), (5, 8), (1, 5, 8)),
    ((2, 3, 4, 8), (2, 8), (2, 1, 1, 8)), ((2, 3, 4, 8), (2, 3, 8), (2, 3, 1, 8)), ((2, 3, 4, 8), (2, 3, 1, 8), (2, 3, 1, 8)),
    ((4, 8), (4, 8), (4, 8)), ((3, 1, 8), (3, 8), (3, 1, 8)), ((8,), (8,), (8,))], ids=str)
def test_residual_gates(eng, shape, gate, spread):
    r = rng(len(shape))
    x, b, g = (r.standard_normal(s).astype(np.float32) for s in (shape, shape, gate))
    T = [dev(eng, v, True) for v in (x, b, g)]
    h = eng.residual_norm(*T)
    h.backward(dev(eng, np.ones(shape)))
    assert np.allclose(h.sync(), x + g.reshape(spread) * b, rtol=0, atol=2 ** -20)
    axes = tuple(i for i, n in enumerate(spread) if n == 1)
    assert np.allclose(T[2].grad.sync().reshape(spread), b.sum(axes, keepdims=True), rtol=0, atol=b.size * 2 ** -22)
    eng.end_batch()


def test_residual_gate_of_tokens_side_by_side(eng):
    r = rng(4)
    x, b, g = (r.standard_normal(s).astype(np.float32) for s in ((12, 8), (12, 8), (3, 8)))
    h = eng.residual_norm(*(dev(eng, v) for v in (x, b, g)))
    assert np.allclose(h.sync(), x + np.repeat(g, 4, 0) * b, rtol=0, atol=2 ** -20)
    eng.end_batch()


@pytest.mark.parametrize("shape,gate", [((3, 5, 8), (5, 8)), ((3, 5, 8), (1, 5, 8)), ((4, 2, 8), (2, 8)), ((2, 4, 8), (4, 8)), ((3, 5, 8), (3, 5)),
                                        ((3, 5, 8), (5, 3, 8)), ((3, 5, 8), (3, 5, 1, 8)), ((2, 3, 4, 8), (6, 8)), ((12, 8), (5, 8)),
                                        ((3, 5, 8), (0, 8)), ((12, 8), (0, 8)), ((12, 8), (2, 2, 8))], ids=str)
def test_residual_gates_refused(eng, shape, gate):
    """A gate for each position, among others, does not say which rows are its."""
    class Shaped:   # no buffer of no values can be made
        gpu_buf, size, requires_grad = None, int(np.prod(gate)), False
    Shaped.shape = gate
    x = dev(eng, np.zeros(shape))
    with pytest.raises(ValueError, match="gate"):
        eng.residual_norm(x, x, gate=Shaped())


def test_scan_lengths_beyond_2_24(eng):
    """A length that is a float of its own, next to a sequence's length that is none."""
    S = 2 ** 24 + 1
    print("gated_scan of", S, "tokens", flush=True)
    x = np.zeros((1, S, 1), np.float32)
    x[0, -3:, 0] = 1, 2, 4
    z = dev(eng, np.zeros((1, S, 1)))
    for n, want in ((2 ** 24 - 1, [0.5, 0, 0]), (2 ** 24, [0.5, 1.25, 0]), (2 ** 24 + 2, [0.5, 1.25, 2.625]), (2.0 ** 40, [0.5, 1.25, 2.625])):
        T = dev(eng, x, True)
        y, last = eng.gated_scan(T, z, lengths=dev(eng, [n]), return_state=True)
        y.backward(dev(eng, np.ones((1, S, 1))))
        live = np.count_nonzero(want)
        assert y.sync()[0, -3:, 0].tolist() == want and last.sync()[0, 0] == want[live - 1], n
        assert (T.grad.sync()[0, -3:, 0] > 0).tolist() == [i < live for i in range(3)], n
        eng.end_batch()


@pytest.mark.parametrize("queries", [1, 40])
def test_attention_lengths_beyond_2_24(eng, queries):
    """The last key would take all weight, if it counted."""
    T, D = 2 ** 24 + 1, 4
    print("attention to", T, "keys", flush=True)
    k, v = np.zeros((1, T, 1, D), np.float32), np.zeros((1, T, 1, D), np.float32)
    k[0, -1], v[0, -1] = 100, 1
    q, k, v = dev(eng, np.ones((1, queries, 1, D))), dev(eng, k), dev(eng, v, True)
    for n, want in ((2 ** 24 - 1, 0), (2 ** 24, 0), (2 ** 24 + 2, 1)):
        v.grad = None
        o = eng.attention(q, k, v, lengths=dev(eng, [n]))
        o.backward(dev(eng, np.ones((1, queries, 1, D))))
        assert np.allclose(o.sync(), want, atol=1e-6), n
        assert np.allclose(v.grad.sync()[0, -1], queries * want, atol=1e-3), n
        eng.end_batch()


def test_gates_below_the_normal_numbers(eng):
    """Gates of e^-87 to e^-104 times values of 2^126: off by 8 roundings of the result and by what the
    gate's own rounding, half of 2^-149, makes of it."""
    z = np.linspace(-104, -86, 400).astype(np.float32)
    big = np.float32(2.0 ** 126)
    want = np.exp(z.astype(np.float64)) * float(big)
    tol = 8 * 2.0 ** -24 * want + 2.0 ** -150 * float(big)

    def vec(v):
        return dev(eng, np.broadcast_to(np.float32(v), (1, 1, 400)), True)
    none, state = vec(0), dev(eng, np.full((1, 400), big), True)
    gate = dev(eng, z.reshape(1, 1, 400), True)
    y = eng.gated_scan(none, gate, state)
    assert (np.abs(y.sync()[0, 0] - want) <= tol).all()
    y.backward(vec(big))
    assert (np.abs(state.grad.sync()[0] - want) <= tol).all()
    x = vec(big)
    y = eng.gated_scan(x, dev(eng, -z.reshape(1, 1, 400)))
    assert (np.abs(y.sync()[0, 0] - want) <= tol).all()
    y.backward(vec(big))
    assert (np.abs(x.grad.sync()[0, 0] - want) <= tol).all()
    for rows in (1, 40):   # each hidden unit its own output
        y = eng.gated_mlp(dev(eng, np.ones((rows, 1))), dev(eng, z[None]), dev(eng, np.full((1, 400), big)), dev(eng, np.eye(400)), "sigmoid")
        assert (np.abs(y.sync() - want) <= tol).all()
    eng.end_batch()


def test_waits_that_end_are_reported(eng):
    """With no looks beyond the first: a run of tokens that does not find the ones before it leaves NaN,
    and the next blocking call an error; runs that do find them are right.  With the usual limit all are."""
    r = rng(9)
    x, z = (dev(eng, r.standard_normal((1, 200_000, 64))) for _ in range(2))
    want = eng.gated_scan(x, z).sync().copy()
    eng.lib.ClearLastError()
    before = eng.lib.SetWaitLimit(0)
    try:
        for _ in range(3):
            got = eng.gated_scan(x, z).sync()
            bad = np.isnan(got)
            assert bad.any() == ("wait" in eng.last_error())
            assert np.array_equal(got[~bad], want[~bad])
            eng.lib.ClearLastError()
    finally:
        assert eng.lib.SetWaitLimit(before) == 0
    assert np.array_equal(eng.gated_scan(x, z).sync(), want) and not eng.last_error()
    eng.end_batch()


def test_scan_of_four_channels_that_no_launch_holds(eng):
    """2^32 threads, where one channel less was refused already."""
    four = dev(eng, np.zeros(4))
    b = four.gpu_buf
    for sizes in ((1, (1 << 30) - 1, 4), (1, (1 << 30) - (1 << 22) + 1, 4), (63, 17_043_520, 4)):
        assert not eng.lib.GatedScanForward(b, b, None, None, *sizes, None) and "2^30" in eng.last_error(), sizes
        eng.lib.ClearLastError()
    assert not eng.lib.GatedScanForward(b, b, None, None, 1, (1 << 30) - (1 << 22), 4, None) and "holds" in eng.last_error()
    eng.lib.ClearLastError()


@pytest.mark.parametrize("width", [3, 30, 100, 300, 771, 1500, 3000, 9001])
def test_norms_of_rows_of_all_sizes(eng, width):
    """Rows of 2^-100 to 2^110 whose squares fp32 does not hold, each beside ordinary ones."""
    r = rng(width)
    sizes = np.exp2(np.array([0, 70, 110, 0, -100, -70, 60, -60, 0, 30, -30, 100]))[:, None]
    M = len(sizes)
    a = {"x": r.standard_normal((M, width)) * sizes, "block": r.standard_normal((M, width)) * sizes[::-1], "post": r.standard_normal(width),
         "pre": r.standard_normal(width), "dh": np.zeros((M, width)), "dn": r.standard_normal((M, width))}
    a = {k: v.astype(np.float32) for k, v in a.items()}
    ref = {k: v.astype(np.float64) for k, v in a.items()}
    T = {k: dev(eng, v, k not in ("dh", "dn")) for k, v in a.items()}
    y = eng.rms_norm(T["block"], T["post"], 0.0)
    want = norm64(ref["block"], np.zeros((M, width)), None, None, ref["post"], 1.0, 0.0, ref["dh"], ref["dn"])
    within("rms_norm", y.sync(), want["n"][0], 24 * EPS * want["n"][1])
    y.backward(T["dn"])
    within("dx", T["block"].grad.sync(), want["dx"][0], 64 * EPS * want["dx"][1])
    eng.end_batch()
    for eps in (0.0, 1e-6):
        T = {k: dev(eng, v, k not in ("dh", "dn")) for k, v in a.items()}
        h, n = eng.residual_norm(T["x"], T["block"], post=T["post"], pre=T["pre"], eps=eps)
        want = norm64(ref["x"], ref["block"], None, ref["post"], ref["pre"], 1.0, eps, ref["dh"], ref["dn"])
        within("h", h.sync(), want["h"][0], 24 * EPS * want["h"][1])
        within("n", n.sync(), want["n"][0], 24 * EPS * want["n"][1])
        n.backward(T["dn"])
        for k in ("x", "block", "post", "pre"):
            within("d" + k, T[k].grad.sync(), want["d" + k][0], 64 * EPS * want["d" + k][1])
        eng.end_batch()
