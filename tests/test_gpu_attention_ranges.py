"""Attention of large calls (fp16 parts) on vectors of very different sizes,
against float64: every result vector is compared with its own length, so that
large vectors elsewhere in the call hide nothing.

Tolerance: P's relative error is the absolute one of its score (nats): two
operands of 22 bits or more, 2 * 2^-23 s_max, and roundings of 2^-24 s_max.  The
four other operands of a gradient (dO / l, V, P or dS, Q or K) round to 2^-23
each, delta and the sums to as much again: (s_max + 4) 2^-22.  The largest error
of thousands of vectors, whose terms cancel to about the root of their number as
their errors do, is taken as four times that: 2^-20 (s_max + 4).
"""
import math

import numpy as np
import pytest
import torch

from tests.helpers import rng

pytestmark = pytest.mark.gpu

N, D, H = 1024, 64, 4   # one sequence: 10^12 operations times keys, on parts both ways
FIRST = np.arange(N) < N // 2


def inputs(seed):
    r = rng(seed)
    return [r.standard_normal((1, N, H, D)).astype(np.float32) for _ in range(4)]


def attend(q, k, v, dy, causal):
    """Float64 results, and the sums of their terms' sizes."""
    ts = [torch.tensor(a, dtype=torch.float64).permute(0, 2, 1, 3).contiguous().requires_grad_(True) for a in (q, k, v)]
    y = torch.tensor(dy, dtype=torch.float64).permute(0, 2, 1, 3).contiguous()
    s = ts[0] @ ts[1].transpose(2, 3) / math.sqrt(D)
    if causal:
        s = s.masked_fill(~torch.ones(N, N, dtype=torch.bool).tril(), -math.inf)
    p = torch.softmax(s, -1)
    o = p @ ts[2]
    o.backward(y)
    with torch.no_grad():
        long = lambda t: t.norm(dim=-1, keepdim=True)  # noqa: E731
        dp = long(y) @ long(ts[2]).transpose(2, 3)
        ds = p * (dp + (p * dp).sum(-1, keepdim=True)) / math.sqrt(D)
        size = [p @ long(ts[2]), ds @ long(ts[1]), ds.transpose(2, 3) @ long(ts[0]), p.transpose(2, 3) @ long(y)]
    back = lambda t: t.detach().permute(0, 2, 1, 3).numpy()  # noqa: E731
    s_max = float(s.detach()[p.detach() > 0].abs().max())
    return [back(o)] + [back(t.grad) for t in ts], [back(t)[..., 0] for t in size], s_max


def check(eng, q, k, v, dy, what, causal=False, by_terms=False, only=range(4)):
    dev = lambda a, g=False: eng.Tensor(np.array(a, np.float32), requires_grad=g, track=False)  # noqa: E731
    ts = [dev(a, True) for a in (q, k, v)]
    out = eng.attention(*ts, causal=causal)
    out.backward(dev(dy))
    ref, size, s_max = attend(q, k, v, dy, causal)
    tol = 2.0 ** -20 * (s_max + 4)
    worst = []
    for got, want, z in zip([out.sync()] + [t.grad.sync() for t in ts], ref, size):
        z = z if by_terms else np.linalg.norm(want, axis=-1)
        z = np.maximum(z, z.max() * 2.0 ** -80)
        worst.append(float((np.linalg.norm(got - want, axis=-1) / z).max()))
    print(what, "o dq dk dv", ["%.2g" % w for w in worst], "tol %.2g" % tol, flush=True)
    assert all(worst[i] <= tol for i in only)
    eng.end_batch()


@pytest.mark.parametrize("apart", [10, 14, 18, 40])
def test_gradients_of_different_sizes(eng, apart):
    """Rows look at their own half of the keys (e^-24 of the weight goes to the
    other); one half's gradients are 2^apart larger."""
    q, k, v, dy = inputs(200)
    q[..., 0] = np.where(FIRST, 8, -8)[None, :, None]
    k[..., 0] = np.where(FIRST, 12, -12)[None, :, None]
    dy[:, FIRST] *= np.float32(2.0 ** apart)
    check(eng, q, k, v, dy, f"gradients 2^{apart} apart")


@pytest.mark.parametrize("apart", [6, 11, 20])
def test_gradients_with_ignored_values_of_different_sizes(eng, apart):
    """Keys of e^-24 of the weight have vectors 2^apart larger."""
    q, k, v, dy = inputs(201)
    q[..., 0] = 8
    k[..., 0] = np.where(FIRST, -24, 0)[None, :, None]
    v[:, FIRST] *= np.float32(2.0 ** apart)
    check(eng, q, k, v, dy, f"values 2^{apart} apart", only=(1, 2, 3))


def test_gradients_with_large_keys_and_queries(eng):
    """Half of the keys are 2^11 larger in dims where the queries that see them
    are zero, and the queries likewise."""
    q, k, v, dy = inputs(202)
    q[:, :, :, 32:] = 0
    q[..., 0] = np.where(FIRST, 8, -8)[None, :, None]
    k[..., 0] = np.where(FIRST, 12, -12)[None, :, None]
    k[:, FIRST, :, 48:] *= np.float32(2.0 ** 11)
    k[:, :, :, 32:48] = 0
    q[:, FIRST, :, 32:48] = rng(203).standard_normal((1, N // 2, H, 16)).astype(np.float32) * np.float32(2.0 ** 11)
    check(eng, q, k, v, dy, "large keys and queries", by_terms=True)


@pytest.mark.parametrize("apart", [11.5, 13])
def test_gradients_of_neighbours_of_different_sizes(eng, apart):
    """Rows side by side whose gradients are 2^apart apart: within what one
    exponent serves, and past it."""
    q, k, v, dy = inputs(204)
    dy *= np.exp2(-apart * rng(205).integers(0, 2, N))[None, :, None, None].astype(np.float32)
    check(eng, q, k, v, dy, f"neighbours 2^{apart} apart", causal=True, by_terms=True)


@pytest.mark.parametrize("swing", [3, 7, 12])
def test_gradients_that_grow_and_shrink(eng, swing):
    """Values and gradients that grow and shrink by up to 2^(2 swing) along the
    sequence: the sums are scaled again and again."""
    q, k, v, dy = inputs(206)
    at = np.arange(N)
    v *= np.exp2(np.round(swing * np.sin(at / 90)))[None, :, None, None].astype(np.float32)
    dy *= np.exp2(np.round(swing * np.cos(at / 70)))[None, :, None, None].astype(np.float32)
    for causal in (False, True):
        check(eng, q, k, v, dy, f"swing {swing} causal {causal}", causal=causal, by_terms=True)


def test_keys_of_almost_no_weight(eng):
    """Keys to which every row gives about 2^-50 of its weight have gradients of
    their own size."""
    q, k, v, dy = inputs(207)
    q[..., 0] = 8
    k[..., 0] = np.where(np.arange(N) % 32 < 16, -35, 0)[None, :, None]
    check(eng, q, k, v, dy, "keys of almost no weight")


@pytest.mark.parametrize("apart", [0, 6, 20])
def test_output_beside_a_key_that_takes_the_weight(eng, apart):
    """One key takes most of every row's weight and has a small vector; keys of
    e^-20 of the weight have vectors 2^apart larger than the others, which make
    the output."""
    q, k, v, dy = inputs(208)
    ignored = np.arange(N) // 32 % 2 == 0    # every other tile, in whatever way the keys are split
    q[..., 0] = 8
    k[..., 0] = np.where(ignored, -20, 0)[None, :, None]
    k[:, 630, :, 0] = 9
    v[:, ignored] *= np.float32(2.0 ** apart)
    v[:, 630] *= np.float32(2.0 ** -9)
    check(eng, q, k, v, dy, f"a key that takes the weight, values 2^{apart} apart")


@pytest.mark.parametrize("keys", [8, N])
@pytest.mark.parametrize("power", [7, 10, 14])
def test_scores_far_from_zero(eng, power, keys):
    """Every row's last key leads by 2^power or more, of scores a thousand times
    as large, whose own rounding is a part of one or more: P is 1 there all the
    same.  The output is that key's vector and its gradient the sum of the
    rows', each off by fp32's roundings of a sum of N terms at most.  The other
    dims add scores of spread sqrt(63) = 8, differences of less than 64 among
    these few million: the other keys have e^-(2^7 - 64) of the weight or less."""
    q, k, v, dy = (a[:, :keys] for a in inputs(209))
    g = np.float32(2.0 ** (power / 2))
    q[..., 0] = g
    k[..., 0] = g * np.arange(1000, 1000 + keys, dtype=np.float32)[None, :, None]
    dev = lambda a: eng.Tensor(np.array(a, np.float32), requires_grad=True, track=False)  # noqa: E731
    ts = [dev(a) for a in (q, k, v)]
    out = eng.attention(*ts, scale=1.0)
    out.backward(eng.Tensor(dy, track=False))
    tol = keys * 2.0 ** -24
    want = dy.astype(np.float64).sum(1)
    e = [np.abs(out.sync() - v[:, -1:]).max() / np.abs(v).max(),
         (np.abs(ts[2].grad.sync()[:, -1] - want).max() / np.abs(dy).sum(1).max())]
    print("scores far from zero", power, keys, ["%.2g" % x for x in e], "tol %.2g" % tol, flush=True)
    assert max(e) <= max(tol, 2.0 ** -22)
    assert np.abs(ts[2].grad.data[:, :-1]).max() <= math.exp(-64) * np.abs(dy).sum(1).max()
    # dS = P (dP - delta): what is left of two sums of D terms that are equal
    left = 4 * D * 2.0 ** -24 * np.abs(dy).max() * np.abs(v).max() * keys
    assert np.abs(ts[0].grad.sync()).max() <= left * np.abs(k).max() and np.abs(ts[1].grad.sync()).max() <= left * np.abs(q).max()
    eng.end_batch()


@pytest.mark.parametrize("rows", [33, 129, 1001])
def test_keys_of_almost_no_weight_under_ragged_rows(eng, rows):
    """As above, where the last tile of rows is not full: what stands in for the
    missing rows takes no bits from the rows beside it."""
    q, k, v, dy = inputs(210)
    q, dy = q[:, :rows], dy[:, :rows]
    q[..., 0] = 8
    k[..., 0] = np.where(np.arange(N) % 32 < 16, -35, 0)[None, :, None]
    check(eng, q, k, v, dy, f"keys of almost no weight, {rows} rows")
