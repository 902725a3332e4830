"""Gradients of graphs whose nodes hand the gradient they get on to several
inputs (add, flatten, reshape, add_bias): one input's later sums must not reach
another's, nor the tensor that the caller gave."""
import math

import numpy as np
import pytest
import torch

from tests.helpers import rng

pytestmark = pytest.mark.gpu


def dev(eng, a, grad=False):
    return eng.Tensor(np.array(a, np.float32), requires_grad=grad, track=False)


@pytest.mark.parametrize("order", ["attention first", "products first"])
def test_parallel_attention_and_products(eng, order):
    """y = x + attention(x) + relu(x U) W, both branches from the same x.  All
    products are of 32 terms or fewer, scores within 30: each gradient is a sum of
    products of at most six factors of 2^-22 (s_max + 4) each, 2^-19 (s_max + 4)
    of its largest value with the cancelling of their signs."""
    B, S, H, D = 2, 19, 2, 16
    C, r = H * D, rng(400)
    x0 = r.standard_normal((B * S, C)).astype(np.float32)
    W0 = {n: (r.standard_normal((C, C)) / math.sqrt(C)).astype(np.float32) for n in ("q", "k", "v", "u", "w")}
    dy0 = r.standard_normal((B * S, C)).astype(np.float32)
    x, W, dy = dev(eng, x0, True), {n: dev(eng, a, True) for n, a in W0.items()}, dev(eng, dy0)
    heads = lambda t: eng.reshape(t, (B, S, H, D))  # noqa: E731
    a = eng.reshape(eng.attention(*(heads(eng.matmul(x, W[n])) for n in "qkv"), causal=True), (B * S, C))
    m = eng.matmul(eng.relu(eng.matmul(x, W["u"])), W["w"])
    y = eng.add(eng.add(x, a), m) if order == "attention first" else eng.add(eng.add(x, m), a)
    y.backward(dy)

    X, R = torch.tensor(x0, dtype=torch.float64, requires_grad=True), {n: torch.tensor(t, dtype=torch.float64, requires_grad=True)
                                                                      for n, t in W0.items()}
    q, k, v = ((X @ R[n]).view(B, S, H, D).permute(0, 2, 1, 3) for n in "qkv")
    s = q @ k.transpose(2, 3) / math.sqrt(D)
    p = torch.softmax(s.masked_fill(~torch.ones(S, S, dtype=torch.bool).tril(), -math.inf), -1)
    z = X + (p @ v).permute(0, 2, 1, 3).reshape(B * S, C) + torch.relu(X @ R["u"]) @ R["w"]
    z.backward(torch.tensor(dy0, dtype=torch.float64))
    tol = 2.0 ** -19 * (float(s.detach().abs().max()) + 4)
    for n, t, want in [("x", x, X)] + [(n, W[n], R[n]) for n in W]:
        e = np.abs(t.grad.sync() - want.grad.numpy()).max() / np.abs(want.grad.numpy()).max()
        print(order, n, "%.2g of %.2g" % (e, tol), flush=True)
        assert e <= tol, n
    assert np.array_equal(dy.sync(), dy0)
    eng.end_batch()


def test_the_callers_gradient_is_left_alone(eng):
    r = rng(401)
    x0, b0, dy0 = (r.standard_normal(s).astype(np.float32) for s in ((6, 8), (8,), (6, 8)))
    for f in (lambda x, b: eng.add(x, eng.relu(x)), lambda x, b: eng.add(x, x), lambda x, b: eng.add_bias(eng.add(x, eng.relu(x)), b),
              lambda x, b: eng.reshape(eng.add(eng.reshape(x, (48, 1)), eng.relu(eng.reshape(x, (48, 1)))), (6, 8))):
        x, b, dy = dev(eng, x0, True), dev(eng, b0, True), dev(eng, dy0)
        y = f(x, b)
        y.backward(dy)
        assert np.array_equal(dy.sync(), dy0)
        once = x.grad.sync().copy()
        for t in (x, b):
            t.grad = None
        f(x, b).backward(dy)
        assert np.array_equal(x.grad.sync(), once)
        eng.end_batch()


def test_gradients_add_up_over_two_passes(eng):
    r = rng(402)
    x0, dy0 = (r.standard_normal((5, 7)).astype(np.float32) for _ in range(2))
    x, dy = dev(eng, x0, True), dev(eng, dy0)
    for _ in range(2):
        eng.add(eng.reshape(x, (5, 7)), eng.relu(x)).backward(dy)
    # sums of up to 4 dy, each rounded to 2^-24 of its size
    assert (np.abs(x.grad.sync() - 2 * (dy0 + dy0 * (x0 > 0))) <= 2.0 ** -21 * np.abs(dy0)).all()
    assert np.array_equal(dy.sync(), dy0)
    eng.end_batch()
