"""Calls of the orthogonalised update that are refused or large: what they leave
as it was, and what they take."""
import math

import numpy as np
import pytest
import torch   # ahead of the engine, which then shares its HIP runtime

from tests.helpers import rel2, rng

pytestmark = pytest.mark.gpu


def dev(eng, a, grad=False):
    return eng.Tensor(np.array(a, np.float32), requires_grad=grad, track=False)


def test_a_refused_step_updates_nothing(eng):
    w, bias = dev(eng, np.ones((4, 3)), True), dev(eng, np.ones(3), True)
    w.grad, bias.grad = dev(eng, np.ones((4, 3))), dev(eng, np.ones(3))
    opt = eng.Muon([bias, w, w])
    with pytest.raises(RuntimeError, match="another one"):
        opt.step()
    assert opt.t == 0
    for t in (w, bias):
        assert np.array_equal(t.sync(), np.ones(t.shape, np.float32))
    assert not opt.m[0].sync().any() and not opt.vectors.m[0].sync().any()
    eng.lib.ClearLastError()


def test_thin_matrices_share_a_bounded_workspace(eng):
    """Sixteen rows of a million values in one call, each 64 times its size where
    it is padded to whole tiles (1 GB with its parts), take turns.  A row's X is
    d / |d| times what the quintic makes of 1 in five steps."""
    n = 1 << 20
    r = rng(2)
    gs = [r.standard_normal(n).astype(np.float32) for _ in range(2)]
    ws = [eng.Tensor(np.zeros((1, n), np.float32), requires_grad=True, track=False) for _ in range(16)]
    for i, w in enumerate(ws):
        w.grad = dev(eng, gs[i % 2].reshape(1, n))
    opt = eng.Muon(ws, lr=1.0, momentum=0.0, rms=1.0)
    eng.lib.FlushGPU()
    free = torch.cuda.mem_get_info()[0]
    opt.step(clip=1e30)
    eng.lib.FlushGPU()
    taken = free - torch.cuda.mem_get_info()[0]
    print("taken: %.2f GB" % (taken / 1e9), flush=True)
    assert taken < 4e9
    s = 1.0
    for _ in range(5):
        s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
    for i, w in enumerate(ws):
        want = -gs[i % 2].astype(np.float64) / np.linalg.norm(gs[i % 2].astype(np.float64)) * s * math.sqrt(n)
        # each step is off by 4 * 2^-23 of X, which the others grow by 3.4445 at most
        assert rel2(w.sync()[0], want) <= 485 * 4 * 2.0 ** -23 / abs(s)


@pytest.mark.parametrize("steps", [2, 5])
def test_large_and_small_matrices_in_one_call(eng, steps):
    """128 x 128 tiles over several steps: a tall and a wide ragged matrix whose
    Gram products are split, beside small ones whose are not.  A step rounds its
    products to 4 * 2^-23 of |X|, and the steps grow |X_0| = 1 by 3.4445 each at
    most: steps * 4 * 2^-23 * 3.4445^steps over the result's length; and the update
    is rounded."""
    r = rng(3)
    shapes = [(4100, 2050), (33, 70), (700, 2300), (5, 5), (130, 3, 3, 3)]
    ws = [dev(eng, np.zeros(s), True) for s in shapes]
    gs = [r.standard_normal(s).astype(np.float32) for s in shapes]
    for w, g in zip(ws, gs):
        w.grad = dev(eng, g)
    eng.Muon(ws, lr=1.0, momentum=0.0, nesterov=False, steps=steps, rms=1.0).step(clip=1e30)
    for w, g in zip(ws, gs):
        x = g.astype(np.float64).reshape(g.shape[0], -1)
        tall = x.shape[0] > x.shape[1]
        x = (x.T if tall else x) / np.linalg.norm(x)
        for _ in range(steps):
            a = x @ x.T
            x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
        want = -(x.T if tall else x).reshape(g.shape) * math.sqrt(max(x.shape))
        e, tol = rel2(w.sync(), want), steps * 4 * 2.0 ** -23 * 3.4445 ** steps / np.linalg.norm(x) + 4 * 2.0 ** -24
        print(g.shape, steps, "%.2g of %.2g" % (e, tol), flush=True)
        assert e <= tol, g.shape
