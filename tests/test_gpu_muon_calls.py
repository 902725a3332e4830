"""Calls of the orthogonalised update that are refused or large: what they leave
as it was, and what they take."""
import math

import numpy as np
import pytest

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
    import torch
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
