"""Calls of the orthogonalised update that are refused or large: what they leave
as it was, and what they take."""
import numpy as np
import pytest

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
