"""The attention kernels' builds for a few rows, and the fp32 code inside the ones
on fp16 parts, at the head dims, shared heads, lengths and splits of each, against
float64.  Every result vector is compared with the sum of its terms' sizes.

Tolerance: P's relative error is the absolute one of its score, whose terms and
sum of D roundings come to 2^-22 s_max; the gradient's other four factors and its
sums to 2^-22 each at the most; the largest of thousands four times that:
2^-20 (s_max + 4).
"""
import math

import numpy as np
import pytest
import torch

from tests.helpers import rng

pytestmark = pytest.mark.gpu


def attend(q, k, v, dy, causal, lengths):
    B, S, H, D = q.shape
    T, G = k.shape[1], k.shape[2]
    t64 = lambda a: torch.tensor(a, dtype=torch.float64).permute(0, 2, 1, 3).contiguous()  # noqa: E731
    share = lambda t: t.repeat_interleave(H // G, 1)  # noqa: E731
    ts = [t64(a).requires_grad_(True) for a in (q, k, v)]
    kk, vv, y = share(ts[1]), share(ts[2]), t64(dy)
    j = torch.arange(T)
    ok = torch.ones(B, 1, S, T, dtype=torch.bool)
    if causal:
        ok = ok & (j <= torch.arange(S)[:, None] + T - S)
    if lengths is not None:
        ok = ok & (j < torch.as_tensor(lengths)[:, None, None, None])
    s = torch.matmul(ts[0], kk.transpose(2, 3).contiguous()) / math.sqrt(D)
    s_max = float(s.detach()[ok.expand_as(s)].abs().max())
    p = torch.softmax(s.masked_fill(~ok, -math.inf), -1)
    p = torch.where(ok.any(-1, keepdim=True), p, torch.zeros_like(p))
    o = torch.matmul(p, vv)
    o.backward(y)
    with torch.no_grad():
        long = lambda t: t.norm(dim=-1, keepdim=True)  # noqa: E731
        own = lambda t: t.reshape(B, G, H // G, T, 1).sum(2)  # noqa: E731
        dp = long(y) * long(vv).transpose(2, 3)
        ds = p * (dp + (p * dp).sum(-1, keepdim=True)) / math.sqrt(D)
        size = [p @ long(vv), ds @ long(kk), own(ds.transpose(2, 3) @ long(ts[0])), own(p.transpose(2, 3) @ long(y))]
    back = lambda t: t.detach().permute(0, 2, 1, 3).numpy()  # noqa: E731
    return [back(t) for t in (o, ts[0].grad, ts[1].grad, ts[2].grad)], [back(t)[..., 0] for t in size], s_max


def check(eng, case, change=lambda q, k, v, dy: None):
    B, S, T, H, G, D, causal, lengths = case
    print(case, end=" ", flush=True)
    r = rng(300 + S + T + D)
    q, dy = (r.standard_normal((B, S, H, D)).astype(np.float32) for _ in range(2))
    k, v = (r.standard_normal((B, T, G, D)).astype(np.float32) for _ in range(2))
    change(q, k, v, dy)
    dev = lambda a, g=False: eng.Tensor(np.array(a, np.float32), requires_grad=g, track=False)  # noqa: E731
    ts = [dev(a, True) for a in (q, k, v)]
    lens = dev(lengths) if lengths is not None else None
    out = eng.attention(*ts, causal=causal, lengths=lens)
    out.backward(dev(dy))
    ref, size, s_max = attend(q, k, v, dy, causal, lengths)
    tol = 2.0 ** -20 * (s_max + 4)
    worst = []
    for got, want, z in zip([out.sync()] + [t.grad.sync() for t in ts], ref, size):
        assert not got[z == 0].any()
        if (z > 0).any():
            worst.append(float((np.linalg.norm(got - want, axis=-1)[z > 0] / z[z > 0]).max()))
    print("o dq dk dv", ["%.2g" % w for w in worst], "tol %.2g" % tol, flush=True)
    assert max(worst) <= tol
    assert np.array_equal(eng.attention(*[dev(a) for a in (q, k, v)], causal=causal, lengths=lens).sync(), out.data)
    eng.end_batch()


NAME = dict(ids=lambda c: "x".join(map(str, c[:6])) + ("c" if c[6] else "") + ("l" if c[7] else ""))
FEW = [  # B, S, T, H, G, D, causal, lengths: S H / G up to 16
    (2, 1, 200, 4, 2, 80, False, [200, 63]),
    (1, 1, 2000, 8, 4, 96, False, None),
    (2, 4, 777, 8, 2, 80, True, [777, 3]),
    (2, 2, 130, 4, 2, 96, True, None),
    (1, 1, 150, 6, 1, 256, False, None),
    (2, 1, 1500, 8, 2, 256, False, [1500, 0]),
    (1, 3, 1111, 5, 1, 200, True, None),
    (1, 2, 300, 7, 1, 131, True, [299]),
    (3, 1, 64, 16, 1, 33, False, [64, 1, 2]),
]


@pytest.mark.parametrize("case", FEW, **NAME)
def test_few_rows(eng, case):
    check(eng, case)


FALLBACK = [  # on parts by their size
    (2, 400, 1500, 1, 1, 128, True, [1500, 700]),
    (3, 515, 777, 6, 3, 96, True, [777, 0, 261]),
    (1, 1500, 1500, 8, 1, 30, True, None),
    (1, 1024, 1024, 8, 8, 64, False, None),
    (2, 700, 700, 12, 4, 40, False, [700, 333]),
    (1, 1100, 1300, 4, 2, 128, True, None),
    (1, 1203, 1203, 3, 1, 97, False, [1111]),
]


@pytest.mark.parametrize("which", ["keys", "gradients"])
@pytest.mark.parametrize("case", FALLBACK, **NAME)
def test_problems_that_parts_do_not_suit(eng, case, which):
    """A key vector, or a row's gradient, 2^20 smaller than its neighbours in each
    head of the first sequence."""
    def change(q, k, v, dy):
        (k if which == "keys" else dy)[0, 5] *= np.float32(2.0 ** -20)
    check(eng, case, change)
