"""Rotary positions and attention over tensors of more than 2^32 bytes: every
result is compared, in pieces, with float64 on the GPU.

Tolerances, relative to the sum of the terms' sizes: rotary 4 * 2^-24 of a
pair's length; attention 2^-20 (s_max + 4), scores carrying 2^-22 s_max and the
four other factors 2^-22 each, times four for the largest of millions.
"""
import ctypes
import math

import pytest
import torch   # ahead of the engine, which then shares its HIP runtime

from tests.helpers import rng

pytestmark = pytest.mark.gpu

LONG, H, D = 1_200_001, 7, 128   # 1.08e9 floats
PIECE = 100_000


class Span:
    def __init__(self, ptr, shape):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<f4", "data": (ptr, False), "strides": None,
                                         "version": 2}


def view(t):
    """The tensor's device memory, for torch (a handle points to a record whose
    first field is the device pointer)."""
    return torch.as_tensor(Span(ctypes.cast(t.gpu_buf, ctypes.POINTER(ctypes.c_void_p))[0], t.shape), device="cuda")


def filled(eng, shape, seed, grad=False):
    t = eng.Tensor.empty(shape, requires_grad=grad, track=False)
    eng.sync_gpu()
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    flat = view(t).view(-1)
    for i in range(0, flat.numel(), 1 << 28):
        flat[i:i + (1 << 28)].normal_(generator=g)
    torch.cuda.synchronize()
    return t


def pieces(n):
    return [slice(i, min(i + PIECE, n)) for i in range(0, n, PIECE)]


def test_rotary_over_a_long_tensor(eng):
    assert LONG * H * D * 4 > 2 ** 32
    print("rotary over", LONG, "tokens", flush=True)
    x = filled(eng, (1, LONG, H, D), 1, True)
    table = eng.rotary_table(500, 96)
    pos = eng.Tensor(rng(1).integers(0, 500, (1, LONG)), track=False)
    y = eng.rotary(x, table, pos)
    y.backward(y)
    eng.sync_gpu()
    X, Y, G, W, P = (view(t) for t in (x, y, x.grad, table, pos))
    for s in pieces(LONG):
        a, b = X[0, s, :, :48].double(), X[0, s, :, 48:96].double()
        w = W.double()[P[0, s].long()][:, None]
        c, n = w[..., 0], w[..., 1]
        want = torch.cat([a * c - b * n, a * n + b * c], -1)
        size = (a * a + b * b).sqrt().repeat(1, 1, 2)
        assert ((Y[0, s, :, :96] - want).abs() <= 4 * 2.0 ** -24 * size).all(), s
        # turned back: two roundings more, and the table's length of a pair
        assert ((G[0, s, :, :96] - torch.cat([a, b], -1)).abs() <= 12 * 2.0 ** -24 * size).all(), s
        assert torch.equal(Y[0, s, :, 96:], X[0, s, :, 96:]) and torch.equal(G[0, s, :, 96:], X[0, s, :, 96:])
    eng.end_batch()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,keys", [(1, LONG), (40, LONG), (LONG, 33)],
                         ids=["token", "rows", "keys"])
def test_attention_over_a_long_tensor(eng, rows, keys):
    """One row and forty over a long cache (fp32 and parts), and many rows over a few keys."""
    print("attention", rows, "x", keys, flush=True)
    q, dy = filled(eng, (1, rows, H, D), 2, True), filled(eng, (1, rows, H, D), 3)
    k, v = filled(eng, (1, keys, H, D), 4, True), filled(eng, (1, keys, H, D), 5, True)
    out = eng.attention(q, k, v)
    out.backward(dy)
    eng.sync_gpu()
    Q, Y, K, V, O, dQ, dK, dV = (view(t)[0] for t in (q, dy, k, v, out, q.grad, k.grad, v.grad))
    long = lambda t: t.norm(dim=-1, keepdim=True)  # noqa: E731

    def off(got, want, size):
        return float(((got - want).norm(dim=-1, keepdim=True) / size).max())
    for h in range(H):
        worst, s_max = {}, 0.0
        if keys > rows:      # rows kept, keys in pieces
            qh, yh = Q[:, h].double(), Y[:, h].double()
            s = torch.cat([qh @ K[p, h].double().t() for p in pieces(keys)], 1) / math.sqrt(D)
            s_max = float(s.abs().max())
            P = torch.softmax(s, 1)
            o = sum(P[:, p] @ V[p, h].double() for p in pieces(keys))
            o_size = sum(P[:, p] @ long(V[p, h].double()) for p in pieces(keys))
            delta = (yh * o).sum(1, keepdim=True)
            dq, dq_size = torch.zeros_like(qh), torch.zeros_like(o_size)
            worst["o"] = off(O[:, h], o, o_size)
            for p in pieces(keys):
                kh, vh = K[p, h].double(), V[p, h].double()
                ds = P[:, p] * (yh @ vh.t() - delta) / math.sqrt(D)
                size = P[:, p] * (long(yh) * long(vh).t() + long(yh) * o_size) / math.sqrt(D)
                dq += ds @ kh
                dq_size += size @ long(kh)
                worst["dk"] = max(worst.get("dk", 0), off(dK[p, h], ds.t() @ qh, size.t() @ long(qh)))
                worst["dv"] = max(worst.get("dv", 0), off(dV[p, h], P[:, p].t() @ yh, P[:, p].t() @ long(yh)))
            worst["dq"] = off(dQ[:, h], dq, dq_size)
        else:                # keys kept, rows in pieces
            kh, vh = K[:, h].double(), V[:, h].double()
            sums = [torch.zeros_like(kh), torch.zeros_like(kh), torch.zeros_like(long(kh)), torch.zeros_like(long(kh))]
            for p in pieces(rows):
                qh, yh = Q[p, h].double(), Y[p, h].double()
                s = qh @ kh.t() / math.sqrt(D)
                s_max = max(s_max, float(s.abs().max()))
                P = torch.softmax(s, 1)
                o, o_size = P @ vh, P @ long(vh)
                ds = P * (yh @ vh.t() - (yh * o).sum(1, keepdim=True)) / math.sqrt(D)
                size = P * (long(yh) * long(vh).t() + long(yh) * o_size) / math.sqrt(D)
                worst["o"] = max(worst.get("o", 0), off(O[p, h], o, o_size))
                worst["dq"] = max(worst.get("dq", 0), off(dQ[p, h], ds @ kh, size @ long(kh)))
                for t, add in zip(sums, (ds.t() @ qh, P.t() @ yh, size.t() @ long(qh), P.t() @ long(yh))):
                    t += add
            worst["dk"], worst["dv"] = off(dK[:, h], sums[0], sums[2]), off(dV[:, h], sums[1], sums[3])
        tol = 2.0 ** -20 * (s_max + 4)
        print(h, {n: "%.2g" % e for n, e in worst.items()}, "tol %.2g" % tol, flush=True)
        assert max(worst.values()) <= tol
    eng.end_batch()
    torch.cuda.empty_cache()
