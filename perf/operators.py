"""Timing cases of the operators that train a transformer block: rotary
positions, attention forward and backward, and the orthogonalised update.

listed() names the cases, draw(rng) gives more of the same ranges, prepare()
builds what a program holds before the call, run() is one pass, work() the
bytes and operations the pass cannot do without, exact() the same outputs in
64 bits.  With `own` false, run() is the plain form: elementary torch
operations in 32 bits.
"""
import ctypes
import math

import torch

own = False
GPU = "cuda"


# --------------------------------------------------------------------------
# The cases
# --------------------------------------------------------------------------
def _rotary(batch, seq, heads, dim, part, interleaved, train, factor=1.0, scattered=0):
    return dict(kind="rotary", batch=batch, seq=seq, heads=heads, dim=dim, part=part, interleaved=interleaved,
                train=train, factor=factor, scattered=scattered)


def _attention(batch, seq, keys, heads, kv, dim, causal, ragged, train):
    return dict(kind="attention", batch=batch, seq=seq, keys=keys, heads=heads, kv=kv, dim=dim, causal=causal,
                ragged=ragged, train=train)


def _muon(shapes):
    return dict(kind="muon", shapes=shapes)


LENET = "6x1x5x5+16x6x5x5+256x120+120x84+84x10"
ALEXNET = "64x3x11x11+192x64x5x5+384x192x3x3+256x384x3x3+256x256x3x3+9216x4096+4096x4096+4096x1000"
UNET = "+".join("%dx%dx3x3" % p for p in [
    (16, 3), (16, 16), (32, 16), (32, 32), (64, 32), (64, 64), (128, 64), (128, 128), (256, 128), (256, 256),
    (128, 384), (128, 128), (64, 192), (64, 64), (32, 96), (32, 32), (16, 48), (16, 16)]) + "+1x16x1x1"


def listed():
    return [
        # One new token for each of eight sequences, at positions of their own: latency alone.
        dict(_rotary(8, 1, 16, 64, 64, 0, 0, scattered=1), name="rotary_token_b8"),
        # Queries of a training batch, forward and backward, three quarters of the head, contexts stretched 8 times.
        dict(_rotary(4, 4096, 32, 128, 96, 0, 1, factor=8.0), name="rotary_train_4096"),
        # A ragged batch in the interleaved layout.
        dict(_rotary(3, 1001, 12, 80, 80, 1, 1), name="rotary_interleaved_1001"),
        # One new token for each of eight sequences over caches of up to 8191 tokens, four queries to a key head.
        dict(_attention(8, 1, 8191, 32, 8, 128, 0, 1, 0), name="attn_token_8191"),
        # An image's patches, all to all, evaluated: an odd length.
        dict(_attention(16, 197, 197, 6, 6, 64, 0, 0, 0), name="attn_patches_197"),
        # A long prompt, evaluated: causal, four queries to a key head.
        dict(_attention(1, 8192, 8192, 16, 4, 128, 1, 0, 0), name="attn_prompt_8192"),
        # The smallest training batch: short sentences.
        dict(_attention(2, 77, 77, 8, 8, 64, 1, 0, 1), name="attn_train_77"),
        # A padded training batch of odd length, three queries to a key head.
        dict(_attention(4, 1000, 1000, 12, 4, 64, 1, 1, 1), name="attn_train_1000_padded"),
        # The largest training batch.
        dict(_attention(2, 4096, 4096, 16, 16, 128, 1, 0, 1), name="attn_train_4096"),
        # The update of LeNet-5's matrices: launches alone.
        dict(_muon(LENET), name="muon_lenet"),
        # The update of the UNet-base16's filters: many small, oblong matrices.
        dict(_muon(UNET), name="muon_unet"),
        # The update of AlexNet's filters and linear layers: few large matrices.
        dict(_muon(ALEXNET), name="muon_alexnet"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "token", "eval", "train", "train", "muon", "muon"])
    if kind == "rotary":
        while True:
            dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
            c = _rotary(_log(rng, 1, 8), _log(rng, 1, 4096), _log(rng, 1, 32), dim, rng.choice([dim, dim, dim // 2, dim // 4 * 3]),
                        rng.choice([0, 1]), rng.choice([0, 1]), rng.choice([1.0, 1.0, 4.0, 8.0]), rng.choice([0, 0, 1]))
            if work(c)["bytes"] <= 1.1e9:
                return c
    if kind == "muon":
        while True:
            n = _log(rng, 1, 20)
            if rng.random() < 0.4:
                k = rng.choice([1, 3, 5])
                shapes = ["%dx%dx%dx%d" % (_log(rng, 4, 384), _log(rng, 1, 384), k, k) for _ in range(n)]
            else:
                shapes = ["%dx%d" % (_log(rng, 10, 4096), _log(rng, 10, 4096)) for _ in range(n)]
            c = _muon("+".join(shapes))
            if work(c)["flops"] <= 2e12:
                return c
    while True:
        kv = rng.choice([1, 2, 4, 6, 8])
        heads = kv * rng.choice([1, 1, 2, 3, 4])
        dim = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
        if kind == "token":
            c = _attention(_log(rng, 1, 32), 1, _log(rng, 1, 16384), heads, kv, dim, 0, rng.choice([0, 1]), 0)
        else:
            seq = _log(rng, 16, 8192 if kind == "eval" else 4096)
            keys = seq if rng.random() < 0.7 else seq + _log(rng, 1, 2048)
            c = _attention(_log(rng, 1, 16), seq, keys, heads, kv, dim, rng.choice([0, 1, 1]), rng.choice([0, 0, 1]),
                           int(kind == "train"))
        w = work(c)
        scores = c["batch"] * heads * c["seq"] * c["keys"]
        if w["flops"] <= 4.5e11 and w["bytes"] <= 2e9 and scores <= 8e8:
            return c


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _shapes(case):
    return [tuple(int(d) for d in s.split("x")) for s in case["shapes"].split("+")]


def _flat(shape):
    return shape[0], math.prod(shape[1:])


ORIGINAL = 4096  # the context a stretched rotary table starts from
BASE = 10000.0
LR, MU, DECAY, STEPS, RMS = 0.02, 0.95, 0.01, 5, 0.2


def _positions(case):
    """Rows of the rotary table."""
    return int(case["seq"] if not case["scattered"] else 4096) if case["factor"] == 1.0 else int(ORIGINAL * case["factor"])


def _lengths(case):
    """Valid keys of each sequence: from all of them down to about half."""
    b, t = case["batch"], case["keys"]
    return [t - (i * t) // (2 * b) for i in range(b)] if case["ragged"] else None


def _data(case, seed):
    g = torch.Generator(device=GPU)
    g.manual_seed(seed)

    def normal(shape, spread=1.0):
        return torch.randn(shape, generator=g, device=GPU).mul_(spread)

    kind = case["kind"]
    if kind == "muon":
        shapes = _shapes(case)
        # weights as initialised, gradients of a norm near 1, a momentum that has run for a while
        return {"w": [normal(s, 1 / math.sqrt(_flat(s)[1])) for s in shapes],
                "g": [normal(s, 1 / math.sqrt(math.prod(s))) for s in shapes],
                "m": [normal(s, 3 / math.sqrt(math.prod(s))) for s in shapes]}
    b, s, h, d = case["batch"], case["seq"], case["heads"], case["dim"]
    if kind == "rotary":
        r = {"x": normal((b, s, h, d)), "pos": None}
        if case["scattered"]:
            r["pos"] = torch.randint(0, _positions(case), (b, s), generator=g, device=GPU).float()
        if case["train"]:
            r["dy"] = normal((b, s, h, d), 1 / math.sqrt(s))
        return r
    t, kv = case["keys"], case["kv"]
    # queries and keys as normalised projections have them: scores of a spread of about 1.5
    r = {"q": normal((b, s, h, d), 1.5), "k": normal((b, t, kv, d)), "v": normal((b, t, kv, d)), "len": None}
    if case["ragged"]:
        r["len"] = torch.tensor(_lengths(case), dtype=torch.float32, device=GPU)
    if case["train"]:
        r["dy"] = normal((b, s, h, d), 1 / math.sqrt(s))
    return r


class _Span:
    def __init__(self, ptr, shape):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<f4", "data": (ptr, False),
                                         "strides": None, "version": 2}


def _view(t):
    """An engine tensor's device memory as a torch tensor (no copy): a handle
    points to a record whose first field is the device pointer."""
    ptr = ctypes.cast(t.gpu_buf, ctypes.POINTER(ctypes.c_void_p))[0]
    return torch.as_tensor(_Span(ptr, t.shape), device=GPU)


def _held(v, grad=False):
    """A torch tensor as the program holds it: as it is, or as the engine's."""
    if not own or v is None:
        return v
    from directcompute_torch_amd import nn_engine as nn
    t = nn.Tensor.empty(tuple(v.shape), requires_grad=grad, track=False)
    nn.sync_gpu()
    _view(t).copy_(v)
    torch.cuda.synchronize()
    return t


def _frequencies(part, factor):
    """Radians per position of each pair, in 64 bits.  A stretched table keeps
    the fast pairs (over 32 turns in the original context), slows the slow ones
    (under one turn) by the factor, and goes linearly between them."""
    f = BASE ** (-torch.arange(0, part, 2, dtype=torch.float64, device=GPU) / part)
    if factor == 1.0:
        return f
    keep = ((ORIGINAL * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
    return f * keep + f / factor * (1 - keep)


def prepare(case, seed):
    d, kind = _data(case, seed), case["kind"]
    s = {"case": case}
    if kind == "muon":
        s["w"], s["g"] = [_held(w, True) for w in d["w"]], [_held(g) for g in d["g"]]
        if own:
            from directcompute_torch_amd import nn_engine as nn
            s["opt"] = nn.Muon(s["w"], lr=LR, momentum=MU, weight_decay=DECAY, steps=STEPS, rms=RMS)
            nn.sync_gpu()  # its zeros are on their way, on another stream than torch's
            for have, m in zip(s["opt"].m, d["m"]):
                _view(have).copy_(m)
        else:
            s["m"] = d["m"]
        return s
    train = bool(case["train"])
    for k in ("x", "q", "k", "v"):
        if k in d:
            s[k] = _held(d[k], train)
    for k in ("dy", "pos", "len"):
        s[k] = _held(d.get(k))
    if kind == "rotary":  # the table, laid out once
        if own:
            from directcompute_torch_amd import nn_engine as nn
            s["table"] = nn.rotary_table(_positions(case), case["part"], base=BASE, factor=case["factor"],
                                         original=None if case["factor"] == 1.0 else ORIGINAL)
        else:
            a = torch.arange(_positions(case), dtype=torch.float64, device=GPU)[:, None] * _frequencies(case["part"], case["factor"])
            s["table"] = torch.stack([a.cos(), a.sin()], -1).float()
    return s


# --------------------------------------------------------------------------
# One pass, plain
# --------------------------------------------------------------------------
def _rotate(x, table, pos, part, interleaved, sign):
    seq = x.shape[1]
    rows = table[pos.long()] if pos is not None else table[:seq][None]
    c, s = rows[..., 0][:, :, None], rows[..., 1][:, :, None] * sign
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:part:2], x[..., 1:part:2]
        y[..., 0:part:2], y[..., 1:part:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :part // 2], x[..., part // 2:part]
        y[..., :part // 2], y[..., part // 2:part] = a * c - b * s, a * s + b * c
    return y


def _allowed(case, lengths):
    """(batch or 1, 1, seq, keys) truth values: query i sits at position i + keys - seq."""
    seq, keys = case["seq"], case["keys"]
    j = torch.arange(keys, device=GPU)
    ok = torch.ones((1, 1, seq, keys), dtype=torch.bool, device=GPU)
    if case["causal"]:
        ok = (j[None] <= torch.arange(seq, device=GPU)[:, None] + (keys - seq))[None, None]
    if lengths is not None:
        ok = ok & (j[None, None, None] < lengths.long()[:, None, None, None])
    return ok


def _attend(case, q, k, v, lengths, dy):
    b, _, h, d = q.shape
    kv, rep, scale = case["kv"], case["heads"] // case["kv"], 1 / math.sqrt(d)
    q = q.permute(0, 2, 1, 3)
    kr, vr = (t.permute(0, 2, 1, 3).repeat_interleave(rep, 1) for t in (k, v))
    p = torch.matmul(q * scale, kr.transpose(2, 3))
    if case["causal"] or lengths is not None:
        p.masked_fill_(~_allowed(case, lengths), -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.mul_(torch.where(total > 0, 1 / total, 0.0))
    out = torch.matmul(p, vr)
    got = {"out": out.permute(0, 2, 1, 3).contiguous()}
    if dy is None:
        return got
    dy = dy.permute(0, 2, 1, 3)
    dv = torch.matmul(p.transpose(2, 3), dy)
    dp = torch.matmul(dy, vr.transpose(2, 3))
    dp.sub_((dy * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dk = torch.matmul(dp.transpose(2, 3), q)
    got["dq"] = torch.matmul(dp, kr).permute(0, 2, 1, 3).contiguous()
    for name, t in (("dk", dk), ("dv", dv)):
        got[name] = t.view(b, kv, rep, -1, d).sum(2).permute(0, 2, 1, 3).contiguous()
    return got


def _orthogonalised(d):
    x = d.t() if d.shape[0] > d.shape[1] else d
    x = x / (x.square().sum().sqrt() + 1e-7)
    for _ in range(STEPS):
        a = x @ x.t()
        x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
    return x.t() if d.shape[0] > d.shape[1] else x


def _update(w, g, m):
    g = g.clamp(-1.0, 1.0)
    m.mul_(MU).add_(g)
    rows, cols = _flat(w.shape)
    o = _orthogonalised((g + MU * m).reshape(rows, cols)).reshape(w.shape)
    w.copy_(w - LR * DECAY * w - LR * RMS * math.sqrt(max(rows, cols)) * o)


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if own:
        from directcompute_torch_amd import nn_engine as nn
        nn.end_batch()  # the previous batch's buffers, as a training loop does after each batch
        if kind == "muon":
            for w, g in zip(s["w"], s["g"]):
                w.grad = g
            s["opt"].step(clip=1.0)
            return {"w": [_view(w) for w in s["w"]], "m": [_view(m) for m in s["opt"].m]}
        if kind == "rotary":
            s["x"].grad = None
            y = nn.rotary(s["x"], s["table"], s["pos"], interleaved=bool(case["interleaved"]))
            if not case["train"]:
                return {"y": _view(y)}
            y.backward(s["dy"])
            return {"y": _view(y), "dx": _view(s["x"].grad)}
        for k in ("q", "k", "v"):
            s[k].grad = None
        out = nn.attention(s["q"], s["k"], s["v"], causal=bool(case["causal"]), lengths=s["len"])
        if not case["train"]:
            return {"out": _view(out)}
        out.backward(s["dy"])
        return {"out": _view(out), "dq": _view(s["q"].grad), "dk": _view(s["k"].grad), "dv": _view(s["v"].grad)}
    if kind == "muon":
        for w, g, m in zip(s["w"], s["g"], s["m"]):
            _update(w, g, m)
        return {"w": s["w"], "m": s["m"]}
    if kind == "rotary":
        got = {"y": _rotate(s["x"], s["table"], s["pos"], case["part"], case["interleaved"], 1.0)}
        if case["train"]:
            got["dx"] = _rotate(s["dy"], s["table"], s["pos"], case["part"], case["interleaved"], -1.0)
        return got
    return _attend(case, s["q"], s["k"], s["v"], s["len"], s["dy"])


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "muon":
        values = flops = 0.0
        for s in _shapes(case):
            m, n = sorted(_flat(s))
            values += m * n
            # two symmetric products (X X^T and A A, half of each) and one whole one
            flops += STEPS * (m * m * n + m ** 3 + 2.0 * m * m * n)
        return {"bytes": 20.0 * values, "flops": flops}
    b, s, h, d = case["batch"], case["seq"], case["heads"], case["dim"]
    if kind == "rotary":
        passes = 1 + case["train"]
        table = 4.0 * case["part"] * (s if not case["scattered"] else b * s)
        return {"bytes": passes * 8.0 * b * s * h * d + table, "flops": passes * 3.0 * b * s * h * case["part"]}
    t, kv = case["keys"], case["kv"]
    lengths = _lengths(case) or [t] * b
    if case["causal"]:  # query i sees keys 0 .. i + t - s, up to the length
        pairs = sum(min(max(i + t - s + 1, 0), n) for n in lengths for i in range(s))
    else:
        pairs = sum(lengths) * s
    q, k = 4.0 * b * s * h * d, 4.0 * sum(lengths) * kv * d
    flops, moved = 4.0 * d * h * pairs, 2 * q + 2 * k
    if case["train"]:  # dy and o read, dq written; k and v read, dk and dv written
        flops, moved = flops * 3.5, moved + 3 * q + 4 * k
    return {"bytes": moved, "flops": flops}


# --------------------------------------------------------------------------
# The same outputs in 64 bits
# --------------------------------------------------------------------------
def _exact_rotary(case, d):
    # as a product of complex numbers
    part, half = case["part"], case["part"] // 2
    pos = d["pos"].double() if d["pos"] is not None else torch.arange(case["seq"], dtype=torch.float64, device=GPU)[None]
    f = torch.pow(torch.tensor(BASE, dtype=torch.float64, device=GPU), -2.0 * torch.arange(half, dtype=torch.float64, device=GPU) / part)
    if case["factor"] != 1.0:
        turns = ORIGINAL * f / (2 * math.pi)
        mix = torch.clamp((turns - 1) / 31, min=0, max=1)
        f = mix * f + (1 - mix) * f / case["factor"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=GPU), pos[..., None] * f)[:, :, None]

    def spun(x, by):
        x = x.double()
        pairs = x[..., :part].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
        if not case["interleaved"]:
            pairs = pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        z = z if case["interleaved"] else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), x[..., part:]], -1)

    got = {"y": spun(d["x"], turn)}
    if case["train"]:
        got["dx"] = spun(d["dy"], turn.conj())
    return got


def _exact_attention(case, d):
    # sequence by sequence and head by head, the gradients from autograd
    lengths, rep = _lengths(case) or [case["keys"]] * case["batch"], case["heads"] // case["kv"]
    seq, keys = case["seq"], case["keys"]
    train = bool(case["train"])
    q, k, v = (d[n].double() for n in ("q", "k", "v"))
    got = {"out": torch.zeros_like(q)}
    if train:
        got.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    last = torch.arange(seq, device=GPU)[:, None] + (keys - seq if case["causal"] else keys)
    for b, n in enumerate(lengths):
        ok = torch.arange(n, device=GPU)[None] <= last
        rows = ok.any(1)
        for h in range(case["heads"]):
            qq, kk, vv = q[b, rows, h], k[b, :n, h // rep], v[b, :n, h // rep]
            if train:
                qq, kk, vv = (t.detach().requires_grad_(True) for t in (qq, kk, vv))
            bias = torch.where(ok[rows], 0.0, -math.inf).double()
            o = torch.softmax(qq @ kk.t() / math.sqrt(case["dim"]) + bias, -1) @ vv
            got["out"][b, rows, h] = o.detach()
            if train:
                gq, gk, gv = torch.autograd.grad(o, (qq, kk, vv), d["dy"][b, rows, h].double())
                got["dq"][b, rows, h] = gq
                got["dk"][b, :n, h // rep] += gk
                got["dv"][b, :n, h // rep] += gv
    return got


def _exact_muon(d):
    # X after k steps is a polynomial P in the Gram matrix G of the first X, times that X
    got = {"w": [], "m": []}
    for w, g, m in zip(d["w"], d["g"], d["m"]):
        w, g, m = w.double(), g.double().clamp(-1, 1), m.double()
        m = MU * m + g
        rows, cols = _flat(w.shape)
        x = (g + MU * m).reshape(rows, cols)
        x = x / (torch.linalg.vector_norm(x) + 1e-7)
        wide = rows <= cols
        gram = x @ x.t() if wide else x.t() @ x
        one = torch.eye(min(rows, cols), dtype=torch.float64, device=GPU)
        p = one
        for _ in range(STEPS):
            a = p @ gram @ p
            p = (3.4445 * one - 4.7750 * a + 2.0315 * (a @ a)) @ p
        o = (p @ x if wide else x @ p).reshape(w.shape)
        got["w"].append(w * (1 - LR * DECAY) - LR * RMS * math.sqrt(max(rows, cols)) * o)
        got["m"].append(m)
    return got


def exact(case, seed):
    d = _data(case, seed)
    if case["kind"] == "muon":
        return _exact_muon(d)
    return (_exact_rotary if case["kind"] == "rotary" else _exact_attention)(case, d)
