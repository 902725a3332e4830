"""Timing cases of the operators beside attention in a block: the norms around
its residual stream, the gated feed-forward block, and the gated linear
recurrence.

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
EPS = 1e-6


# --------------------------------------------------------------------------
# The cases
# --------------------------------------------------------------------------
def _norm(batch, seq, width, gate, post, pre, scale, train):
    """gate: "none", "channel" (one row), "sequence" (a row each) or "token" (every value's own)."""
    return dict(kind="norm", batch=batch, seq=seq, width=width, gate=gate, post=post, pre=pre, scale=scale, train=train)


def _mlp(rows, width, hidden, act, train):
    return dict(kind="mlp", rows=rows, width=width, hidden=hidden, act=act, train=train)


def _scan(batch, seq, width, ragged, state, train):
    return dict(kind="scan", batch=batch, seq=seq, width=width, ragged=ragged, state=state, train=train)


def listed():
    return [
        # One new token for each of eight sequences between two halves of a block: latency alone.
        dict(_norm(8, 1, 2048, "channel", 1, 1, 1.0, 0), name="norm_token_b8"),
        # A padded training batch of odd width whose gate comes from a condition of each sequence.
        dict(_norm(4, 1001, 771, "sequence", 0, 1, 0.5, 1), name="norm_adaptive_1001"),
        # A long prompt, evaluated: every value has a gate of its own.
        dict(_norm(1, 8191, 4096, "token", 1, 1, 1.0, 0), name="norm_prompt_8191"),
        # The largest training batch: both norms, a gate for each channel.
        dict(_norm(2, 4096, 2048, "channel", 1, 1, 1.0, 1), name="norm_train_4096"),
        # One new token for each of eight sequences: the weights are read once.
        dict(_mlp(8, 1024, 2816, "silu", 0), name="mlp_token_b8"),
        # A training batch of two short sentences, odd widths.
        dict(_mlp(154, 384, 1001, "gelu", 1), name="mlp_train_154"),
        # A long prompt, evaluated.
        dict(_mlp(4096, 1024, 2816, "gelu", 0), name="mlp_prompt_4096"),
        # The largest training batch.
        dict(_mlp(8192, 1024, 4096, "silu", 1), name="mlp_train_8192"),
        # One new token for each of eight sequences, from their states.
        dict(_scan(8, 1, 2048, 0, 1, 0), name="scan_token_b8"),
        # A padded training batch of odd length and width that goes on from a state.
        dict(_scan(3, 1001, 771, 1, 1, 1), name="scan_train_1001_padded"),
        # One very long prompt of few channels, evaluated.
        dict(_scan(1, 32768, 512, 0, 0, 0), name="scan_prompt_32768"),
        # The largest training batch.
        dict(_scan(4, 4096, 1024, 0, 0, 1), name="scan_train_4096"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "mlp", "mlp", "scan"])
    while True:
        train = rng.choice([0, 1])
        if kind == "norm":
            post, pre = rng.choice([(0, 1), (1, 1), (1, 1), (1, 0)])
            width = _log(rng, 32, 8192) if rng.random() < 0.5 else 64 * _log(rng, 1, 128)
            c = _norm(_log(rng, 1, 16), _log(rng, 1, 8192), width, rng.choice(["none", "channel", "sequence", "token"]),
                      post, pre, rng.choice([1.0, 1.0, 0.5]), train)
        elif kind == "mlp":
            if rng.random() < 0.5:
                width, hidden = _log(rng, 32, 2048), _log(rng, 32, 8192)
            else:
                width, hidden = 64 * _log(rng, 1, 32), 64 * _log(rng, 1, 128)
            rows = _log(rng, 1, 16) if rng.random() < 0.25 else _log(rng, 16, 8192)
            c = _mlp(rows, width, hidden, rng.choice(["silu", "silu", "gelu", "relu", "sigmoid"]), train)
        else:
            c = _scan(_log(rng, 1, 16), _log(rng, 1, 32768), _log(rng, 32, 4096), rng.choice([0, 0, 1]), rng.choice([0, 1]), train)
        w = work(c)
        if w["flops"] <= 6.2e11 and w["bytes"] <= 7e8:
            return c


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _gate_rows(case):
    return {"none": 0, "channel": 1, "sequence": case["batch"], "token": case["batch"] * case["seq"]}[case["gate"]]


def _lengths(case):
    """Tokens of each sequence: from all of them down to about half."""
    b, s = case["batch"], case["seq"]
    return [s - (i * s) // (2 * b) for i in range(b)] if case["ragged"] else None


def _data(case, seed):
    g = torch.Generator(device=GPU)
    g.manual_seed(seed)

    def normal(shape, spread=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device=GPU).mul_(spread).add_(mean)

    kind, d = case["kind"], {}
    if kind == "mlp":
        m, c, f = case["rows"], case["width"], case["hidden"]
        # a normalised input and weights as initialised
        d.update(x=normal((m, c)), wg=normal((c, f), c ** -0.5), wu=normal((c, f), c ** -0.5), wd=normal((f, c), f ** -0.5))
        if case["train"]:
            d["dy"] = normal((m, c), m ** -0.5)
        return d
    shape = b, s, c = case["batch"], case["seq"], case["width"]
    if kind == "norm":
        # a residual stream that has grown, and a block's output
        d.update(x=normal(shape, 3.0), block=normal(shape))
        if case["gate"] != "none":
            d["gate"] = normal((_gate_rows(case), c), 0.3, 0.5)
        for k in ("post", "pre"):
            if case[k]:
                d[k] = normal((c,), 0.2, 1.0)
        if case["train"]:
            d["dh"] = normal(shape, s ** -0.5)
            if case["pre"]:
                d["dn"] = normal(shape, s ** -0.5)
        return d
    # gates that remember: from a few to some hundred tokens
    d.update(x=normal(shape), z=normal(shape, 1.5, 2.0))
    if case["state"]:
        d["state"] = normal((b, c))
    if case["ragged"]:
        d["len"] = torch.tensor(_lengths(case), dtype=torch.float32, device=GPU)
    if case["train"]:
        d["dy"] = normal(shape, s ** -0.5)
    return d


class _Span:
    def __init__(self, ptr, shape):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": "<f4", "data": (ptr, False),
                                         "strides": None, "version": 2}


def _view(t):
    """An engine tensor's device memory as a torch tensor (no copy): a handle
    points to a record whose first field is the device pointer."""
    ptr = ctypes.cast(t.gpu_buf, ctypes.POINTER(ctypes.c_void_p))[0]
    return torch.as_tensor(_Span(ptr, t.shape), device=GPU)


def _held(v, grad):
    """A torch tensor as the program holds it: as it is, or as the engine's."""
    if not own:
        return v
    from directcompute_torch_amd import nn_engine as nn
    t = nn.Tensor.empty(tuple(v.shape), requires_grad=grad, track=False)
    nn.sync_gpu()
    _view(t).copy_(v)
    torch.cuda.synchronize()
    return t


FIXED = ("dy", "dh", "dn", "len")  # what needs no gradient


def prepare(case, seed):
    s = {k: _held(v, bool(case["train"]) and k not in FIXED) for k, v in _data(case, seed).items()}
    s["case"] = case
    return s


# --------------------------------------------------------------------------
# One pass, plain
# --------------------------------------------------------------------------
def _rstd(x):
    return torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _unnormed(x, r, gain, dy):
    """Gradients of x r gain, r = _rstd(x), with respect to x and gain."""
    w = dy * gain
    dx = r * (w - x * (r * r * (w * x).mean(-1, keepdim=True)))
    return dx, (dy * x * r).flatten(0, 1).sum(0)


def _norms(case, s):
    b, seq, c = shape = s["x"].shape
    x, block, post, pre = s["x"], s["block"], s.get("post"), s.get("pre")
    gate = None
    if "gate" in s:
        rows = s["gate"].shape[0]
        gate = s["gate"].view((b, 1, c) if rows == b else (1, 1, c) if rows == 1 else shape)
    got = {}
    u = block
    if post is not None:
        r1 = _rstd(block)
        u = block * r1 * post
    h = case["scale"] * x + (u if gate is None else gate * u)
    got["h"] = h
    if pre is not None:
        r2 = _rstd(h)
        got["n"] = h * r2 * pre
    if not case["train"]:
        return got
    t = s["dh"]
    if pre is not None:
        dt, got["dpre"] = _unnormed(h, r2, pre, s["dn"])
        t = t + dt
    got["dx"] = case["scale"] * t
    du = t
    if gate is not None:
        du = gate * t
        dgate = t * u
        got["dgate"] = dgate.flatten(0, 1) if rows == b * seq else dgate.sum(1) if rows == b else dgate.sum((0, 1)).view(1, c)
    if post is not None:
        du, got["dpost"] = _unnormed(block, r1, post, du)
    got["dblock"] = du
    return got


def _activated(g, act):
    """act(g) and its derivative."""
    if act == "relu":
        on = (g > 0).float()
        return g * on, on
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    p = 1 / (1 + torch.exp(-g))
    if act == "sigmoid":
        return p, p * (1 - p)
    return g * p, p + g * p * (1 - p)


def _feed(case, s):
    x, wg, wu, wd = s["x"], s["wg"], s["wu"], s["wd"]
    u = x @ wu
    a, da = _activated(x @ wg, case["act"])
    m = a * u
    got = {"y": m @ wd}
    if case["train"]:
        dm = s["dy"] @ wd.t()
        du, dg = dm * a, dm * u * da
        got.update(dx=dg @ wg.t() + du @ wu.t(), dwg=x.t() @ dg, dwu=x.t() @ du, dwd=m.t() @ s["dy"])
    return got


def _scanned(a, b):
    """h_t = a_t h_(t-1) + b_t along the second axis: pairs (a, b) of runs of 1, 2, 4, ... tokens."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _recur(case, s):
    x, z, seq = s["x"], s["z"], s["x"].shape[1]
    f, k = 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))
    first = s["state"] if "state" in s else torch.zeros_like(x[:, 0])
    ins = k * x
    if "len" in s:  # tokens past the last leave the state as it is
        live = (torch.arange(seq, device=GPU)[None] < s["len"].long()[:, None])[..., None]
        f, ins = torch.where(live, f, 1.0), torch.where(live, ins, 0.0)
    ins = torch.cat([ins[:, :1] + f[:, :1] * first[:, None], ins[:, 1:]], 1)
    h = _scanned(f, ins)
    y = torch.where(live, h, 0.0) if "len" in s else h
    got = {"y": y, "last": h[:, -1].contiguous()}
    if not case["train"]:
        return got
    dy = torch.where(live, s["dy"], 0.0) if "len" in s else s["dy"]
    later = torch.cat([f[:, 1:], torch.zeros_like(f[:, :1])], 1)
    dh = _scanned(later.flip(1), dy.flip(1)).flip(1)
    before = torch.cat([first[:, None], h[:, :-1]], 1)
    dx, dz = k * dh, dh * (before - x) * f * k
    got["dx"] = torch.where(live, dx, 0.0) if "len" in s else dx
    got["dz"] = torch.where(live, dz, 0.0) if "len" in s else dz
    if "state" in s:
        got["dstate"] = f[:, 0] * dh[:, 0]
    return got


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def _own(case, s):
    from directcompute_torch_amd import nn_engine as nn
    nn.end_batch()  # the previous batch's buffers, as a training loop does after each batch
    train = bool(case["train"])
    names = {"norm": ("x", "block", "gate", "post", "pre"), "mlp": ("x", "wg", "wu", "wd"), "scan": ("x", "z", "state")}
    leaves = [k for k in names[case["kind"]] if k in s]
    for k in leaves:
        s[k].grad = None
    if case["kind"] == "norm":
        got = nn.residual_norm(s["x"], s["block"], gate=s.get("gate"), post=s.get("post"), pre=s.get("pre"),
                               scale=case["scale"], eps=EPS)
        h, n = got if case["pre"] else (got, None)
        got = {"h": h} if n is None else {"h": h, "n": n}
        if train and n is not None:
            h.grad = s["dh"]  # as the rest of the network has left it
            n.backward(s["dn"])
        elif train:
            h.backward(s["dh"])
    elif case["kind"] == "mlp":
        got = {"y": nn.gated_mlp(s["x"], s["wg"], s["wu"], s["wd"], act=case["act"])}
        if train:
            got["y"].backward(s["dy"])
    else:
        y, last = nn.gated_scan(s["x"], s["z"], state=s.get("state"), lengths=s.get("len"), return_state=True)
        got = {"y": y, "last": last}
        if train:
            y.backward(s["dy"])
    if train:
        got.update({"d" + k: s[k].grad for k in leaves})
    return {k: _view(t) for k, t in got.items()}


def run(s):
    case = s["case"]
    if own:
        return _own(case, s)
    return {"norm": _norms, "mlp": _feed, "scan": _recur}[case["kind"]](case, s)


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    train = case["train"]
    if case["kind"] == "mlp":
        m, c, f = case["rows"], case["width"], case["hidden"]
        return {"bytes": (1 + train) * 4.0 * (2 * m * c + 3 * c * f), "flops": (1 + 2 * train) * 6.0 * m * c * f}
    n = float(case["batch"] * case["seq"] * case["width"])
    if case["kind"] == "norm":
        gate = 4.0 * _gate_rows(case) * case["width"]
        gains = 4.0 * case["width"] * (case["post"] + case["pre"])
        moved, ops = 4.0 * (3 + case["pre"]) * n + gate + gains, 4.0 + 4 * case["post"] + 4 * case["pre"]
        if train:  # dh, dn read, dx and the block's gradient written; x is read only once
            moved, ops = moved + 4.0 * (3 + case["pre"]) * n + gate + gains, ops * 3
        return {"bytes": moved, "flops": ops * n}
    lengths = _lengths(case)
    live = float(sum(lengths) * case["width"]) if lengths else n
    state = 4.0 * case["batch"] * case["width"]
    moved = 8.0 * live + 4.0 * n + state * (1 + case["state"])
    if train:  # dy read, dx and dz written
        moved += 4.0 * live + 8.0 * n + state * case["state"]
    return {"bytes": moved, "flops": (6.0 + 10.0 * train) * live}


# --------------------------------------------------------------------------
# The same outputs in 64 bits
# --------------------------------------------------------------------------
def _exact_norm(case, d):
    # the gradients from autograd
    leaves = {k: d[k].double().requires_grad_(bool(case["train"])) for k in ("x", "block", "gate", "post", "pre") if k in d}
    b, s, c = d["x"].shape

    def normed(v, gain):
        return v / torch.sqrt(torch.linalg.vector_norm(v, dim=-1, keepdim=True) ** 2 / c + EPS) * gain

    u = normed(leaves["block"], leaves["post"]) if "post" in leaves else leaves["block"]
    if "gate" in leaves:
        g = leaves["gate"]
        u = u * g.repeat_interleave(b * s // g.shape[0], 0).view(b, s, c)
    h = case["scale"] * leaves["x"] + u
    outs, seeds = {"h": h}, [d.get("dh")]
    if "pre" in leaves:
        outs["n"] = normed(h, leaves["pre"])
        seeds.append(d.get("dn"))
    got = {k: t.detach() for k, t in outs.items()}
    if case["train"]:
        grads = torch.autograd.grad(list(outs.values()), list(leaves.values()), [t.double() for t in seeds])
        got.update({"d" + k: g for k, g in zip(leaves, grads)})
    return got


def _exact_mlp(case, d):
    # the gradients from autograd
    train = bool(case["train"])
    x, wg, wu, wd = leaves = [d[k].double().requires_grad_(train) for k in ("x", "wg", "wu", "wd")]
    g = x @ wg
    a = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid}[case["act"]](g)
    y = (a * (x @ wu)) @ wd
    got = {"y": y.detach()}
    if train:
        got.update(zip(("dx", "dwg", "dwu", "dwd"), torch.autograd.grad(y, leaves, d["dy"].double())))
    return got


def _exact_scan(case, d):
    # token by token, forwards and then backwards
    x, z = d["x"].double(), d["z"].double()
    b, seq, c = x.shape
    f, k = torch.sigmoid(z), torch.sigmoid(-z)
    n = d["len"].long() if "len" in d else torch.full((b,), seq, device=GPU)
    live = (torch.arange(seq, device=GPU)[:, None] < n)[..., None].double()  # (seq, b, 1)
    first = d["state"].double() if "state" in d else torch.zeros((b, c), dtype=torch.float64, device=GPU)
    y, before, h = torch.zeros_like(x), torch.empty_like(x), first
    for t in range(seq):
        before[:, t] = h
        h = torch.lerp(h, f[:, t] * h + k[:, t] * x[:, t], live[t])
        y[:, t] = h * live[t]
    got = {"y": y, "last": h}
    if not case["train"]:
        return got
    dy = d["dy"].double()
    dh, back = torch.zeros_like(x), torch.zeros((b, c), dtype=torch.float64, device=GPU)
    for t in reversed(range(seq)):
        dh[:, t] = (dy[:, t] + back) * live[t]
        back = torch.lerp(back, f[:, t] * dh[:, t], live[t])
    got.update(dx=k * dh, dz=dh * (before - x) * f * k)
    if "state" in d:
        got["dstate"] = back
    return got


def exact(case, seed):
    d = _data(case, seed)
    return {"norm": _exact_norm, "mlp": _exact_mlp, "scan": _exact_scan}[case["kind"]](case, d)
