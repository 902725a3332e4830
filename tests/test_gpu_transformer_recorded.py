"""Recorded training steps of attention on fp16 parts: two graphs of different
sizes, which share the engine's workspace, replayed in turn with eager work
between, train exactly as eager steps do."""
import numpy as np
import pytest
import torch  # noqa: F401  (ahead of the engine, which then shares its HIP runtime)

from tests import test_gpu_transformer as base
from tests.helpers import rng

pytestmark = pytest.mark.gpu

SIZES = [(2, 1024, 4, 64, 9), (3, 700, 4, 32, 5), (2, 40, 4, 16, 7)]   # batch, tokens, heads, dims, classes


def test_two_graphs_replayed_in_turn(eng):
    r = rng(500)
    runs = []
    for B, S, H, D, classes in SIZES:
        P0, _, _ = base.block_data(r, B, S, H * D, classes)
        data = [(r.standard_normal((B * S, H * D)).astype(np.float32), r.integers(0, classes, B * S).astype(np.float32))
                for _ in range(4)]
        table = eng.rotary_table(S, D)

        def fresh(P0=P0):
            P = {n: base.dev(eng, a, True) for n, a in P0.items()}
            return P, eng.Muon(list(P.values()), lr=0.01)
        P, opt = fresh()
        losses = []
        for x, y in data:
            opt.zero_grad()
            loss = eng.softmax_ce(base.block_forward(eng, P, base.dev(eng, x), table, B, S, H, D), base.dev(eng, y))
            loss.backward()
            opt.step(clip=1.0)
            losses.append(float(loss.sync()[0]))
            eng.end_batch()
        want = {n: t.sync().copy() for n, t in P.items()}
        runs.append(dict(dims=(B, S, H, D), data=data, table=table, fresh=fresh, losses=losses, want=want))
    for run in runs:
        run["P"], run["opt"] = run["fresh"]()
        run["graph"] = eng.ComputeGraph()
        P, table, dims = run["P"], run["table"], run["dims"]
        run["graph"].trace(lambda x, P=P, table=table, dims=dims: base.block_forward(eng, P, x, table, *dims), run["opt"],
                           *run["data"][0], list(P.values()), clip=1.0)
    other = eng.Muon([base.dev(eng, np.ones((900, 800)), True)], lr=0.1)
    for i in range(1, 4):
        for run in runs:
            run["graph"].replay(*run["data"][i])
            # eager work over the same workspace between the replays, larger than any before it at last
            other.params[0].grad = base.dev(eng, r.standard_normal((900, 800)))
            other.step()
            q = base.dev(eng, r.standard_normal((1, 1100 + 600 * i, 4, 64)), True)
            eng.attention(q, q, q, causal=True).backward(q)
            assert run["graph"].read_loss() == run["losses"][i], (run["dims"], i)
            eng.end_batch()
    for run in runs:
        assert run["opt"].t == 4
        for n, t in run["P"].items():
            assert np.array_equal(t.sync(), run["want"][n]), n
        run["graph"].release()
    eng.end_batch()
