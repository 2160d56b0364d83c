"""examples/draft_step.py: the serving operators together on one cache, against the certified attention (B200 only)."""

import os
import subprocess
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
sys.path.insert(0, os.path.join(ROOT, "examples"))


@pytest.mark.parametrize("kw", [dict(), dict(nodes=(1, 1, 1), seed=1), dict(contexts=(0, 15, 16), nodes=(70, 3, 9), page=24, seed=2),
                                dict(q_heads=8, kv_heads=1, d=64, contexts=(300,), nodes=(33,), seed=3)])
def test_step_agrees_with_the_certified_attention(kw):
    import draft_step

    r = draft_step.run(**kw)
    assert int(r["plan"].status) == 0 and int(r["flags"].max()) == 0
    # both are roundings of the same sums: the certified one of the exact value, the draft's of one whose weights carry
    # a 16-bit rounding each (2^-8 of the mean magnitude, which a value of N(0, 1) data stays below 6 of)
    off = (r["drafted"].float() - r["certified"].float()).abs()
    bound = 2.0**-7 * r["certified"].float().abs() + 6 * 2.0**-8
    assert bool((off <= bound).all())
    assert bool(torch.isfinite(r["lse"]).all())
    assert bool(torch.isfinite(r["scores"].gather(1, r["chosen"][:, None])).all())


def test_example_runs_as_a_program():
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "draft_step.py")], capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    assert "flags [0]" in out.stdout


def test_steps_in_a_graph():
    """The whole chain captured once and replayed with new lengths: nothing in it depends on the host."""
    from exactattention_b200 import serving

    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(4)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    B, hq, hk, d, ps, cap = 3, 4, 2, 64, 16, 24
    ctx, new = i32([5, 40, 0]), i32([3, 1, 8])
    pages = torch.arange(B * 8, dtype=torch.int32, device=dev).reshape(B, 8)
    table = pages.clone()
    free = torch.arange(100, 140, dtype=torch.int32, device=dev)
    kc = torch.randn((160, hk, ps, d), generator=g, device=dev, dtype=torch.bfloat16)
    vc = torch.randn((160, hk, ps, d), generator=g, device=dev, dtype=torch.bfloat16)
    qkv = torch.randn((cap, hq + 2 * hk, d), generator=g, device=dev, dtype=torch.bfloat16)
    freq = (1e4 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)).float().to(dev)
    logits = torch.randn((cap, 999), generator=g, device=dev)
    hist, lens = torch.randint(0, 999, (B, 30), generator=g, device=dev, dtype=torch.int32), i32([30, 4, 0])
    pen = torch.full((B,), 1.2, device=dev)

    def step():
        p = serving.plan_step(ctx, new, table, free, ps, cap)
        q = serving.rope_append(qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:], p.positions, freq, p.slot_map, kc, vc)
        o = serving.tree_attention(q, kc, vc, table, p.seq_lens, p.q_start, 0.18, max_new=8)
        return p.q_start, o, serving.process_logits(logits, p.token_seq, history=hist, history_lens=lens, repetition=pen)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for c, n in (([5, 40, 0], [3, 1, 8]), ([100, 0, 17], [1, 0, 20]), ([0, 1, 2], [8, 8, 8])):
        ctx.copy_(i32(c)), new.copy_(i32(n)), table.copy_(pages)  # every case starts from the same pages: none is shared
        graph.replay()
        torch.cuda.synchronize()
        res = [x.clone() for x in got]
        table.copy_(pages)
        want = step()
        t = int(np.sum(n))
        assert torch.equal(res[0], want[0]) and torch.equal(res[1][:t], want[1][:t]) and torch.equal(res[2], want[2])
