"""The serving operators on the GPU against plain 64-bit implementations: sizes, strides and masks where
they can go wrong. Bounds are derived in serving_ref.py."""

import math

import numpy as np
import pytest
import torch

import serving_ref as ref
from exactattention_b200 import serving

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(DEV)


# ---------------------------------------------------------------------------
# plan_step
# ---------------------------------------------------------------------------

def check_plan(ctx, new, ps, width, n_free, cap, head=0, depths=None, seed=0):
    rng = np.random.default_rng(seed)
    table = rng.integers(0, 1 << 20, size=(len(ctx), width)).astype(np.int32)
    free = (1 << 21) + rng.permutation(n_free).astype(np.int32)
    want = ref.plan_step(ctx, new, table, free, ps, cap, head, depths)
    td = i32(table)
    for _ in range(2):  # the same plan again gives the same pages
        p = serving.plan_step(i32(ctx), i32(new), td, i32(free), ps, cap, free_head=None if head is None else i32([head]),
                              depths=None if depths is None else i32(depths))
        got = dict(p._asdict(), page_table=td)
        for k, w in want.items():
            assert np.array_equal(got[k].cpu().numpy(), w), k


@pytest.mark.parametrize("batch,ps,ctx_max,new_max", [(1, 16, 50, 1), (3, 1, 9, 5), (64, 16, 3000, 1), (300, 24, 500, 40),
                                                      (257, 128, 1000, 700), (5000, 16, 100, 3)])
@pytest.mark.parametrize("pad", [0, 37])
def test_plan_step(batch, ps, ctx_max, new_max, pad):
    rng = np.random.default_rng(batch)
    ctx, new = rng.integers(0, ctx_max + 1, batch), rng.integers(0, new_max + 1, batch)
    width = -(-(ctx_max + new_max) // ps)
    total = int(new.sum())
    fresh = int((-(-(ctx + new) // ps) - -(-ctx // ps)).sum())
    depths = rng.integers(0, 9, total + pad) if pad else None
    check_plan(ctx, new, ps, width, fresh + 3, total + pad, head=2, depths=depths)


def test_plan_step_edges():
    check_plan([0], [0], 16, 1, 0, 0)                         # nothing at all
    check_plan([], [], 16, 4, 3, 8)                           # no sequence
    check_plan([16, 0, 31], [0, 0, 0], 16, 2, 0, 5)           # no token
    check_plan([16, 0, 31], [1, 40, 2], 16, 4, 2, 64)         # the free list runs out
    check_plan([16, 0, 31], [1, 40, 2], 16, 2, 9, 64)         # a table row is too short
    check_plan([5, 6], [30, 30], 16, 4, 9, 41)                # more tokens than room
    check_plan([-3, 7], [4, -9], 16, 4, 9, 8)                 # negative lengths count as zero
    check_plan([100000] * 7, [100000] * 7, 16, 13000, 43760, 700000)


def test_plan_step_table_rows_apart():
    table = torch.full((3, 9), -7, dtype=torch.int32, device=DEV)
    serving.plan_step(i32([1, 2, 3]), i32([40, 1, 9]), table[:, 2:6], i32(np.arange(20)), 16, 64)
    assert bool((table[:, :2] == -7).all()) and bool((table[:, 6:] == -7).all())
    assert table[0, 2:6].tolist() == [-7, 0, 1, -7]


# ---------------------------------------------------------------------------
# rope
# ---------------------------------------------------------------------------

def rope_inputs(n, hq, hk, d, rot, axes, dtype, seed=0, pos_max=1 << 15):
    g = torch.Generator(device=DEV).manual_seed(seed)
    qkv = torch.randn((n, hq + 2 * hk, d), generator=g, device=DEV).to(dtype)
    pos = torch.randint(0, pos_max, (axes, n), generator=g, device=DEV, dtype=torch.int32)
    freq = (1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).float().to(DEV)
    ax = torch.randint(0, axes, (rot // 2,), generator=g, device=DEV, dtype=torch.int32)
    return qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:], pos, freq, ax


def check_rope(got, x, pos, freq, ax, pairs, inverse):
    want, off = ref.rope(x, pos, freq, ax, pairs, inverse)
    ref.assert_within(got, want, off + ref.HALF_ULP[x.dtype] * want.abs() + ref.TINY[x.dtype])
    assert torch.equal(got[..., 2 * freq.numel():], x[..., 2 * freq.numel():])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("n,hq,hk,d,rot,axes", [(1, 16, 8, 128, 128, 1), (37, 7, 1, 96, 64, 3), (5, 3, 3, 80, 80, 2),
                                                (3, 2, 1, 70, 34, 4), (130, 1, 1, 64, 2, 1), (2, 2, 2, 6, 0, 1),
                                                (4099, 28, 4, 128, 96, 3)])
def test_rope(dtype, pairs, n, hq, hk, d, rot, axes):
    q, k, v, pos, freq, ax = rope_inputs(n, hq, hk, d, rot, axes, dtype, seed=n)
    for inverse in (False, True):
        qo, ko = serving.rope(q, k, pos, freq, axes=ax, pairs=pairs, inverse=inverse)
        check_rope(qo, q, pos, freq, ax, pairs, inverse)
        check_rope(ko, k, pos, freq, ax, pairs, inverse)


def test_rope_far_positions_one_tensor_and_layouts():
    q, k, v, pos, freq, ax = rope_inputs(33, 4, 2, 128, 128, 1, torch.float32, pos_max=2**31 - 1)
    qo, ko = serving.rope(q, None, pos[0], freq)
    assert ko is None
    check_rope(qo, q, pos, freq, None, "half", False)
    # heads before tokens, and rows off the 16-byte boundary
    x = torch.randn((4, 33, 130), device=DEV).to(torch.bfloat16)
    for y in (x[..., :128].transpose(0, 1), x[..., 1:129].transpose(0, 1), x[..., :50].transpose(0, 1)):
        check_rope(serving.rope(None, y, pos, freq[:24])[1], y, pos, freq[:24], None, "half", False)
    e = torch.empty((0, 4, 128), device=DEV)
    assert serving.rope(e, None, pos[:, :0], freq)[0].shape == e.shape


def test_rope_gradient_by_differences():
    q, _, _, pos, freq, ax = rope_inputs(6, 2, 1, 64, 48, 2, torch.float32, seed=3)
    dy = torch.randn_like(q)
    dx = serving.rope(dy, None, pos, freq, axes=ax, inverse=True)[0]
    rng = np.random.default_rng(0)
    for _ in range(40):
        at = tuple(int(rng.integers(0, s)) for s in q.shape)
        # the map is linear: its difference quotient has no truncation error; a step of 1 keeps rounding small
        lo, hi = q.clone(), q.clone()
        lo[at] -= 1
        hi[at] += 1
        f = lambda x: serving.rope(x, None, pos, freq, axes=ax)[0].double()  # noqa: E731
        diff = float(((f(hi) - f(lo)) * dy.double()).sum()) / (float(hi[at]) - float(lo[at]))
        # two changed outputs a side, each within 2^-19 of the pair's size, times |dy|
        bound = 2.0**-18 * (float(q[at[0], at[1]].abs().max()) + 1) * float(dy[at[0], at[1]].abs().max()) * 4
        assert abs(diff - float(dx[at])) <= bound


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["heads first", "rows first"])
@pytest.mark.parametrize("d,ps", [(128, 16), (80, 24), (36, 5)])
def test_rope_append(dtype, layout, d, ps):
    n, hq, hk, rot = 77, 6, 2, 32
    q, k, v, pos, freq, ax = rope_inputs(n, hq, hk, d, rot, 2, dtype, seed=5)
    pages = -(-n // ps) + 2
    shape = (pages, hk, ps, d) if layout == "heads first" else (pages, ps, hk, d)
    kc, vc = torch.full(shape, 3.0, dtype=dtype, device=DEV), torch.full(shape, 4.0, dtype=dtype, device=DEV)
    if layout != "heads first":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    slots = torch.randperm(pages * ps, device=DEV)[:n]
    slots[::9] = -1
    slots[1] = pages * ps  # outside the cache: skipped
    qo = serving.rope_append(q, k, v, pos, freq, slots, kc, vc, axes=ax)
    check_rope(qo, q, pos, freq, ax, "half", False)
    ok = (slots >= 0) & (slots < pages * ps)
    pg, off = slots[ok] // ps, slots[ok] % ps
    check_rope(kc[pg, :, off], k[ok], pos[:, ok], freq, ax, "half", False)
    assert torch.equal(vc[pg, :, off], v[ok])
    left = torch.ones((pages, ps), dtype=torch.bool, device=DEV)
    left[pg, off] = False
    assert bool((kc.transpose(1, 2)[left] == 3).all()) and bool((vc.transpose(1, 2)[left] == 4).all())


# ---------------------------------------------------------------------------
# tree_attention
# ---------------------------------------------------------------------------

def attention_inputs(ctx, new, hq, hk, d, ps, dtype, seed=0, layout="heads first", mask="tree", spread=1.0):
    rng = np.random.default_rng(seed)
    ctx, new = np.asarray(ctx), np.asarray(new)
    lens = ctx + new
    need = -(-lens // ps)
    pages = int(need.sum()) + 2
    perm = rng.permutation(pages).astype(np.int32)
    table = np.full((len(ctx), max(1, int(need.max(initial=0)))), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    g = torch.Generator(device=DEV).manual_seed(seed)
    shape = (pages, hk, ps, d) if layout == "heads first" else (pages, ps, hk, d)
    kc = (spread * torch.randn(shape, generator=g, device=DEV)).to(dtype)
    vc = torch.randn(shape, generator=g, device=DEV).to(dtype)
    if layout != "heads first":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    n = int(new.sum())
    q = torch.randn((n, hq + 3, d), generator=g, device=DEV).to(dtype)[:, 2:2 + hq]
    words = None
    if mask != "chain":
        w = max(1, -(-int(new.max(initial=1)) // 32))
        words = np.zeros((n, w), np.int32)
        r0 = 0
        for c in new:
            c = int(c)
            if mask == "tree":
                m = serving.tree_mask([int(rng.integers(-1, i)) if i else -1 for i in range(c)])
                words[r0:r0 + c, :m.shape[1]] = m
            else:  # any bits, bits past the step's tokens and empty rows among them
                words[r0:r0 + c] = rng.integers(-2**31, 2**31, (c, w)) * (rng.random((c, 1)) < 0.7)
            r0 += c
        words = torch.from_numpy(words).to(DEV)
    return dict(q=q, k_cache=kc, v_cache=vc, page_table=torch.from_numpy(table).to(DEV), seq_lens=i32(lens),
                q_start=i32(np.concatenate([[0], np.cumsum(new)])), alpha=math.log2(math.e) / math.sqrt(d),
                tree_mask=words)


def check_attention(x, **kw):
    out, lse = serving.tree_attention(**x, return_lse=True, **kw)
    o, ls, ob, lb = ref.tree_attention(x["q"], x["k_cache"], x["v_cache"], x["page_table"], x["seq_lens"], x["q_start"],
                                       x["alpha"], None if x["tree_mask"] is None else x["tree_mask"].cpu().numpy())
    ref.assert_within(out, o, ob)
    ref.assert_within(lse, ls, lb)
    again = serving.tree_attention(**x, return_lse=True, **kw)
    assert torch.equal(out.view(torch.int16), again[0].view(torch.int16)) and torch.equal(lse.view(torch.int32),
                                                                                            again[1].view(torch.int32))
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,ps", [(128, 16), (64, 24), (8, 1), (80, 5), (120, 128), (96, 256)])
@pytest.mark.parametrize("hq,hk", [(4, 4), (14, 2), (32, 1)])
def test_tree_attention_one_token(dtype, d, ps, hq, hk):
    check_attention(attention_inputs([0, 1, 15, 16, 63, 64, 65, 700], [1] * 8, hq, hk, d, ps, dtype, mask="chain"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mask", ["tree", "chain", "any"])
@pytest.mark.parametrize("ctx,new,hq,hk,d,ps", [
    ([300, 0, 17, 5], [7, 3, 0, 33], 4, 2, 128, 16),
    ([127, 128, 129], [1, 64, 65], 8, 1, 128, 32),
    ([1000], [130], 4, 2, 64, 24),
    ([511, 90], [20, 100], 7, 1, 112, 8),
    ([250, 0], [300, 257], 2, 1, 128, 64),
    ([0, 0, 0], [1, 31, 96], 16, 2, 40, 7),
])
def test_tree_attention(dtype, mask, ctx, new, hq, hk, d, ps):
    check_attention(attention_inputs(ctx, new, hq, hk, d, ps, dtype, mask=mask, seed=sum(ctx)))


@pytest.mark.parametrize("new", [1, 5, 40])
def test_tree_attention_many_sequences(new):
    rng = np.random.default_rng(new)
    ctx = rng.integers(0, 400, 90)
    check_attention(attention_inputs(ctx, rng.integers(0, new + 1, 90), 4, 2, 64, 16, torch.bfloat16))


def test_tree_attention_layouts_and_hints():
    for layout in ("heads first", "rows first"):
        x = attention_inputs([90, 200], [9, 40], 8, 2, 128, 16, torch.bfloat16, layout=layout)
        a = check_attention(x)
        for hint in (1, 40, 1000):  # a hint, no part of the result
            check_attention(x, max_new=hint)
        y = dict(x, q=x["q"].transpose(0, 1).contiguous().transpose(0, 1))
        assert torch.equal(serving.tree_attention(**y), a[0])


@pytest.mark.parametrize("spread", [0.0, 30.0])
def test_tree_attention_flat_and_sharp_scores(spread):
    check_attention(attention_inputs([400, 3], [3, 30], 8, 2, 128, 16, torch.bfloat16, spread=spread))


@pytest.mark.parametrize("step", [0.02, 0.6, 20.0, -0.6])
@pytest.mark.parametrize("new,hk", [(1, 4), (1, 1), (5, 4), (40, 4)])
def test_tree_attention_scores_that_grow_along_the_keys(new, hk, step):
    """A row's reference moves seldom, or with every key, or never again."""
    x = attention_inputs([500], [new], 8, hk, 64, 16, torch.float16)
    at = torch.zeros(x["k_cache"].shape[0] * 16, device=DEV)
    n = x["page_table"].shape[1] * 16
    slots = (x["page_table"][0].long()[:, None] * 16 + torch.arange(16, device=DEV)).reshape(-1)
    at[slots] = step * torch.arange(n, device=DEV, dtype=torch.float32)
    x["q"][..., 0] = 1.0
    x["k_cache"][..., 0] = (at.reshape(-1, 16)[:, None, :] / x["alpha"]).clamp(-6e4, 6e4).half()
    check_attention(x)


@pytest.mark.parametrize("new,hk", [(1, 4), (1, 1), (5, 4), (40, 4), (300, 4)])
def test_tree_attention_rows_do_not_depend_on_one_another(new, hk):
    x = attention_inputs([300], [new], 8, hk, 128, 16, torch.bfloat16)
    want = serving.tree_attention(**x)
    q = x["q"].clone()
    q[1:] *= 8
    q[:, 1::2] *= 8
    got = serving.tree_attention(**dict(x, q=q))
    assert torch.equal(got[0, ::2], want[0, ::2])


@pytest.mark.parametrize("new", [2, 30, 90])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tree_attention_values_that_are_not_seen(new, dtype):
    """NaN and infinities in drafted keys and values reach the rows that see them and no other; unread rows of a
    sequence's last page and missing pages reach nothing."""
    x = attention_inputs([70, 130], [new, 3], 4, 2, 128, 16, dtype, mask="chain")
    clean = serving.tree_attention(**x)
    kc, vc, tab = x["k_cache"].clone(), x["v_cache"].clone(), x["page_table"].cpu().numpy()
    used = np.zeros((kc.shape[0], 16), bool)
    for b, n in enumerate(x["seq_lens"].tolist()):
        used[tab[b, np.arange(n) // 16], np.arange(n) % 16] = True
    idle = torch.from_numpy(~used).to(DEV)
    kc.transpose(1, 2)[idle] = math.nan
    vc.transpose(1, 2)[idle] = math.inf
    last = 70 + new - 1  # seen by the last token of sequence 0 alone
    pg, off = tab[0, last // 16], last % 16
    kc[pg, 0, off] = math.nan
    vc[pg, 1, off, 5], vc[pg, 1, off, 6], vc[pg, 1, off, 7] = math.inf, -math.inf, math.nan
    y = dict(x, k_cache=kc, v_cache=vc)
    out, _ = check_attention(y)
    keep = torch.ones(new + 3, dtype=torch.bool, device=DEV)
    keep[new - 1] = False
    assert torch.equal(out[keep], clean[keep])
    # a page that is no page of the cache
    y["page_table"] = x["page_table"].clone()
    y["page_table"][1, 1], y["page_table"][1, 3] = -1, 1 << 30
    check_attention(y)


def test_tree_attention_infinite_values_in_the_context():
    x = attention_inputs([200], [4], 4, 1, 64, 16, torch.bfloat16)
    x["v_cache"][x["page_table"][0, 2].item(), 0, 3, :2] = torch.tensor([math.inf, -math.inf], device=DEV).bfloat16()
    check_attention(x)
    y = attention_inputs([200], [40], 4, 1, 64, 16, torch.bfloat16)
    y["v_cache"][y["page_table"][0, 2].item(), 0, 3, :2] = torch.tensor([math.inf, -math.inf], device=DEV).bfloat16()
    check_attention(y)


@pytest.mark.parametrize("alpha", [-0.2, 0.0, 1e-9])
@pytest.mark.parametrize("new", [1, 30])
def test_tree_attention_any_alpha(alpha, new):
    x = attention_inputs([150, 0], [new, 3], 8, 2, 128, 16, torch.bfloat16)
    check_attention(dict(x, alpha=alpha))


def test_tree_attention_more_sequences_than_the_tensor_core_kernel_takes():
    x = attention_inputs([3] * 6100, [1] * 6099 + [40], 2, 1, 64, 16, torch.bfloat16, mask="chain")
    check_attention(x, max_new=40)


def test_tree_attention_out_and_unused_rows():
    x = attention_inputs([90, 20], [9, 40], 8, 2, 128, 16, torch.bfloat16)
    want = serving.tree_attention(**x)
    q = torch.cat([x["q"], x["q"][:7]])  # rows past the step's tokens, as a padded step has them
    mask = torch.cat([x["tree_mask"], x["tree_mask"][:7]])
    out = torch.full(q.shape, 5.0, dtype=q.dtype, device=DEV)
    assert serving.tree_attention(**dict(x, q=q, tree_mask=mask), out=out) is out
    assert torch.equal(out[:49], want) and bool((out[49:] == 5).all())


def test_tree_attention_cache_past_32_bit_offsets():
    hk, ps, d = 2, 64, 128
    pages = 2**31 // (hk * ps * d) + 60
    for new in (1, 50):
        x = attention_inputs([300], [new], 4, hk, d, ps, torch.bfloat16)
        kc = torch.empty((pages, hk, ps, d), dtype=torch.bfloat16, device=DEV)
        vc = torch.empty_like(kc)
        n = x["page_table"].shape[1]
        far = torch.arange(pages - n, pages, device=DEV)
        kc[far], vc[far] = x["k_cache"][x["page_table"][0].long()], x["v_cache"][x["page_table"][0].long()]
        y = dict(x, k_cache=kc, v_cache=vc, page_table=far.int()[None].contiguous())
        assert torch.equal(serving.tree_attention(**x), serving.tree_attention(**y))
        del kc, vc
        torch.cuda.empty_cache()


def test_tree_attention_long_context():
    for new in (1, 24):
        check_attention(attention_inputs([200003], [new], 8, 2, 64, 16, torch.float16, mask="chain"))


def test_tree_attention_another_stream_and_graph():
    x = attention_inputs([90, 300], [5, 40], 8, 2, 128, 16, torch.bfloat16)
    want = serving.tree_attention(**x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = serving.tree_attention(**x)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = serving.tree_attention(**x)
    x["q"].mul_(-1)
    graph.replay()
    assert torch.equal(out, serving.tree_attention(**x)) and not torch.equal(out, want)


# ---------------------------------------------------------------------------
# process_logits
# ---------------------------------------------------------------------------

def logits_inputs(rows, vocab, batch, dtype, seed=0, hist=40, nb=5, grammar=True, tree=None, pad=0):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.standard_normal((rows, vocab + pad)) * 4).to(dtype)[:, :vocab]
    row_seq = np.sort(rng.integers(0, batch, rows)).astype(np.int32)
    q_start = np.searchsorted(row_seq, np.arange(batch + 1)).astype(np.int32)
    hl = rng.integers(0, hist + 1, batch).astype(np.int32)
    kw = dict(row_seq=row_seq, history=rng.integers(-2, vocab + 2, (batch, hist)).astype(np.int32), history_lens=hl,
              prompt_lens=(hl // 3).astype(np.int32), repetition=rng.choice([1.0, 1.25, 0.7], batch).astype(np.float32),
              frequency=rng.choice([0.0, 0.3], batch).astype(np.float32),
              presence=rng.choice([0.0, 0.5], batch).astype(np.float32),
              bias_ids=rng.integers(-1, vocab, (batch, nb)).astype(np.int32),
              bias_values=rng.standard_normal((batch, nb)).astype(np.float32))
    if grammar:
        kw["allowed_bits"] = rng.integers(-2**31, 2**31, (3, (vocab + 31) // 32)).astype(np.int32)
        kw["allowed_bits"][1] = 0  # a state that allows nothing
        kw["mask_rows"] = rng.integers(-1, 3, rows).astype(np.int32)
    if tree:
        kw["draft_tokens"] = rng.integers(0, vocab, rows).astype(np.int32)
        kw["q_start"] = q_start
        if tree == "tree":
            kw["tree_mask"] = rng.integers(-2**31, 2**31, (rows, 2)).astype(np.int32)
    return x, kw


def check_logits(x, kw, **more):
    names = ("history", "history_lens", "prompt_lens", "repetition", "frequency", "presence", "bias_ids", "bias_values",
             "allowed_bits", "mask_rows", "draft_tokens", "q_start", "tree_mask")
    want, bound = ref.process_logits(x, kw.get("row_seq"), *(kw.get(n) for n in names))
    dk = {k: torch.from_numpy(v).to(DEV) for k, v in kw.items()}
    base = torch.zeros((x.shape[0], x.stride(0)), dtype=x.dtype, device=DEV)
    xd = base[:, :x.shape[1]]
    xd.copy_(x)
    got = serving.process_logits(xd, **dk, **more)
    ref.assert_within(got, want, bound)
    assert torch.equal(xd.cpu(), x)
    assert serving.process_logits(xd, **dk, out=xd) is xd  # in place
    assert torch.equal(xd.view(torch.uint8) if xd.is_contiguous() else xd, got.view(torch.uint8) if xd.is_contiguous() else got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,batch,pad", [(1, 1, 1, 0), (3, 37, 2, 0), (5, 1000, 3, 8), (9, 4099, 4, 0), (2, 33000, 2, 3),
                                                  (7, 131072, 2, 0)])
@pytest.mark.parametrize("tree", [None, "chain", "tree"])
def test_process_logits(dtype, rows, vocab, batch, pad, tree):
    check_logits(*logits_inputs(rows, vocab, batch, dtype, seed=vocab, tree=tree, pad=pad))


def test_process_logits_parts_and_rows_without_a_sequence():
    x, kw = logits_inputs(6, 5003, 6, torch.float32, tree=None)
    kw["row_seq"] = np.array([-1, 5, 6, 0, 0, 1 << 30], np.int32)
    check_logits(x, kw)
    for names in (("history", "history_lens", "frequency"), ("bias_ids", "bias_values"), ("allowed_bits", "mask_rows"), ("presence",)):
        check_logits(x, {k: kw[k] for k in names})
    assert torch.equal(serving.process_logits(x.to(DEV)).cpu(), x)
    e = serving.process_logits(x[:0].to(DEV))
    assert e.shape == (0, 5003)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,pad", [(650, 37, 0), (611, 1000, 8), (700, 4099, 0), (90, 131075, 5)])
@pytest.mark.parametrize("tree", [None, "chain", "tree"])
def test_process_logits_many_rows(dtype, rows, vocab, pad, tree):
    """More blocks than the kernel for few rows is taken for."""
    check_logits(*logits_inputs(rows, vocab, 11, dtype, seed=vocab, tree=tree, pad=pad))


@pytest.mark.parametrize("parts", [("history", "history_lens", "frequency"), ("bias_ids", "bias_values"),
                                   ("allowed_bits", "mask_rows"), ("history", "history_lens", "presence", "allowed_bits", "mask_rows")])
def test_process_logits_many_rows_parts(parts):
    x, kw = logits_inputs(660, 2003, 660, torch.float32)
    kw["row_seq"][::7] = -1
    kw["row_seq"][3] = 1 << 30
    check_logits(x, {k: kw[k] for k in parts + ("row_seq",)})


@pytest.mark.parametrize("rows,vocab,hist", [(70, 131075, 9000), (600, 601, 1500), (50, 200000, 13000)])
def test_process_logits_many_rows_long_histories(rows, vocab, hist):
    """Lists that fit the table, that are many times the vocabulary, and that take several passes."""
    x, kw = logits_inputs(rows, vocab, 5, torch.bfloat16, hist=hist, nb=400)
    check_logits(x, kw)
    x, kw = logits_inputs(rows, vocab, 5, torch.bfloat16, hist=hist, nb=40, grammar=False)
    kw["bias_ids"][:] = kw["bias_ids"] % 7  # every id several times
    check_logits(x, kw)


def test_process_logits_same_bias_twice_adds_in_order():
    x, kw = logits_inputs(2, 300, 2, torch.float32, nb=40, grammar=False)
    kw["bias_ids"][:] = kw["bias_ids"] % 7  # every id several times
    check_logits(x, kw)


def test_process_logits_long_history_and_many_biases():
    x, kw = logits_inputs(4, 9000, 2, torch.bfloat16, hist=30011, nb=2000, tree="chain")
    check_logits(x, kw)


def test_process_logits_special_values():
    x, kw = logits_inputs(4, 700, 4, torch.float32, grammar=True)
    x[0, :50], x[1, :50], x[2, :50], x[3, 100:150] = math.nan, math.inf, -math.inf, -3.4e38
    kw.pop("bias_ids"), kw.pop("bias_values")
    dk = {k: torch.from_numpy(v).to(DEV) for k, v in kw.items()}
    got = serving.process_logits(x.to(DEV), **dk).cpu()
    want, bound = ref.process_logits(x, kw["row_seq"], kw["history"], kw["history_lens"], kw["prompt_lens"], kw["repetition"],
                                     kw["frequency"], kw["presence"], None, None, kw["allowed_bits"], kw["mask_rows"], None,
                                     None, None)
    want = torch.where(want.abs() > 3.4028235e38, torch.copysign(torch.tensor(math.inf).double(), want), want)
    ref.assert_within(got, want, bound)
