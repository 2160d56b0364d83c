"""The serving operators on the GPU where they are easily wrong, beyond test_gpu_serving.py: each test holds a case
that one of the kernels or its host side once got wrong."""

import ctypes
import fractions
import math
import threading

import numpy as np
import pytest
import torch

import serving_ref as ref
from exactattention_b200 import _lib, serving
from test_gpu_serving import DEV, attention_inputs, check_attention, check_rope, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 40])
def test_tree_attention_out_off_a_16_byte_boundary_is_refused(new):
    """A contiguous slice of a larger buffer. Refused on the host: nothing is launched."""
    x = attention_inputs([90], [new], 8, 2, 128, 16, torch.bfloat16)
    want = serving.tree_attention(**x)
    buf = torch.zeros(want.numel() + 8, dtype=want.dtype, device=DEV)
    for off in (1, 2, 4, 7):
        with pytest.raises(ValueError, match="16-byte"):
            serving.tree_attention(**x, out=buf[off:off + want.numel()].view(want.shape))
    out = buf[8:].view(want.shape)
    assert serving.tree_attention(**x, out=out) is out and torch.equal(out, want)
    assert not bool(buf[:8].any())


@pytest.mark.parametrize("tail", [-26.0, -30.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("seqs,new,hq,hk", [(24, 1, 32, 16), (12, 24, 32, 16), (4, 130, 64, 16)])
def test_tree_attention_long_tail_behind_dominant_keys(dtype, seqs, new, hq, hk, tail):
    """A few keys with values of 0 dominate the sum, and thousands some 2^26 below them make the output: fp16 holds
    no weight below 2^-25 of its reference. The dominant keys lie where every warp, and every slot of the tensor-core
    kernel, has one; there are enough items for most to lie in one share."""
    d, ctx = 32, 8192
    x = attention_inputs([ctx] * seqs, [new] * seqs, hq, hk, d, 16, dtype, mask="chain")
    g = torch.Generator(device=DEV).manual_seed(1)
    kc, vc = x["k_cache"], x["v_cache"]
    x["q"].zero_()
    x["q"][..., 0] = 1
    kc.zero_()
    kc[..., 0] = ((tail + 4 * torch.rand(kc.shape[:3], generator=g, device=DEV) - 2) / x["alpha"]).to(dtype)
    vc.copy_(64 * (1 + 0.25 * torch.randn(vc.shape, generator=g, device=DEV)))
    for key in (0, 16, 32, 48, 128):
        page = x["page_table"][:, key // 16].long()
        kc[page, :, key % 16], vc[page, :, key % 16] = 0, 0
    check_attention(x, max_new=new)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("size,step", [(2.0**24, 4.0), (2.0**24, 16.0), (2.0**26, 8.0), (2.0**26, 16.0), (2.0**29, 64.0)])
def test_tree_attention_huge_scores_that_grow(dtype, new, size, step):
    """Scores of a size at which 32-bit numbers are as far apart as the distance at which a row's reference moves: no
    weight may overflow its type. Every score is size + step * (0 .. 3), exact in 32 bits, so only the weights' and the
    output's roundings are left: 2^-14 for exp2 and the sums, half a unit of the type for each of the two."""
    x = attention_inputs([300], [new], 4, 2, 16, 16, dtype, mask="chain")
    q, kc, vc = x["q"], x["k_cache"], x["v_cache"]
    q.zero_(), kc.zero_()
    q[..., 0], q[..., 1] = 2.0**12, 1.0
    n = 300 + new
    key = torch.arange(n, device=DEV)
    page, row = x["page_table"][0].long()[key // 16], key % 16
    level = (4 * key // n).double()  # grows along the keys
    kc[page, :, row, 0] = size / 2.0**14
    kc[page, :, row, 1] = (step / 4 * level).to(dtype)[:, None]
    out, lse = serving.tree_attention(**dict(x, alpha=4.0), return_lse=True)
    v = vc[page, :, row].double()  # (key, kv head, d)
    w = torch.exp2(step * (level - 3))[None] * (key[None] <= 300 + torch.arange(new, device=DEV)[:, None])
    o, mag = (torch.einsum("tn,nhd->thd", w, y).repeat_interleave(2, 1) / w.sum(1)[:, None, None] for y in (v, v.abs()))
    u = ref.HALF_ULP[dtype]
    ref.assert_within(out, o, u * o.abs() + (u + 2.0**-14) * mag + ref.TINY[dtype])
    assert bool(((lse - size).abs() <= 3 * step + 16 + size * 2.0**-23).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("key", [0, 130, 199])
@pytest.mark.parametrize("new,hq,ps", [(4, 4, 16), (40, 4, 16), (40, 4, 24), (300, 4, 16), (40, 40, 16)])
def test_tree_attention_infinite_values_beside_the_drafted_keys(dtype, key, new, hq, ps):
    """A context key in the tile where the drafted keys begin (128 .. 255): every row sees its infinities and NaN."""
    x = attention_inputs([200], [new], hq, 1, 64, ps, dtype)
    v = x["v_cache"][x["page_table"][0, key // ps].item(), 0, key % ps]
    v[:3] = torch.tensor([math.inf, -math.inf, math.nan], device=DEV).to(dtype)
    check_attention(x)


def reference(x, table=None):
    return ref.tree_attention(x["q"], x["k_cache"], x["v_cache"], x["page_table"] if table is None else table, x["seq_lens"],
                              x["q_start"], x["alpha"], None if x["tree_mask"] is None else x["tree_mask"].cpu().numpy())


@pytest.mark.parametrize("new,hq", [(6, 2), (40, 4), (300, 4)])
@pytest.mark.parametrize("mask", ["chain", "tree"])
@pytest.mark.parametrize("ps", [16, 24])
def test_tree_attention_sequence_longer_than_its_table(new, hq, mask, ps):
    """A step that plan_step reports as PLAN_TABLE_FULL: keys past the table's columns are not seen, and which of the others
    are the step's own still follows from the sequence's length."""
    x = attention_inputs([10 * ps - new // 2, 20], [new, 3], hq, 1, 64, ps, torch.bfloat16, mask=mask)
    wide = x["page_table"].clone()
    wide[0, 10:] = -1
    o, ls, ob, lb = reference(x, wide)
    out, lse = serving.tree_attention(**dict(x, page_table=wide[:, :10].contiguous()), return_lse=True)
    ref.assert_within(out, o, ob)
    ref.assert_within(lse, ls, lb)


@pytest.mark.parametrize("new,hq", [(6, 2), (40, 4), (300, 4)])
@pytest.mark.parametrize("mask", ["chain", "tree"])
def test_tree_attention_more_tokens_than_rows(new, hq, mask):
    """A step that plan_step reports as PLAN_TOO_MANY: the last sequence has tokens without a row of q."""
    x = attention_inputs([50, 90], [3, new], hq, 1, 64, 16, torch.bfloat16, mask=mask)
    o, ls, ob, lb = reference(x)
    n = x["q"].shape[0] - 2
    y = dict(x, q=x["q"][:n], tree_mask=None if x["tree_mask"] is None else x["tree_mask"][:n].contiguous())
    out, lse = serving.tree_attention(**y, return_lse=True)
    ref.assert_within(out, o[:n], ob[:n])
    ref.assert_within(lse, ls[:n], lb[:n])


def test_plan_step_of_two_sizes_from_two_threads():
    """Large and small batches planned at the same time by two host threads through the C entry (the Python binding holds
    the interpreter's lock): neither call may take the other's shared memory away."""
    lib = _lib.load()
    failed = []

    def work(batch):
        zeros = torch.zeros(batch, dtype=torch.int32, device=DEV)
        outs = [torch.zeros(batch + 1, dtype=torch.int32, device=DEV) for _ in range(5)]
        slots = torch.zeros(8, dtype=torch.int64, device=DEV)
        a = _lib.PlanStepArgs()
        a.context_lens = a.new_lens = zeros.data_ptr()
        a.slot_map, a.positions, a.token_seq = slots.data_ptr(), outs[0].data_ptr(), outs[1].data_ptr()
        a.q_start, a.seq_lens = outs[2].data_ptr(), outs[3].data_ptr()
        a.next_free_head, a.status = outs[4].data_ptr(), outs[4].data_ptr() + 4
        a.batch, a.page_size, a.max_tokens = batch, 16, 8
        for _ in range(3000):
            rc = lib.ea_plan_step_cuda(ctypes.byref(a), None)
            if rc:
                failed.append((batch, rc, lib.ea_serving_last_error()))
        torch.cuda.synchronize()

    threads = [threading.Thread(target=work, args=(b,)) for b in (16384, 6000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, (len(failed), failed[0])


def test_plan_step_page_counts_past_32_bits():
    """Pages of one row: a context of 2^31 - 1 and one token need 2^31 pages, which no table has."""
    table = torch.full((2, 3), -1, dtype=torch.int32, device=DEV)
    big = 2**31 - 1
    p = serving.plan_step(i32([big, 0]), i32([1, 2]), table, i32(np.arange(8)), 1, 8)
    assert int(p.status) == serving.PLAN_TABLE_FULL
    assert p.slot_map.tolist() == [-1, 1, 2, -1, -1, -1, -1, -1] and p.token_seq.tolist() == [0, 1, 1, -1, -1, -1, -1, -1]
    assert p.q_start.tolist() == [0, 1, 3] and p.seq_lens.tolist() == [big, 2] and int(p.free_head) == 3
    assert table.tolist() == [[-1, -1, -1], [1, 2, -1]]


@pytest.mark.parametrize("rows", [3, 1500])
def test_process_logits_masks_alone_for_late_sequences(rows):
    """Masks need no tensor of the sequences, so nothing says how many there are: the rows of a few late sequences of a
    server (numbers above the row count) are masked like any others."""
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn((rows, 70), generator=g, device=DEV)
    seqs = torch.arange(rows, device=DEV, dtype=torch.int32) * 7 + 5
    seqs[1] = -1
    states = torch.arange(rows, device=DEV, dtype=torch.int32) % 4
    bits = torch.randint(-2**31, 2**31, (4, 3), generator=g, device=DEV).to(torch.int32)
    bits[0] = 0
    at = torch.arange(70, device=DEV)
    allowed = ((bits[:, at // 32] >> (at % 32)) & 1).bool()[states.long()]
    allowed[1] = True
    want = x.masked_fill(~allowed, -math.inf)
    assert torch.equal(serving.process_logits(x, seqs, allowed_bits=bits, mask_rows=states), want)


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("top", [0.5, 50.0, 1000.0, 3e4])
def test_rope_large_angles(top, inverse):
    """Positions below 2^24 with frequencies above 1, whose products lie far past 2^24, and the ends of the positions'
    range. Their products are exact in binary64, up to the last two bits of the largest ones."""
    g = torch.Generator(device=DEV).manual_seed(0)
    n, d = 200, 64
    q = torch.randn((n, 2, d), generator=g, device=DEV)
    pos = torch.randint(0, 2**24, (n,), generator=g, device=DEV, dtype=torch.int32)
    freq = top * torch.rand(d // 2, generator=g, device=DEV) + top / 50
    if top < 1:
        pos[:4] = torch.tensor([-2**31, 2**31 - 1, -2**24, 2**24], device=DEV)
    check_rope(serving.rope(q, None, pos, freq, inverse=inverse)[0], q, pos, freq, None, "half", inverse)


def test_rope_huge_angles():
    """Angles up to 2^71, reduced for the comparison with 1 / (2 pi) to 192 bits."""
    inv_2pi = fractions.Fraction(0x28BE60DB9391054A7F09D5F47D4D377036D8A5664F10E410, 2**192)  # 1 / (2 pi) to 2^-192
    pos = [1, 3, 12345677, 2**31 - 1, -2**31, 2**24 + 1]
    f0 = torch.tensor([1.0, 1.25, 0.7853982, 0.001], dtype=torch.float32)
    q = torch.zeros((len(pos), 1, 8), device=DEV)
    q[..., :4] = 1  # the result is (cos, sin)
    got = serving.rope(q, None, i32(pos), (2.0**40 * f0).to(DEV))[0].cpu().double()
    for t, p in enumerate(pos):
        for i, f in enumerate(f0.tolist()):
            turns = p * fractions.Fraction(f) * 2**40 * inv_2pi
            a = 2 * math.pi * float(turns - round(turns))
            assert abs(float(got[t, 0, i]) - math.cos(a)) <= 2.0**-20 and abs(float(got[t, 0, 4 + i]) - math.sin(a)) <= 2.0**-20


@pytest.mark.parametrize("new,pages", [(1, 1), (1, 7), (40, 1), (40, 9)])
def test_tree_attention_strides_of_extents_of_one(new, pages):
    """A stride over an extent of one says nothing: one token, one kv head or one page of a buffer of odd rows."""
    ps = 64 if pages == 1 else 16
    x = attention_inputs([min(ps * pages, 130) - new - 3], [new], 4, 1, 64, ps, torch.bfloat16)
    if pages == 1:
        page = int(x["page_table"][0, 0])
        x.update(k_cache=x["k_cache"][page:page + 1], v_cache=x["v_cache"][page:page + 1], page_table=i32([[0]]))
    want = serving.tree_attention(**x)

    def odd(t):
        strides = [n if size > 1 else 7777777 for n, size in zip(t.stride(), t.shape)]
        return torch.as_strided(t, t.shape, strides, t.storage_offset())

    y = dict(x, q=odd(x["q"]), k_cache=odd(x["k_cache"]), v_cache=odd(x["v_cache"]))
    assert any(s % 8 for s in y["k_cache"].stride())
    assert torch.equal(serving.tree_attention(**y), want)


def test_rope_in_a_training_step():
    """rope and its inverse as the two directions of an autograd function; called bare, it refuses what requires grad."""
    g = torch.Generator(device=DEV).manual_seed(0)
    q = torch.randn((9, 4, 64), generator=g, device=DEV, requires_grad=True)
    dy = torch.randn((9, 4, 64), generator=g, device=DEV)
    pos, freq = i32(np.arange(9) * 100), 1e4 ** (-torch.arange(0, 64, 2, device=DEV) / 64)

    class Rope(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return serving.rope(x, None, pos, freq)[0]

        @staticmethod
        def backward(ctx, d):
            return serving.rope(d, None, pos, freq, inverse=True)[0]

    with pytest.raises(ValueError, match="requires grad"):
        serving.rope(q, None, pos, freq)
    Rope.apply(q).backward(dy)
    check_rope(q.grad, dy, pos, freq, None, "half", True)


@pytest.mark.parametrize("new,hq,ps", [(40, 4, 16), (40, 4, 24), (300, 4, 16), (300, 4, 24)])
def test_tree_attention_waits_that_run_out(new, hq, ps):
    """With the hook the tensor-core kernel's queries are never announced, so its products, copies and softmax wait in vain
    for 20 ms: the rows come back as NaN, what was under way has landed, and the next call is right."""
    x = attention_inputs([500, 90, 3000], [new, 3, 20], hq, 1, 64, ps, torch.bfloat16)
    want = serving.tree_attention(**x, return_lse=True)
    try:
        _lib.set_test_hooks(0, 0, 1)
        out, lse = serving.tree_attention(**x, return_lse=True)
        torch.cuda.synchronize()
    finally:
        _lib.set_test_hooks(0, 0, 0)
    assert bool(torch.isnan(out).all()) and bool(torch.isnan(lse).all())
    for a, b in zip(serving.tree_attention(**x, return_lse=True), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq", [2, 7, 8, 16])
def test_tree_attention_few_rows_carry_weights_as_pairs(dtype, hq):
    """Up to 16 rows a kv head take a weight as two 16-bit numbers, 2^-17 off in all. Pairs of keys with almost the same score and
    opposite values leave next to nothing but the weights' errors: a single 16-bit rounding is 4 to 20 times the bound."""
    n, d = 80, 8
    x = attention_inputs([n - 1] * 6, [1] * 6, hq, 1, d, 16, dtype, mask="chain")
    g = torch.Generator(device=DEV).manual_seed(hq)
    low = torch.randn((6, n // 2), generator=g, device=DEV).to(dtype)
    up = (low.float() * (1 + 2.0**-7 if dtype == torch.bfloat16 else 1 + 2.0**-10)).to(dtype)
    score = torch.stack([low, up], -1).reshape(6, n)
    x["q"].zero_(), x["k_cache"].zero_()
    x["q"][..., 0] = 1
    for b in range(6):
        key = torch.arange(n, device=DEV)
        page = x["page_table"][b].long()[key // 16]
        x["k_cache"][page, 0, key % 16, 0] = score[b]
        x["v_cache"][page, 0, key % 16] = (1.0 - 2.0 * (key % 2))[:, None].to(dtype)
    out = serving.tree_attention(**dict(x, alpha=1.0), max_new=1).double()
    w, sign = torch.exp2(score.double()), 1.0 - 2.0 * (torch.arange(n, device=DEV) % 2)
    o = (w * sign).sum(1) / w.sum(1)
    # scores of d terms in 32 bits, a weight's pair, exp2 and the sums of at most 16 steps
    rel = 2 * math.log(2) * d * 2.0**-23 * score.double().abs().amax(1) + 2.0**-17 + 2.0**-18
    bound = ref.HALF_ULP[dtype] * o.abs() + rel + ref.TINY[dtype]
    ref.assert_within(out, o[:, None, None].expand_as(out), bound[:, None, None].expand_as(out))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,limit", [(1, 1.05), (8, 1.05), (40, 1.6), (300, 1.6)])
def test_tree_attention_error_over_a_long_context(dtype, new, limit):
    """The root mean square error against the output's own rounding: the same for up to 16 rows a kv head, whose weights'
    errors do not show; up to 2^(1/2) times it (and a tenth for the sample) on the tensor cores, where a weight's
    rounding is one of the same size and sign."""
    x = attention_inputs([3000], [new], 8, 4, 128, 16, dtype)
    o, _, _, _ = reference(x)
    out = serving.tree_attention(**x, max_new=new).double()
    rms = lambda e: float(e.square().mean().sqrt())  # noqa: E731
    assert rms(out - o) <= limit * rms(o.to(dtype).double() - o)


def test_tree_attention_padded_step_over_a_wide_table():
    """Rows for 32768 tokens and a table for a million keys, of which a step uses 300 and 800."""
    x = attention_inputs([500], [300], 64, 8, 64, 16, torch.bfloat16, mask="chain")
    want = serving.tree_attention(**x, max_new=300)
    q = torch.zeros((32768, 64, 64), dtype=torch.bfloat16, device=DEV)
    q[:300] = x["q"]
    table = torch.full((1, 65536), -1, dtype=torch.int32, device=DEV)
    table[:, :x["page_table"].shape[1]] = x["page_table"]
    assert torch.equal(serving.tree_attention(**dict(x, q=q, page_table=table), max_new=300)[:300], want)
