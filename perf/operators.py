"""The operators of one decoding step over draft trees: what is measured, on which inputs, and their plain forms.

  plan        page allocation, slot map and positions of a step, from request lengths
  rope        rotary positions (one or several axes), with the rotated keys' write into the paged cache or as a gradient
  attention   attention of drafted tokens (a tree, a chain, or one token) over a paged cache
  logits      penalties for repeated tokens, biases and grammar masks

`run` computes them through exactattention_b200.serving where `own` is true, and otherwise with elementary
torch operations in 32 bits. Lengths follow from the case alone; which sequence has which length, the pages, the trees
and all values follow from the seed.
"""

import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # every token step of a server with 64 running requests: contexts as in the paged decode benchmark
        dict(name="plan_decode", op="plan", seqs=64, ctx_min=4096, ctx_max=32768, new_min=1, new_max=1, page=16,
             free=512, tree=False),
        # a step that admits prompts in chunks beside draft trees: many requests, a quarter of a million tokens, odd pages
        dict(name="plan_prompts", op="plan", seqs=509, ctx_min=0, ctx_max=20011, new_min=1, new_max=1031, page=24,
             free=40000, tree=True),
        # prompt with images / video: three position axes, 16 q and 8 kv heads, keys and values written to the cache
        dict(name="rope_video", op="rope", tokens=16927, q_heads=16, kv_heads=8, d=128, rot=128, axes=3, pos_max=32768,
             pairs="half", way="append", page=16, type="bf16"),
        # the gradient (rotation back) of a long text, adjacent pairs over part of the head, 32-bit values, odd sizes
        dict(name="rope_gradient", op="rope", tokens=4099, q_heads=28, kv_heads=4, d=96, rot=64, axes=1, pos_max=32768,
             pairs="adjacent", way="gradient", page=16, type="fp32"),
        # the smallest call: one request, one token
        dict(name="attention_one", op="attention", seqs=1, ctx_min=777, ctx_max=777, new_min=1, new_max=1, q_heads=16,
             kv_heads=8, d=128, page=16, mask="chain", type="bf16"),
        # paged decode of a full server (the framework's paged decode configuration)
        dict(name="attention_decode", op="attention", seqs=64, ctx_min=4096, ctx_max=32768, new_min=1, new_max=1,
             q_heads=16, kv_heads=8, d=128, page=16, mask="chain", type="bf16"),
        # draft trees of up to 64 nodes over prefixes around 8K tokens (the framework's tree configuration, made ragged)
        dict(name="attention_tree", op="attention", seqs=16, ctx_min=1021, ctx_max=15362, new_min=17, new_max=64,
             q_heads=16, kv_heads=8, d=128, page=16, mask="tree", type="fp16"),
        # chunks of 256 tokens behind a long cache with wide head groups: bound by the tensor cores
        dict(name="attention_chunk", op="attention", seqs=4, ctx_min=16384, ctx_max=16384, new_min=256, new_max=256,
             q_heads=32, kv_heads=4, d=128, page=64, mask="chain", type="bf16"),
        # ragged small trees, seven heads a group, 64 channels, pages that are no power of two, an empty context
        dict(name="attention_ragged", op="attention", seqs=23, ctx_min=0, ctx_max=3001, new_min=1, new_max=33,
             q_heads=28, kv_heads=4, d=64, page=24, mask="tree", type="fp16"),
        # one request's next token
        dict(name="logits_one", op="logits", seqs=1, new_min=1, new_max=1, vocab=32000, history=700, biases=16,
             grammar=True, tree=False, type="bf16"),
        # a batch of running requests with long histories
        dict(name="logits_batch", op="logits", seqs=256, new_min=1, new_max=1, vocab=131072, history=4096, biases=64,
             grammar=True, tree=False, type="bf16"),
        # every node of 16 draft trees: the penalties follow each node's path; odd vocabulary, 32-bit logits
        dict(name="logits_tree", op="logits", seqs=16, new_min=64, new_max=64, vocab=100003, history=1500, biases=32,
             grammar=True, tree=True, type="fp32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["plan", "rope", "rope", "attention", "attention", "attention", "attention", "logits", "logits"])
    if op == "plan":
        seqs, new = _log(rng, 1, 1024), _log(rng, 1, 512)
        page, ctx = rng.choice([1, 8, 16, 24, 64, 128]), _log(rng, 1, 32768)
        need = seqs * (-(-new // page) + 1)
        return dict(op=op, seqs=seqs, ctx_min=rng.choice([0, ctx // 7]), ctx_max=ctx, new_min=rng.choice([0, 1]), new_max=new,
                    page=page, free=need + rng.randrange(100), tree=rng.random() < 0.5)
    if op == "rope":
        kv, g, d = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8]), rng.choice([64, 80, 96, 128])
        axes = rng.choice([1, 1, 2, 3])
        return dict(op=op, tokens=_log(rng, 1, 20000), q_heads=kv * g, kv_heads=kv, d=d,
                    rot=rng.choice([d, d, 64, 48]), axes=axes, pos_max=_log(rng, 128, 32768),
                    pairs=rng.choice(["half", "half", "adjacent"]), way=rng.choice(["append", "plain", "gradient"]),
                    page=rng.choice([8, 16, 24, 64]), type=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if op == "attention":
        kv, g, d = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8]), rng.choice([64, 80, 96, 128, 128])
        seqs, new = _log(rng, 1, 64), rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 256)])
        # no more key / value bytes than the largest listed decode, and few enough scores for the plain form
        ctx = min(_log(rng, 16, 131072), 1000000 * 8 // (seqs * kv), 1200000000 // (seqs * kv * g * new))
        ctx = max(16, ctx)
        return dict(op=op, seqs=seqs, ctx_min=rng.choice([0, ctx // 8, ctx]), ctx_max=ctx, new_min=rng.choice([1, new]),
                    new_max=new, q_heads=kv * g, kv_heads=kv, d=d, page=rng.choice([8, 16, 16, 24, 32, 64, 128]),
                    mask=rng.choice(["tree", "chain"]), type=rng.choice(["bf16", "bf16", "fp16"]))
    vocab = _log(rng, 1000, 160000)
    rows = min(_log(rng, 1, 1024), 100000000 // vocab)
    tree = rows >= 4 and rng.random() < 0.5
    new = _log(rng, 2, min(64, rows)) if tree else 1
    return dict(op=op, seqs=max(1, rows // new), new_min=rng.choice([1, new]), new_max=new, vocab=vocab,
                history=_log(rng, 1, 16384), biases=_log(rng, 1, 256), grammar=rng.random() < 0.7, tree=tree,
                type=rng.choice(["bf16", "fp16", "fp32"]))


def _spread(lo, hi, n, step):
    """n lengths over lo..hi, the ends among them, the same for every seed."""
    if n == 1:
        return np.array([hi], np.int64)
    order = (np.arange(n, dtype=np.int64) * step) % n if math.gcd(step, n) == 1 else np.arange(n, dtype=np.int64)
    return lo + (hi - lo) * order // (n - 1)


def _lengths(case):
    n = case["seqs"]
    return _spread(case.get("ctx_min", 0), case.get("ctx_max", 0), n, 1), _spread(case["new_min"], case["new_max"], n, 7)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _tree_rows(rng, new):
    """A random draft tree per sequence: (depth of every node, visibility rows as Python integers)."""
    depth, rows = [], []
    for n in new:
        seen, dep = [], []
        for i in range(int(n)):
            parent = rng.randrange(max(0, i - 8), i + 1) - 1 if i else -1  # -1: a child of the last accepted token
            seen.append((seen[parent] if parent >= 0 else 0) | (1 << i))
            dep.append(dep[parent] + 1 if parent >= 0 else 0)
        depth += dep
        rows += seen
    return depth, rows


def _words(rows, width):
    """Visibility rows packed into int32 words, bit j of word j // 32."""
    out = np.zeros((len(rows), width), np.uint32)
    for w in range(width):
        out[:, w] = [(r >> (32 * w)) & 0xFFFFFFFF for r in rows]
    return torch.from_numpy(out.view(np.int32)).cuda()


def _pages(gen, used, page, extra):
    """A page table over one pool, its pages in random order: (table, number of pages, the pages left over)."""
    need = -(-used // page)
    width = max(1, int(need.max()) + extra)
    pool = torch.randperm(int(need.sum()) + 1, generator=gen, device="cuda", dtype=torch.int32)
    col = torch.arange(width, device="cuda")
    cnt = torch.from_numpy(need).cuda()
    at = torch.cumsum(cnt, 0) - cnt
    idx = at[:, None] + col[None, :]
    table = torch.where(col[None, :] < cnt[:, None], pool[idx.clamp(max=pool.numel() - 1)], 0)
    return table.to(torch.int32).contiguous(), pool.numel()


def _ints(x):
    return torch.from_numpy(np.ascontiguousarray(x).astype(np.int32)).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = random.Random(seed)
    return {"plan": _prepare_plan, "rope": _prepare_rope, "attention": _prepare_attention,
            "logits": _prepare_logits}[case["op"]](case, gen, rng)


def _normal(gen, shape, dtype, scale=None):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16 if dtype == torch.bfloat16 else torch.float32)
    return (x if scale is None else x * scale.to(x.dtype)).to(dtype)


def _prepare_plan(case, gen, rng):
    ctx, new = _lengths(case)
    order = np.array(rng.sample(range(case["seqs"]), case["seqs"]))
    ctx, new = ctx[order], new[order]
    page = case["page"]
    extra = int((-(-(ctx + new) // page)).max() - (-(-ctx // page)).max()) + 1
    table, pool = _pages(gen, ctx, page, extra)
    total = int(new.sum())
    cap = -(-max(total, 1) // 64) * 64  # steps are padded to a multiple of 64 tokens
    depths = None
    if case["tree"]:
        depths = np.zeros(cap, np.int64)
        d = np.concatenate([np.minimum(np.arange(n), rng.randrange(3, 12)) for n in new] + [np.zeros(0, np.int64)])
        depths[:total] = d
        depths = _ints(depths)
    free = pool + torch.randperm(case["free"], generator=gen, device="cuda", dtype=torch.int32)
    return dict(case=case, context_lens=_ints(ctx), new_lens=_ints(new), page_table=table, free_pages=free,
                free_head=torch.full((1,), rng.randrange(0, 3), dtype=torch.int32, device="cuda"), max_tokens=cap,
                depths=depths)


def _inv_freq(rot):
    return (1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().cuda()


def _prepare_rope(case, gen, rng):
    n, hq, hk, d, dt = case["tokens"], case["q_heads"], case["kv_heads"], case["d"], TYPES[case["type"]]
    page = case["page"]
    # q, k and v are slices of one projection's output, as a model has them
    qkv = _normal(gen, (n, hq + 2 * hk, d), dt)
    pos = torch.randint(0, case["pos_max"], (case["axes"], n), generator=gen, device="cuda", dtype=torch.int32)
    half = case["rot"] // 2
    cut = [half * (a + 1) // (case["axes"] + 1) for a in range(case["axes"] - 1)] + [half]  # the last axes get more
    axes = torch.zeros(half, dtype=torch.int32)
    for a in range(1, case["axes"]):
        axes[cut[a - 1]:] = a
    s = dict(case=case, q=qkv[:, :hq], k=qkv[:, hq:hq + hk], v=qkv[:, hq + hk:], positions=pos, axes=axes.cuda(),
             inv_freq=_inv_freq(case["rot"]))
    if case["way"] == "append":
        pages = -(-n // page) + 3
        slots = torch.randperm(pages * page, generator=gen, device="cuda")[:n]
        s["slot_map"] = torch.where(torch.arange(n, device="cuda") % 64 == 63, -1, slots)  # padding among them
        s["k_cache"] = torch.zeros((pages, hk, page, d), dtype=dt, device="cuda")
        s["v_cache"] = torch.zeros_like(s["k_cache"])
    return s


def _prepare_attention(case, gen, rng):
    ctx, new = _lengths(case)
    order = np.array(rng.sample(range(case["seqs"]), case["seqs"]))
    ctx, new = ctx[order], new[order]
    hq, hk, d, dt, page = case["q_heads"], case["kv_heads"], case["d"], TYPES[case["type"]], case["page"]
    table, pool = _pages(gen, ctx + new, page, 0)
    total = int(new.sum())
    scale = torch.exp2(torch.rand((hk, 1, d), generator=gen, device="cuda") * 2 - 1)
    s = dict(case=case, q=_normal(gen, (total, hq, d), dt),
             k_cache=_normal(gen, (pool, hk, page, d), dt, scale), v_cache=_normal(gen, (pool, hk, page, d), dt),
             page_table=table, seq_lens=_ints(ctx + new), q_start=_ints(np.concatenate([[0], np.cumsum(new)])),
             alpha=1.0 / math.sqrt(d) / math.log(2), max_new=int(new.max()), max_len=int((ctx + new).max()), tree_mask=None)
    if case["mask"] == "tree":
        s["tree_mask"] = _words(_tree_rows(rng, new)[1], -(-int(new.max()) // 32))
    return s


def _prepare_logits(case, gen, rng):
    _, new = _lengths(case)
    b, v, h = case["seqs"], case["vocab"], case["history"]
    new = new[np.array(rng.sample(range(b), b))]
    total = int(new.sum())
    lens = _spread(max(1, h // 4), h, b, 5)
    u = torch.rand((b, h), generator=gen, device="cuda")
    history = (v * u ** 3).to(torch.int32).clamp(max=v - 1)  # few tokens often, many seldom
    ids = (torch.arange(case["biases"], device="cuda")[None, :] * 7919
           + torch.randint(0, v, (b, 1), generator=gen, device="cuda")) % v
    if math.gcd(7919, v) != 1 or case["biases"] > v:
        ids = torch.arange(case["biases"], device="cuda")[None, :].expand(b, -1) % v
    pick = lambda *vals: torch.tensor([rng.choice(vals) for _ in range(b)], dtype=torch.float32, device="cuda")  # noqa: E731
    s = dict(case=case, logits=_normal(gen, (total, v), TYPES[case["type"]]) * 3,
             row_seq=torch.repeat_interleave(torch.arange(b, device="cuda", dtype=torch.int32),
                                             torch.from_numpy(new).cuda()),
             history=history, history_lens=_ints(lens), prompt_lens=_ints(lens // 2), repetition=pick(1.0, 1.1, 1.3),
             frequency=pick(0.0, 0.2, 0.5), presence=pick(0.0, 0.4), bias_ids=ids.to(torch.int32).contiguous(),
             bias_values=torch.randn((b, case["biases"]), generator=gen, device="cuda") * 5,
             q_start=_ints(np.concatenate([[0], np.cumsum(new)])), draft_tokens=None, tree_mask=None,
             max_new=int(new.max()), allowed_bits=None, mask_rows=None)
    if case["tree"]:
        s["draft_tokens"] = (v * torch.rand(total, generator=gen, device="cuda") ** 3).to(torch.int32).clamp(max=v - 1)
        s["tree_mask"] = _words(_tree_rows(rng, new)[1], -(-int(new.max()) // 32))
    if case["grammar"]:
        words = -(-v // 32)
        states = max(1, total // 2)  # rows share grammar states; every fourth row is free of a grammar
        a = torch.randint(-2**31, 2**31, (states, words), generator=gen, device="cuda")
        keep = torch.rand((states, 1), generator=gen, device="cuda") < 0.5
        b2 = torch.randint(-2**31, 2**31, (states, words), generator=gen, device="cuda")
        s["allowed_bits"] = torch.where(keep, a & b2, a | b2).to(torch.int32)
        rows = torch.randint(0, states, (total,), generator=gen, device="cuda", dtype=torch.int32)
        s["mask_rows"] = torch.where(torch.arange(total, device="cuda") % 4 == 3, -1, rows).to(torch.int32)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "rope": _own_rope, "attention": _own_attention, "logits": _own_logits}[op](state)
    return {"plan": _plain_plan, "rope": _plain_rope, "attention": _plain_attention, "logits": _plain_logits}[op](state)


def _own_plan(s):
    from exactattention_b200 import serving

    p = serving.plan_step(s["context_lens"], s["new_lens"], s["page_table"], s["free_pages"], s["case"]["page"],
                          s["max_tokens"], free_head=s["free_head"], depths=s["depths"])
    return dict(page_table=s["page_table"], slot_map=p.slot_map, positions=p.positions, token_seq=p.token_seq,
                q_start=p.q_start, seq_lens=p.seq_lens, free_head=p.free_head, status=p.status)


def _own_rope(s):
    from exactattention_b200 import serving

    kw = dict(axes=s["axes"], pairs=s["case"]["pairs"])
    if s["case"]["way"] == "append":
        q = serving.rope_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["slot_map"], s["k_cache"],
                                s["v_cache"], **kw)
        return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])
    q, k = serving.rope(s["q"], s["k"], s["positions"], s["inv_freq"], inverse=s["case"]["way"] == "gradient", **kw)
    return dict(q=q, k=k)


def _own_attention(s):
    from exactattention_b200 import serving

    out, lse = serving.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["seq_lens"], s["q_start"],
                                      s["alpha"], tree_mask=s["tree_mask"], max_new=s["max_new"], return_lse=True)
    return dict(out=out, lse=lse)


def _own_logits(s):
    from exactattention_b200 import serving

    return serving.process_logits(
        s["logits"], s["row_seq"], history=s["history"], history_lens=s["history_lens"], prompt_lens=s["prompt_lens"],
        repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"], bias_ids=s["bias_ids"],
        bias_values=s["bias_values"], allowed_bits=s["allowed_bits"], mask_rows=s["mask_rows"],
        draft_tokens=s["draft_tokens"], q_start=s["q_start"], tree_mask=s["tree_mask"])


def _plain_plan(s):
    ps, cap = s["case"]["page"], s["max_tokens"]
    ctx, new, table, free = s["context_lens"].long(), s["new_lens"].long(), s["page_table"], s["free_pages"]
    width = table.shape[1]
    have, need = (ctx + ps - 1) // ps, (ctx + new + ps - 1) // ps
    fresh = need - have
    first = torch.cumsum(fresh, 0) - fresh + s["free_head"].long()
    col = torch.arange(width, device=table.device)
    at = first[:, None] + col[None, :] - have[:, None]
    got = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    table = torch.where((col >= have[:, None]) & (col < need[:, None]), got, table)
    q_start = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    t = torch.arange(cap, device=table.device)
    seq = torch.searchsorted(q_start[1:].contiguous(), t, right=True)
    valid = seq < new.numel()
    b = seq.clamp(max=new.numel() - 1)
    i = t - q_start[b]
    p = ctx[b] + i
    pg = table[b, (p // ps).clamp(max=width - 1)].long()
    slot = torch.where(valid & (p // ps < width) & (pg >= 0), pg * ps + p % ps, -1)
    pos = torch.where(valid, ctx[b] + (i if s["depths"] is None else s["depths"].long()), 0)
    end = s["free_head"].long() + fresh.sum()
    status = (end > free.numel()).int() + 2 * (need > width).any().int() + 4 * (q_start[-1:] > cap).int()
    return dict(page_table=table, slot_map=slot, positions=pos.int(), token_seq=torch.where(valid, seq, -1).int(),
                q_start=q_start.int(), seq_lens=(ctx + new).int(), free_head=end.clamp(max=free.numel()).int(),
                status=status.int())


def _cos_sin(pos, freq):
    """cos and sin of pos * freq in 32 bits: freq = hi + lo with few enough bits in hi that pos * hi is exact."""
    hi = (freq.view(torch.int32) & -65536).view(torch.float32)
    a, b = pos * hi, pos * (freq - hi)
    ca, sa, cb, sb = torch.cos(a), torch.sin(a), torch.cos(b), torch.sin(b)
    return ca * cb - sa * sb, sa * cb + ca * sb


def _rotate(x, cos, sin, rot, pairs):
    y = x.float()
    if pairs == "half":
        a, b, rest = y[..., :rot // 2], y[..., rot // 2:rot], y[..., rot:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    else:
        a, b, rest = y[..., 0:rot:2], y[..., 1:rot:2], y[..., rot:]
        y = torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)
    return y.to(x.dtype)


def _plain_rope(s):
    c = s["case"]
    cos, sin = _cos_sin(s["positions"].float()[s["axes"].long()].T, s["inv_freq"])
    cos, sin = cos[:, None, :], (-sin if c["way"] == "gradient" else sin)[:, None, :]
    q, k = _rotate(s["q"], cos, sin, c["rot"], c["pairs"]), _rotate(s["k"], cos, sin, c["rot"], c["pairs"])
    if c["way"] != "append":
        return dict(q=q, k=k)
    t = torch.nonzero(s["slot_map"] >= 0)[:, 0]
    page, off = s["slot_map"][t] // c["page"], s["slot_map"][t] % c["page"]
    kc, vc = s["k_cache"].clone(), s["v_cache"].clone()
    kc[page, :, off], vc[page, :, off] = k[t], s["v"][t]
    return dict(q=q, k_cache=kc, v_cache=vc)


def _visible(mask, rows, width):
    """Packed visibility rows as truth values (rows, width)."""
    j = torch.arange(width, device=rows.device)
    return ((mask[rows][..., j // 32] >> (j % 32)) & 1).bool()


def _plain_attention(s):
    c = s["case"]
    b, hk, d, g, t = c["seqs"], c["kv_heads"], c["d"], c["q_heads"] // c["kv_heads"], s["max_new"]
    pages = -(-s["max_len"] // c["page"])
    n = pages * c["page"]
    gather = lambda x: x[s["page_table"][:, :pages].long()].transpose(1, 2).reshape(b, hk, n, d).float()  # noqa: E731
    start, new = s["q_start"][:-1].long(), s["q_start"].long().diff()
    ctx = s["seq_lens"].long() - new
    i = torch.arange(t, device="cuda")
    rows = (start[:, None] + i).clamp(max=s["q"].shape[0] - 1)  # (b, t), padded with other rows
    q = s["q"][rows].float().reshape(b, t, hk, g, d).permute(0, 2, 1, 3, 4).reshape(b, hk, t * g, d)
    node = torch.arange(n, device="cuda") - ctx[:, None]  # (b, n): which drafted token a key is
    if s["tree_mask"] is None:
        among = i[:, None] >= i[None, :]
        among = among[None].expand(b, t, t)
    else:
        among = _visible(s["tree_mask"], rows, t)
    sees = (node < 0)[:, None, :] | (((node >= 0) & (node < new[:, None]))[:, None, :]
                                     & among.gather(2, node.clamp(0, t - 1)[:, None, :].expand(b, t, n)))
    sees = sees[:, None, :, None, :].expand(b, 1, t, g, n).reshape(b, 1, t * g, n)
    x = (q @ gather(s["k_cache"]).transpose(2, 3)) * s["alpha"]
    x = x.masked_fill_(~sees, -math.inf)
    m = x.amax(-1, keepdim=True)
    x = torch.exp2(x.sub_(torch.where(m == -math.inf, 0, m)))
    z = x.sum(-1, keepdim=True)
    o = (x @ gather(s["v_cache"])) / torch.where(z == 0, 1, z)
    lse = (m + torch.log2(z)).reshape(b, hk, t, g).permute(0, 2, 1, 3).reshape(b, t, hk * g)
    o = o.reshape(b, hk, t, g, d).permute(0, 2, 1, 3, 4).reshape(b, t, hk * g, d)
    real = i[None, :] < new[:, None]
    return dict(out=o[real].to(s["q"].dtype), lse=lse[real])


def _counts(s, rows, vocab):
    """How often each token was generated before each row's next one, and whether the prompt holds it."""
    h = s["history"].long()
    j = torch.arange(h.shape[1], device=h.device)
    prompt = j < s["prompt_lens"][:, None]
    made = (j >= s["prompt_lens"][:, None]) & (j < s["history_lens"][:, None])
    zero = torch.zeros((h.shape[0], vocab), dtype=torch.int32, device=h.device)
    in_prompt = zero.scatter_add(1, h, prompt.int())[rows]
    count = zero.scatter_add(1, h, made.int())[rows]
    if s["draft_tokens"] is not None:
        start, t = s["q_start"].long()[rows], s["max_new"]
        node = start[:, None] + torch.arange(t, device=h.device)
        inside = node < s["q_start"].long()[rows + 1][:, None]
        sees = _visible(s["tree_mask"], torch.arange(rows.numel(), device=h.device), t) & inside
        count.scatter_add_(1, s["draft_tokens"].long()[node.clamp(max=rows.numel() - 1)], sees.int())
    return in_prompt, count


def _plain_logits(s):
    x = s["logits"].float()
    rows, vocab = s["row_seq"].long(), x.shape[1]
    in_prompt, count = _counts(s, rows, vocab)
    rep = s["repetition"][rows][:, None]
    x = torch.where((in_prompt + count) > 0, torch.where(x > 0, x / rep, x * rep), x)
    del in_prompt
    x = x - s["frequency"][rows][:, None] * count
    x = x - s["presence"][rows][:, None] * (count > 0)
    del count
    bias = torch.zeros((s["bias_ids"].shape[0], vocab), device=x.device)
    x = x + bias.scatter_add_(1, s["bias_ids"].long(), s["bias_values"])[rows]
    if s["allowed_bits"] is not None:
        j = torch.arange(vocab, device=x.device)
        allowed = ((s["allowed_bits"][:, j // 32] >> (j % 32)) & 1).bool()
        m = s["mask_rows"].long()
        x = x.masked_fill_(~allowed[m.clamp(min=0)] & (m >= 0)[:, None], -math.inf)
    return x.to(s["logits"].dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "plan":
        ctx, new = _lengths(case)
        fresh = -(-(ctx + new) // case["page"]) - -(-ctx // case["page"])
        touched = np.where(new > 0, -(-(ctx + new) // case["page"]) - ctx // case["page"], 0)
        return dict(bytes=int(case["seqs"] * 16 + 8 * fresh.sum() + 4 * (touched - fresh).sum()
                              + new.sum() * (20 if case["tree"] else 16)), flops=0)
    if op == "rope":
        n, hq, hk, d, e = case["tokens"], case["q_heads"], case["kv_heads"], case["d"], BYTES[case["type"]]
        heads = hq + (2 * hk if case["way"] == "append" else hk)
        return dict(bytes=n * (2 * heads * d * e + 4 * case["axes"] + (8 if case["way"] == "append" else 0)),
                    flops=n * (hq + hk) * case["rot"] * 3)
    if op == "attention":
        ctx, new = _lengths(case)
        hq, hk, d = case["q_heads"], case["kv_heads"], case["d"]
        words = -(-int(new.max()) // 32) if case["mask"] == "tree" else 0
        pairs = int((ctx * new + (new if case["mask"] == "tree" else new * (new + 1) // 2)).sum())
        return dict(bytes=int((ctx + new).sum()) * hk * d * 4 + int(new.sum()) * (hq * (4 * d + 4) + 4 * words)
                    + 4 * int((-(-(ctx + new) // case["page"])).sum()), flops=4 * d * hq * pairs)
    _, new = _lengths(case)
    rows, v = int(new.sum()), case["vocab"]
    masks = max(1, rows // 2) * -(-v // 32) * 4 if case["grammar"] else 0
    lens = int(_spread(max(1, case["history"] // 4), case["history"], case["seqs"], 5).sum())
    return dict(bytes=2 * rows * v * BYTES[case["type"]] + masks + 4 * lens + 8 * case["seqs"] * case["biases"],
                flops=rows * v)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None  # whole numbers
    if case["op"] == "rope":
        angle = s["positions"][s["axes"].long()].double().T * s["inv_freq"].double()
        turn = torch.polar(torch.ones_like(angle), -angle if case["way"] == "gradient" else angle)[:, None, :]
        rot = case["rot"]

        def turned(x):
            x = x.double()
            head = x[..., :rot]
            z = head.unflatten(-1, (2, rot // 2)).transpose(-1, -2) if case["pairs"] == "half" else head.unflatten(-1, (rot // 2, 2))
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
            z = (z.transpose(-1, -2) if case["pairs"] == "half" else z).reshape(head.shape)
            return torch.cat([z, x[..., rot:]], -1)

        if case["way"] != "append":
            return dict(q=turned(s["q"]), k=turned(s["k"]))
        out = {}
        ok = s["slot_map"] >= 0
        for name, x in (("k_cache", turned(s["k"])), ("v_cache", s["v"].double())):
            flat = torch.zeros((s[name].shape[0] * case["page"], case["kv_heads"], case["d"]), dtype=torch.float64, device="cuda")
            flat[s["slot_map"][ok]] = x[ok]
            out[name] = flat.unflatten(0, (-1, case["page"])).transpose(1, 2).contiguous()
        return dict(q=turned(s["q"]), **out)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    return _exact_logits(case, s)


def _exact_attention(case, s):
    hk, d = case["kv_heads"], case["d"]
    g = case["q_heads"] // hk
    ends, lens = s["q_start"].tolist(), s["seq_lens"].tolist()
    outs, lses = [], []
    for b in range(case["seqs"]):
        lo, hi, n = ends[b], ends[b + 1], lens[b]
        new, ctx = hi - lo, n - (hi - lo)
        pg = s["page_table"][b, :-(-n // case["page"])].long()
        k = s["k_cache"][pg].permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :n].double()
        v = s["v_cache"][pg].permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :n].double()
        q = s["q"][lo:hi].double().reshape(new, hk, g, d)
        hidden = torch.zeros((new, n), dtype=torch.bool, device="cuda")
        if s["tree_mask"] is None:
            hidden[:, ctx:] = torch.ones((new, new), dtype=torch.bool, device="cuda").triu(1)
        else:
            bits = s["tree_mask"][lo:hi].cpu().numpy().view(np.uint8)
            hidden[:, ctx:] = torch.from_numpy(np.unpackbits(bits, axis=1, bitorder="little")[:, :new] == 0).cuda()
        x = torch.einsum("thgd,hnd->htgn", q, k) * (s["alpha"] * math.log(2))
        x = x.masked_fill(hidden[None, :, None, :], -math.inf)
        outs.append(torch.einsum("htgn,hnd->thgd", torch.softmax(x, -1), v).reshape(new, hk * g, d))
        lses.append((torch.logsumexp(x, -1) / math.log(2)).permute(1, 0, 2).reshape(new, hk * g))
    return dict(out=torch.cat(outs), lse=torch.cat(lses))


def _exact_logits(case, s):
    x = s["logits"].double()
    v = x.shape[1]
    seqs, ends = s["row_seq"].tolist(), s["q_start"].tolist()
    words = None if s["tree_mask"] is None else s["tree_mask"].cpu().numpy().view(np.uint8)
    out = torch.empty_like(x)
    for r, b in enumerate(seqs):
        n, p = int(s["history_lens"][b]), int(s["prompt_lens"][b])
        made = s["history"][b, p:n].long()
        if words is not None:
            path = np.flatnonzero(np.unpackbits(words[r], bitorder="little")[:ends[b + 1] - ends[b]])
            made = torch.cat([made, s["draft_tokens"][ends[b] + torch.from_numpy(path).cuda()].long()])
        count = torch.bincount(made, minlength=v).double()
        seen = count > 0
        seen[s["history"][b, :p].long()] = True
        rep, y = s["repetition"][b].double(), x[r]
        y = torch.where(seen, torch.where(y > 0, y / rep, y * rep), y)
        y = y - s["frequency"][b].double() * count - s["presence"][b].double() * (count > 0)
        y[s["bias_ids"][b].long()] += s["bias_values"][b].double()
        if s["allowed_bits"] is not None and int(s["mask_rows"][r]) >= 0:
            bits = s["allowed_bits"][int(s["mask_rows"][r])].cpu().numpy().view(np.uint8)
            y[torch.from_numpy(np.unpackbits(bits, bitorder="little")[:v] == 0).cuda()] = -math.inf
        out[r] = y
    return out
