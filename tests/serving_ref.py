"""Plain 64-bit implementations of the serving operators, written as loops over sequences and rows."""

import math

import numpy as np
import torch

# half a unit in the last place of a result, relative
HALF_ULP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24, torch.float32: 2.0**-149}


def plan_step(ctx, new, table, free, ps, cap, head=0, depths=None):
    table = table.copy()
    n_free, width = len(free), table.shape[1]
    slot, pos, seq, q_start, lens = [], [], [], [0], []
    status, used = 0, 0
    for b in range(len(ctx)):
        c, n = max(0, int(ctx[b])), max(0, int(new[b]))
        have, need = -(-c // ps), -(-(c + n) // ps)
        if need > width:
            status |= 2
        for col in range(have, need):
            at = head + used
            if col < width:
                table[b, col] = free[at] if at < n_free else -1
            used += 1
        for i in range(n):
            col = (c + i) // ps
            pg = table[b, col] if col < width else -1
            slot.append(int(pg) * ps + (c + i) % ps if pg >= 0 else -1)
            t = len(pos)
            pos.append(c + (i if depths is None or t >= cap else int(depths[t])))
            seq.append(b)
        q_start.append(q_start[-1] + n)
        lens.append(c + n)
    if head + used > n_free:
        status |= 1
    if q_start[-1] > cap:
        status |= 4
    pad = cap - len(pos)
    fix = lambda x, v, t: np.asarray((x + [v] * max(0, pad))[:cap], t)  # noqa: E731
    return dict(page_table=table, slot_map=fix(slot, -1, np.int64), positions=fix(pos, 0, np.int32),
                token_seq=fix(seq, -1, np.int32), q_start=np.asarray(q_start, np.int32),
                seq_lens=np.asarray(lens, np.int32), free_head=np.asarray([min(n_free, head + used)], np.int32),
                status=np.asarray([status], np.int32))


def rope(x, positions, inv_freq, axes, pairs, inverse):
    """(result, bound on what 32-bit arithmetic may be off by) in float64, for (tokens, heads, d)."""
    y = x.double().clone()
    half = inv_freq.numel()
    ax = torch.zeros(half, dtype=torch.long, device=x.device) if axes is None else axes.long()
    ang = positions.reshape(-1, x.shape[0])[ax].double().T * inv_freq.double()
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None] * (-1 if inverse else 1)
    i0, i1 = ((slice(0, half), slice(half, 2 * half)) if pairs == "half" else
              (slice(0, 2 * half, 2), slice(1, 2 * half, 2)))
    a, b = x[..., i0].double(), x[..., i1].double()
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    off = torch.zeros_like(y)
    # the reduced angle rounds at 2^-26 turns (1e-7 rad), sincospif at 2 ulp, the two products and the sum
    # at 2^-24 each: below 2^-20 of |a| + |b|
    off[..., i0] = off[..., i1] = 2.0**-20 * (a.abs() + b.abs())
    return y, off


def tree_attention(q, k_cache, v_cache, table, lens, q_start, alpha, mask):
    """(out, lse, bound on out, bound on lse) in float64."""
    n, hq, d = q.shape
    hk, ps = k_cache.shape[1], k_cache.shape[2]
    g, dev = hq // hk, q.device
    out = torch.zeros((n, hq, d), dtype=torch.float64, device=dev)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device=dev)
    bound, lbound = torch.zeros_like(out), torch.zeros_like(lse)
    u = HALF_ULP[q.dtype]
    lens, q_start, tab = lens.tolist(), q_start.tolist(), table.cpu().numpy()
    for b in range(len(lens)):
        lo, hi, L = q_start[b], q_start[b + 1], lens[b]
        ctx = L - (hi - lo)
        keys = np.arange(L)
        pages = tab[b, keys // ps]
        real = (pages >= 0) & (pages < k_cache.shape[0])
        pg = torch.from_numpy(np.where(real, pages, 0).astype(np.int64)).to(dev)
        off = torch.from_numpy(keys % ps).to(dev)
        kk, vv = k_cache[pg, :, off].double(), v_cache[pg, :, off].double()  # (L, hk, d)
        for t in range(lo, hi):
            vis = real.copy()
            for j in range(hi - lo):
                if ctx + j < 0:
                    continue
                if mask is None:
                    see = j <= t - lo
                else:
                    w = j // 32
                    see = w < mask.shape[1] and bool((int(mask[t, w]) >> (j % 32)) & 1)
                vis[ctx + j] &= see
            idx = torch.from_numpy(np.flatnonzero(vis)).to(dev)
            if idx.numel() == 0:
                continue
            qt = q[t].double().reshape(hk, g, d)
            x = alpha * torch.einsum("hgd,nhd->hgn", qt, kk[idx])
            # 32-bit dot product of d terms
            dx = abs(alpha) * d * 2.0**-23 * torch.einsum("hgd,nhd->hgn", qt.abs(), kk[idx].abs()).nan_to_num().amax(-1)
            m = x.amax(-1, keepdim=True)
            w = torch.exp2(x - m)
            z = w.sum(-1)
            o = torch.einsum("hgn,nhd->hgd", w, vv[idx]) / z[..., None]
            mag = torch.einsum("hgn,nhd->hgd", w, vv[idx].abs()) / z[..., None]
            out[t] = o.reshape(hq, d)
            lse[t] = (m[..., 0] + torch.log2(z)).reshape(hq)
            # weights: score error, exp2, rounding to 16 bits, the sums' roundings; output rounded once
            rel = 2 * math.log(2) * dx + u + 2.0**-14
            bound[t] = (u * o.abs() + mag * rel[..., None]).reshape(hq, d) + TINY[q.dtype]
            lbound[t] = (dx + 2.0**-18 + m[..., 0].abs() * 2.0**-22).reshape(hq)
    return out, lse, bound, lbound


def process_logits(x, row_seq, history, history_lens, prompt_lens, rep, freq, pres, bias_ids, bias_vals, bits, mask_rows,
                   draft, q_start, tree):
    """(result, bound) in float64 on the CPU; all inputs numpy or None, x a CPU torch tensor."""
    y = x.double().clone()
    bound = torch.zeros_like(y)
    rows, vocab = x.shape
    batch = max([len(t) for t in (history, rep, freq, pres, bias_ids) if t is not None] + [0]) or \
        (rows if q_start is None else len(q_start) - 1)
    for r in range(rows):
        b = r if row_seq is None else int(row_seq[r])
        if not 0 <= b < batch:
            continue
        prompt, made = [], []
        if history is not None:
            n = int(history_lens[b])
            p = 0 if prompt_lens is None else min(int(prompt_lens[b]), n)
            prompt, made = list(history[b, :p]), list(history[b, p:n])
        if draft is not None:
            for j in range(int(q_start[b + 1] - q_start[b])):
                see = j <= r - q_start[b] if tree is None else j // 32 < tree.shape[1] and (int(tree[r, j // 32]) >> (j % 32)) & 1
                if see:
                    made.append(draft[q_start[b] + j])
        count = {}
        for t in made:
            count[int(t)] = count.get(int(t), 0) + 1
        re, fr, pr = (1.0 if rep is None else float(rep[b]), 0.0 if freq is None else float(freq[b]),
                      0.0 if pres is None else float(pres[b]))
        for t in set(count) | {int(p) for p in prompt}:
            if not 0 <= t < vocab:
                continue
            v, c = float(y[r, t]), count.get(t, 0)
            v = v / re if v > 0 else v * re
            mag = abs(v) + abs(fr * c) + (abs(pr) if c else 0)
            y[r, t] = v - fr * c - (pr if c else 0)
            bound[r, t] = 2.0**-21 * mag  # at most five 32-bit roundings of the sum's terms
        if bias_ids is not None:
            for t, v in zip(bias_ids[b], bias_vals[b]):
                if 0 <= t < vocab:
                    bound[r, t] += 2.0**-21 * (abs(float(y[r, t])) + abs(float(v)))
                    y[r, t] += float(v)
        if bits is not None:
            mr = r if mask_rows is None else int(mask_rows[r])
            if 0 <= mr < len(bits):
                ok = np.unpackbits(bits[mr].view(np.uint8), bitorder="little")[:vocab].astype(bool)
                y[r, torch.from_numpy(~ok)] = -math.inf
    return y, bound + HALF_ULP[x.dtype] * y.abs().nan_to_num(posinf=0, neginf=0) + TINY[x.dtype]


def assert_within(got, want, bound):
    """|got - want| <= bound where want is finite, and the same infinities and NaN elsewhere."""
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    special = ~fin & ~torch.isnan(want)
    assert torch.equal(got[special], want[special])
    d = (got - want).abs()[fin]
    over = d > bound[fin]
    assert not bool(over.any()), (f"{int(over.sum())} of {d.numel()} values off: worst {float((d / bound[fin]).max()):.3g} "
                                  "times the bound")
