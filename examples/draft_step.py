"""One step of a speculative decoding server over draft trees, on synthetic data: the serving operators together,
and the certified attention over the same paged cache as the check on the draft model's attention.

    python examples/draft_step.py            # prints what each part did

A few sequences hold contexts of different lengths in a paged cache. Each receives a draft tree. The step then runs
  plan_step       pages for the trees, slots, positions (a node's position is the context plus its depth), lengths
  rope_append     rotary positions on the nodes' queries and keys, keys and values into the cache
  tree_attention  every node over its context and its ancestors
  process_logits  penalties that follow each node's path, and a grammar mask, before the greedy choice
and cuda.launch computes the certified bits of the same attention, the ones a verifier would go by.
"""

from __future__ import annotations

import os
import random
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.abspath(os.path.join(os.path.dirname(__file__), "..")))

from exactattention_b200 import cuda, default_alpha, serving  # noqa: E402


def draft_tree(rng: random.Random, nodes: int):
    """A random tree in breadth-first order: (parents, depths); -1 is the last accepted token."""
    parents, depths = [], []
    for i in range(nodes):
        p = rng.randrange(max(-1, i - 4), i) if i else -1
        parents.append(p)
        depths.append(depths[p] + 1 if p >= 0 else 0)
    return parents, depths


def run(contexts=(700, 33, 1290), nodes=(12, 1, 40), q_heads=16, kv_heads=8, d=128, page=16, vocab=4099, seed=0):
    """Runs the step; returns the plan, the attention of the step's tokens (draft and certified) and the chosen tokens."""
    dev = torch.device("cuda")
    rng, gen = random.Random(seed), torch.Generator(device=dev).manual_seed(seed)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)  # noqa: E731
    rand = lambda *shape: torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16)  # noqa: E731
    contexts, nodes = np.asarray(contexts), np.asarray(nodes)
    batch, total = len(contexts), int(nodes.sum())

    # what the server holds: a pool of pages, the sequences' tables, the pages that are free
    owned = -(-contexts // page)
    width = int((-(-(contexts + nodes) // page)).max())
    pool = np.array(rng.sample(range(int(owned.sum()) + 4 * batch + total), int(owned.sum()) + 4 * batch + total))
    table = np.full((batch, width), -1)
    for b, n in enumerate(owned):
        table[b, :n], pool = pool[:n], pool[n:]
    pages = int(owned.sum()) + 4 * batch + total
    k_cache, v_cache = rand(pages, kv_heads, page, d), rand(pages, kv_heads, page, d)
    page_table = i32(table)

    # the draft: trees, tokens, and what the draft model's projection gave for them
    trees = [draft_tree(rng, int(n)) for n in nodes]
    words = max(1, -(-int(nodes.max()) // 32))
    mask = np.concatenate([np.pad(m, ((0, 0), (0, words - m.shape[1]))) for m in (serving.tree_mask(p) for p, _ in trees)])
    tree_mask, depths = torch.from_numpy(mask).to(dev), i32(np.concatenate([dp for _, dp in trees]))
    draft_tokens = torch.randint(0, vocab, (total,), generator=gen, device=dev, dtype=torch.int32)
    qkv = rand(total, q_heads + 2 * kv_heads, d)

    plan = serving.plan_step(i32(contexts), i32(nodes), page_table, i32(pool), page, total, depths=depths)
    inv_freq = (1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)).float().to(dev)
    q = serving.rope_append(qkv[:, :q_heads], qkv[:, q_heads:q_heads + kv_heads], qkv[:, q_heads + kv_heads:],
                            plan.positions, inv_freq, plan.slot_map, k_cache, v_cache)
    alpha = default_alpha(d)
    drafted, lse = serving.tree_attention(q, k_cache, v_cache, page_table, plan.seq_lens, plan.q_start, alpha,
                                          tree_mask=tree_mask, max_new=int(nodes.max()), return_lse=True)

    logits = torch.randn((total, vocab), generator=gen, device=dev) * 3
    history = torch.randint(0, vocab, (batch, 200), generator=gen, device=dev, dtype=torch.int32)
    lens = i32([200, 50, 120][:batch] + [200] * (batch - 3))
    allowed = torch.randint(-2**31, 2**31, (2, -(-vocab // 32)), generator=gen, device=dev).to(torch.int32)
    scores = serving.process_logits(
        logits, plan.token_seq, history=history, history_lens=lens, prompt_lens=lens // 2,
        repetition=torch.full((batch,), 1.1, device=dev), presence=torch.full((batch,), 0.2, device=dev),
        allowed_bits=allowed, mask_rows=plan.token_seq % 3 - 1, draft_tokens=draft_tokens, q_start=plan.q_start,
        tree_mask=tree_mask)

    # the certified bits: each (node, head) row lists the cache rows of its context and its ancestors
    tab, starts = page_table.cpu().numpy(), plan.q_start.cpu().numpy()
    row_ptr, keys = [0], []
    for t in range(total):
        b = int(np.searchsorted(starts, t, side="right")) - 1
        i = np.flatnonzero(np.unpackbits(mask[t].view(np.uint8), bitorder="little"))
        at = np.concatenate([np.arange(contexts[b]), contexts[b] + i])
        for h in range(q_heads):
            rows = (tab[b, at // page].astype(np.int64) * kv_heads + h // (q_heads // kv_heads)) * page + at % page
            keys.append(rows)
            row_ptr.append(row_ptr[-1] + len(rows))
    bits, flags = cuda.launch(q.reshape(-1, d).view(torch.int16), k_cache.reshape(-1, d).view(torch.int16),
                              v_cache.reshape(-1, d).view(torch.int16), alpha,
                              row_ptr=torch.tensor(row_ptr, dtype=torch.int64, device=dev),
                              key_idx=torch.from_numpy(np.concatenate(keys)).to(dev))
    certified = bits.view(torch.bfloat16).reshape(total, q_heads, d)
    return dict(plan=plan, drafted=drafted, lse=lse, certified=certified, flags=flags, scores=scores,
                chosen=scores.argmax(-1))


def main() -> None:
    r = run()
    off = (r["drafted"].float() - r["certified"].float()).abs()
    p = r["plan"]
    print(f"planned {int(p.q_start[-1])} drafted tokens over {p.seq_lens.numel()} sequences, status {int(p.status)}, "
          f"{int(p.free_head)} pages taken")
    print(f"draft attention against the certified bits: {float((off == 0).float().mean()):.1%} of the values equal, largest "
          f"difference {float(off.max()):.2g}; flags {sorted(set(r['flags'].tolist()))}")
    print("next token of each node:", r["chosen"].tolist())


if __name__ == "__main__":
    main()
