"""What a serving loop over draft trees runs next to the certified attention: the step's paging, rotary
positions, the draft model's attention over the paged cache, and the logits' penalties and masks.

  plan_step       page allocation, slot map, positions and lengths of a step, from the request lengths
  rope            rotary positions with one to four axes (`inverse`: its gradient)
  rope_append     the same, with the keys and values written into the paged cache
  tree_attention  attention of drafted tokens (a tree, a chain, a single token) over the paged cache
  process_logits  penalties for repeated tokens, biases and grammar masks

Ordinary floating-point operators, hand-written CUDA behind include/exactattn_serving.h: 32-bit arithmetic and
outputs rounded once, except that tree_attention takes its weights into the product with the values as 16-bit
numbers (a pair of them for up to 16 query rows a kv head, one for more). Drafts are proposals: the bits that count come from the certified
`cuda.launch`, which verifies them over the same cache. Torch CUDA tensors in and out, asynchronous on
the current stream, no host synchronisation, capturable in CUDA graphs. There is no CPU path. Nothing is
recorded for autograd: tensors that require grad are refused (ValueError) unless under torch.no_grad; a
training loop calls rope and its `inverse` from a torch.autograd.Function of its own.
"""

from __future__ import annotations

from typing import NamedTuple

import numpy as np
import torch

from . import _lib

PLAN_NO_PAGES, PLAN_TABLE_FULL, PLAN_TOO_MANY = 1, 2, 4


class StepPlan(NamedTuple):
    """What plan_step returns; the page table is updated in place."""
    slot_map: torch.Tensor   # (max_tokens,) int64: cache row of each token, -1: none
    positions: torch.Tensor  # (max_tokens,) int32
    token_seq: torch.Tensor  # (max_tokens,) int32: the sequence of each token, -1: padding
    q_start: torch.Tensor    # (batch + 1,) int32: first token of each sequence
    seq_lens: torch.Tensor   # (batch,) int32: keys after the step
    free_head: torch.Tensor  # (1,) int32: first unused entry of the free list
    status: torch.Tensor     # (1,) int32: 0, or PLAN_* bits


def _native():
    """The binding (csrc/ea_serving_py.cpp); raises if it is not built."""
    global _mod
    if _mod is None:
        _lib.load()  # the library it calls, and a clear error if that is missing
        try:
            from . import _serving_native
        except ImportError as e:
            raise RuntimeError(f"{e}: build it with `python -m exactattention_b200.build`") from e
        built = getattr(_serving_native, "torch_version", "built against another torch")
        if built != f"built against torch {torch.__version__}":
            raise RuntimeError(f"{_serving_native.__file__} was {built}, this is {torch.__version__}: "
                               "build it with `python -m exactattention_b200.build`")
        _mod = _serving_native
    return _mod


_mod = None


def plan_step(context_lens, new_lens, page_table, free_pages, page_size: int, max_tokens: int, *, free_head=None,
              depths=None) -> StepPlan:
    """Paging of one step (ea_plan_step_cuda). Sequence b holds context_lens[b] keys and receives
    new_lens[b] tokens (int32, (batch,)); pages it lacks are taken from free_pages[free_head:] (int32) in
    sequence order and written into page_table (batch, max_pages) int32, in place. Token t's position is its
    sequence's context + depths[t] (its depth in the draft tree; None: its number in the step). max_tokens
    sizes the outputs; tokens past the step's are padding (slot -1). Running out of pages, table columns or
    tokens sets bits of `status` (PLAN_*), with slot -1 for tokens without a page. The same plan twice gives
    the same pages: pass the returned free_head on to the next step."""
    return StepPlan(*_native().plan_step(context_lens, new_lens, page_table, free_pages, page_size, max_tokens, free_head,
                                         depths))


def rope_axes(sections, interleaved: bool = False) -> np.ndarray:
    """The axis of every frequency (int32) from the number of frequencies each axis gets: consecutive
    sections, or (interleaved) one frequency of every axis in turn until an axis has had its share."""
    sections = [int(s) for s in sections]
    if not sections or min(sections) < 0:
        raise ValueError("sections must be counts")
    if not interleaved:
        return np.repeat(np.arange(len(sections)), sections).astype(np.int32)
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return np.asarray(out, np.int32)


def _adjacent(pairs: str) -> bool:
    if pairs not in ("half", "adjacent"):
        raise ValueError("pairs must be 'half' or 'adjacent'")
    return pairs == "adjacent"


def rope(q, k, positions, inv_freq, *, axes=None, pairs: str = "half", inverse: bool = False):
    """Rotary positions (ea_rope_cuda): q (tokens, q_heads, d) and k (tokens, kv_heads, d), either may be
    None, any token and head strides (slices of a fused projection). Pair i is turned by
    positions[axes[i]] * inv_freq[i]: positions int32 (tokens,) or (axes, tokens), inv_freq float32
    (rot / 2,), axes int32 (rot / 2,) (from rope_axes; None: the first axis). pairs "half": channels i and
    i + rot / 2; "adjacent": 2 i and 2 i + 1; channels from rot on are copied. inverse turns back, which is
    also the gradient: with dq, dk of the outputs, rope(dq, dk, ..., inverse=True) gives those of the inputs.
    Returns new contiguous (q, k)."""
    return _native().rope(q, k, None, positions, inv_freq, axes, _adjacent(pairs), bool(inverse), None, None, None)


def rope_append(q, k, v, positions, inv_freq, slot_map, k_cache, v_cache, *, axes=None, pairs: str = "half"):
    """rope, with the turned k and the v written to the paged caches (pages, kv_heads, page_size, d; any
    page, head and row strides) at rows slot_map (int64 (tokens,), from plan_step; -1 writes nothing).
    Slots of one call must differ. Returns the turned q."""
    if slot_map is None:
        raise ValueError("rope_append needs slot_map")
    return _native().rope(q, k, v, positions, inv_freq, axes, _adjacent(pairs), False, slot_map, k_cache, v_cache)[0]


def tree_mask(parents) -> np.ndarray:
    """Visibility rows for tree_attention of one draft tree: parents[i] < i is node i's parent, -1 for a child
    of the last accepted token; node i sees itself and its ancestors. (nodes, words) int32, bit j % 32 of
    word j // 32."""
    parents = np.asarray(parents, np.int64)
    n = len(parents)
    if n and not ((parents < np.arange(n)).all() and parents.min() >= -1):
        raise ValueError("a parent must come before its child")
    out = np.zeros((n, max(1, (n + 31) // 32)), np.uint32)
    for i, p in enumerate(parents):
        if p >= 0:
            out[i] = out[p]
        out[i, i // 32] |= np.uint32(1 << (i % 32))
    return out.view(np.int32)


def tree_attention(q, k_cache, v_cache, page_table, seq_lens, q_start, alpha, *, tree_mask=None, max_new=None,
                   return_lse: bool = False, out=None):
    """Attention of a step's tokens over the paged cache, which already holds their keys and values
    (ea_tree_attention_cuda). q (tokens, q_heads, d) bf16 or fp16, any token and head strides; caches
    (pages, kv_heads, page_size, d), any page, head and row strides; page_table (batch, max_pages),
    seq_lens (batch,) (the step's tokens included), q_start (batch + 1,) int32, as plan_step gives them.
    Rows of q, of the caches and of `out` (contiguous) start on 16-byte boundaries.
    A token sees its sequence's earlier keys and, of the step's tokens, those whose bit is set in its row
    of tree_mask ((tokens, words) int32, see `tree_mask`); None: itself and the ones before it. Weights are
    2^(alpha q.k) (formats.default_alpha), as in `cuda.launch`. max_new (the most tokens of any sequence;
    None: all of q's) picks the kernel and its tiles, and any value is right: pass 1 for single tokens.
    Rows past q_start[batch] are not written. Returns out (tokens, q_heads, d), and with return_lse the log2
    of the weights' sums (tokens, q_heads) float32; a row that sees no key gives 0 and -inf. Values of keys
    that a row does not see cannot reach it. The result is not certified: it is the draft model's attention.
    For up to 16 query rows a kv head (by max_new) its error is that of the output's rounding; for more,
    the weights are rounded to the caches' type for the product with the values, and the root mean square
    error is up to 1.4 times that."""
    r = _native().tree_attention(q, k_cache, v_cache, page_table, seq_lens, q_start, alpha, tree_mask, max_new,
                                 bool(return_lse), out)
    return r if return_lse else r[0]


def process_logits(logits, row_seq=None, *, history=None, history_lens=None, prompt_lens=None, repetition=None,
                   frequency=None, presence=None, bias_ids=None, bias_values=None, allowed_bits=None, mask_rows=None,
                   draft_tokens=None, q_start=None, tree_mask=None, out=None):
    """Penalties, biases and grammar masks (ea_process_logits_cuda) on logits (rows, vocab) of bf16, fp16 or
    fp32; row r belongs to sequence row_seq[r] (int32; None: r; outside the batch: the row is copied, its mask too
    left out). The batch is the length of the sequences' tensors (history, repetition, frequency, presence, bias_ids, else
    q_start); with masks alone every row_seq from 0 to 2^30 - 1 is a sequence.
    history (batch, width) int32 holds each sequence's tokens, the first prompt_lens[b] of its
    history_lens[b] being the prompt; draft_tokens (rows,) int32 with q_start (batch + 1,) and tree_mask (as
    for tree_attention; None: a chain) add the drafted tokens on each row's path. Then, in 32 bits and
    rounded once: tokens that occurred are divided (positive logits) or multiplied by repetition[b]; minus
    frequency[b] times the generated occurrences, minus presence[b] if there is one; plus bias_values (batch,
    entries) at bias_ids (int32, negative: unused); -inf where the token's bit of allowed_bits[mask_rows[r]]
    ((states, words) int32, bit v % 32 of word v // 32; mask_rows None: r, negative: unrestricted) is clear.
    Steps whose tensors are None are left out. Returns `out` (may be logits), or a new tensor."""
    return _native().process_logits(logits, row_seq, history, history_lens, prompt_lens, repetition, frequency, presence,
                                    bias_ids, bias_values, allowed_bits, mask_rows, draft_tokens, q_start, tree_mask, out)
