"""What a serving loop over draft trees runs next to the certified attention: the step's paging, rotary
positions, the draft model's attention over the paged cache, and the logits' penalties and masks.

  plan_step       page allocation, slot map, positions and lengths of a step, from the request lengths
  rope            rotary positions with one to four axes (`inverse`: its gradient)
  rope_append     the same, with the keys and values written into the paged cache
  tree_attention  attention of drafted tokens (a tree, a chain, a single token) over the paged cache
  process_logits  penalties for repeated tokens, biases and grammar masks

Ordinary floating-point operators (32-bit arithmetic, outputs rounded once), hand-written CUDA behind
include/exactattn_serving.h. Drafts are proposals: the bits that count come from the certified
`cuda.launch`, which verifies them over the same cache. Torch CUDA tensors in and out, asynchronous on
the current stream, no host synchronisation, capturable in CUDA graphs. There is no CPU path.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import numpy as np
import torch

from . import _lib

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
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


def _check(rc: int, what: str) -> None:
    if rc:
        msg = _lib.load().ea_serving_last_error().decode(errors="replace")
        raise (RuntimeError if rc == -4 else ValueError)(f"{msg or what} (code {rc})")


def _call(fn, args, dev, what):
    """Calls fn(&args, stream) with `dev` current."""
    if dev.type != "cuda":
        raise RuntimeError(f"{what} needs CUDA tensors (there is no CPU path)")
    stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
    if dev.index == torch.cuda.current_device():
        rc = fn(ctypes.byref(args), stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(ctypes.byref(args), stream)
    if rc:
        _check(rc, what)


def _need(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _i32(t, name, dev, *shape):
    """Pointer of a contiguous int32 tensor of the given shape (None: any) on dev, or None for None."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor on {dev}")
    if len(t.shape) != len(shape) or any(w is not None and w != s for w, s in zip(shape, t.shape)):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    return t.data_ptr()


def _f32(t, name, dev, *shape):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.device != dev or not t.is_contiguous() or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape {shape} on {dev}")
    return t.data_ptr()


def plan_step(context_lens, new_lens, page_table, free_pages, page_size: int, max_tokens: int, *, free_head=None,
              depths=None) -> StepPlan:
    """Paging of one step (ea_plan_step_cuda). Sequence b holds context_lens[b] keys and receives
    new_lens[b] tokens (int32, (batch,)); pages it lacks are taken from free_pages[free_head:] (int32) in
    sequence order and written into page_table (batch, max_pages) int32, in place. Token t's position is its
    sequence's context + depths[t] (its depth in the draft tree; None: its number in the step). max_tokens
    sizes the outputs; tokens past the step's are padding (slot -1). Running out of pages, table columns or
    tokens sets bits of `status` (PLAN_*), with slot -1 for tokens without a page. The same plan twice gives
    the same pages: pass the returned free_head on to the next step."""
    dev = context_lens.device
    batch = context_lens.shape[0]
    _need(max_tokens >= 0 and page_size > 0, "max_tokens must not be negative and page_size must be positive")
    _need(page_table.dtype == torch.int32 and page_table.device == dev and page_table.dim() == 2
          and page_table.shape[0] == batch and (page_table.stride(1) == 1 or page_table.numel() <= batch),
          f"page_table must be a (batch, max_pages) int32 tensor on {dev} with contiguous rows")
    a = _lib.PlanStepArgs()
    a.context_lens = _i32(context_lens, "context_lens", dev, None)
    a.new_lens = _i32(new_lens, "new_lens", dev, batch)
    a.page_table = page_table.data_ptr()
    a.free_pages = _i32(free_pages, "free_pages", dev, None)
    a.free_head = _i32(free_head, "free_head", dev, 1)
    a.depths = _i32(depths, "depths", dev, max_tokens)
    slots = torch.empty(max_tokens, dtype=torch.int64, device=dev)
    ints = torch.empty(2 * max_tokens + 2 * batch + 3, dtype=torch.int32, device=dev)
    pos, seq, q_start, lens, head, status = ints.split([max_tokens, max_tokens, batch + 1, batch, 1, 1])
    p = ints.data_ptr()
    a.slot_map, a.positions, a.token_seq = slots.data_ptr(), p, p + 4 * max_tokens
    p += 8 * max_tokens
    a.q_start, a.seq_lens, a.next_free_head, a.status = p, p + 4 * (batch + 1), p + 4 * (2 * batch + 1), p + 8 * (batch + 1)
    a.table_stride = page_table.stride(0)
    a.batch, a.max_pages, a.page_size, a.num_free, a.max_tokens = (batch, page_table.shape[1], page_size,
                                                                   free_pages.shape[0], max_tokens)
    _call(_lib.load().ea_plan_step_cuda, a, dev, "plan_step")
    return StepPlan(slots, pos, seq, q_start, lens, head, status)


def rope_axes(sections, interleaved: bool = False) -> np.ndarray:
    """The axis of every frequency (int32) from the number of frequencies each axis gets: consecutive
    sections, or (interleaved) one frequency of every axis in turn until an axis has had its share."""
    sections = [int(s) for s in sections]
    _need(sections and min(sections) >= 0, "sections must be counts")
    if not interleaved:
        return np.repeat(np.arange(len(sections)), sections).astype(np.int32)
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return np.asarray(out, np.int32)


def _rope(q, k, v, positions, inv_freq, axes, pairs, inverse, slot_map, k_cache, v_cache):
    _need(pairs in ("half", "adjacent"), "pairs must be 'half' or 'adjacent'")
    ref = q if q is not None else k
    _need(ref is not None, "rope needs q or k")
    dev, dt = ref.device, ref.dtype
    _need(dt in _TYPES, "rope takes bfloat16, float16 or float32")
    n, d = ref.shape[0], ref.shape[2] if ref.dim() == 3 else -1
    for name, x in (("q", q), ("k", k), ("v", v)):
        _need(x is None or (x.dim() == 3 and x.shape[0] == n and x.shape[2] == d and x.dtype == dt and x.device == dev
                            and (x.stride(2) == 1 or x.shape[2] == 1)),
              f"{name} must be a (tokens, heads, d) tensor like q, with contiguous channels")
    if positions.dim() == 1:
        positions = positions[None]
    _need(positions.dtype == torch.int32 and positions.device == dev and positions.dim() == 2 and positions.shape[1] == n
          and (n <= 1 or positions.stride(1) == 1),
          f"positions must be int32 (tokens,) or (axes, tokens) on {dev}")
    half = inv_freq.shape[0]
    _need(2 * half <= d, "inv_freq has more frequencies than the head has pairs")
    a = _lib.RopeArgs()
    a.inv_freq = _f32(inv_freq, "inv_freq", dev, half)
    a.axes = _i32(axes, "axes", dev, half)
    a.positions, a.axis_stride, a.num_axes = positions.data_ptr(), positions.stride(0), positions.shape[0]
    q_out = k_out = None
    if q is not None:
        q_out = torch.empty((n, q.shape[1], d), dtype=dt, device=dev)
        a.q, a.q_stride, a.q_head_stride, a.q_heads = q.data_ptr(), q.stride(0), q.stride(1), q.shape[1]
        a.q_out = q_out.data_ptr()
    if k is not None:
        a.k, a.k_stride, a.k_head_stride, a.kv_heads = k.data_ptr(), k.stride(0), k.stride(1), k.shape[1]
    if slot_map is not None:
        _need(k is not None and v is not None and v.shape == k.shape, "rope_append needs k and v of one shape")
        _need(slot_map.dtype == torch.int64 and slot_map.device == dev and slot_map.is_contiguous()
              and tuple(slot_map.shape) == (n,), f"slot_map must be a contiguous (tokens,) int64 tensor on {dev}")
        for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
            _need(c.dim() == 4 and c.shape == k_cache.shape and c.shape[1] == k.shape[1] and c.shape[3] == d
                  and c.dtype == dt and c.device == dev and c.stride(3) == 1,
                  f"{name} must be a (pages, kv_heads, page_size, d) tensor of q's type with contiguous channels")
        a.v, a.v_stride, a.v_head_stride = v.data_ptr(), v.stride(0), v.stride(1)
        a.slot_map, a.k_cache, a.v_cache = slot_map.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
        a.k_page_stride, a.k_cache_head_stride, a.k_row_stride = k_cache.stride()[:3]
        a.v_page_stride, a.v_cache_head_stride, a.v_row_stride = v_cache.stride()[:3]
        a.page_size, a.num_slots = k_cache.shape[2], k_cache.shape[0] * k_cache.shape[2]
    elif k is not None:
        k_out = torch.empty((n, k.shape[1], d), dtype=dt, device=dev)
        a.k_out = k_out.data_ptr()
    a.tokens, a.d, a.rot, a.dtype = n, d, 2 * half, _TYPES[dt]
    a.adjacent, a.inverse = int(pairs == "adjacent"), int(inverse)
    _call(_lib.load().ea_rope_cuda, a, dev, "rope")
    return q_out, k_out


def rope(q, k, positions, inv_freq, *, axes=None, pairs: str = "half", inverse: bool = False):
    """Rotary positions (ea_rope_cuda): q (tokens, q_heads, d) and k (tokens, kv_heads, d), either may be
    None, any token and head strides (slices of a fused projection). Pair i is turned by
    positions[axes[i]] * inv_freq[i]: positions int32 (tokens,) or (axes, tokens), inv_freq float32
    (rot / 2,), axes int32 (rot / 2,) (from rope_axes; None: the first axis). pairs "half": channels i and
    i + rot / 2; "adjacent": 2 i and 2 i + 1; channels from rot on are copied. inverse turns back, which is
    also the gradient: with dq, dk of the outputs, rope(dq, dk, ..., inverse=True) gives those of the inputs.
    Returns new contiguous (q, k)."""
    return _rope(q, k, None, positions, inv_freq, axes, pairs, inverse, None, None, None)


def rope_append(q, k, v, positions, inv_freq, slot_map, k_cache, v_cache, *, axes=None, pairs: str = "half"):
    """rope, with the turned k and the v written to the paged caches (pages, kv_heads, page_size, d; any
    page, head and row strides) at rows slot_map (int64 (tokens,), from plan_step; -1 writes nothing).
    Slots of one call must differ. Returns the turned q."""
    return _rope(q, k, v, positions, inv_freq, axes, pairs, False, slot_map, k_cache, v_cache)[0]


def tree_mask(parents) -> np.ndarray:
    """Visibility rows for tree_attention of one draft tree: parents[i] < i is node i's parent, -1 for a child
    of the last accepted token; node i sees itself and its ancestors. (nodes, words) int32, bit j % 32 of
    word j // 32."""
    parents = np.asarray(parents, np.int64)
    n = len(parents)
    _need(n == 0 or (parents < np.arange(n)).all() and parents.min() >= -1, "a parent must come before its child")
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
    A token sees its sequence's earlier keys and, of the step's tokens, those whose bit is set in its row
    of tree_mask ((tokens, words) int32, see `tree_mask`); None: itself and the ones before it. Weights are
    2^(alpha q.k) (formats.default_alpha), as in `cuda.launch`. max_new (the most tokens of any sequence)
    only tunes tile sizes. Rows past q_start[batch] are not written. Returns out (tokens, q_heads, d), and
    with return_lse the log2 of the weights' sums (tokens, q_heads) float32; a row that sees no key gives 0
    and -inf. Values of keys that a row does not see cannot reach it. The result is not certified: it is the
    draft model's attention, accurate to its type's rounding."""
    dev, dt = q.device, q.dtype
    _need(dt in (torch.bfloat16, torch.float16), "tree_attention takes bfloat16 or float16")
    _need(q.dim() == 3 and q.stride(2) == 1, "q must be (tokens, q_heads, d) with contiguous channels")
    n, hq, d = q.shape
    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.shape[3] == d
          and k_cache.dtype == dt and v_cache.dtype == dt and k_cache.device == dev and v_cache.device == dev
          and k_cache.stride(3) == 1 and v_cache.stride(3) == 1,
          "caches must be (pages, kv_heads, page_size, d) tensors of q's type with contiguous channels")
    batch = seq_lens.shape[0]
    _need(page_table.dtype == torch.int32 and page_table.device == dev and page_table.dim() == 2
          and page_table.shape[0] == batch and (page_table.stride(1) == 1 or page_table.numel() <= batch),
          f"page_table must be a (batch, max_pages) int32 tensor on {dev} with contiguous rows")
    a = _lib.TreeAttentionArgs()
    a.seq_lens = _i32(seq_lens, "seq_lens", dev, None)
    a.q_start = _i32(q_start, "q_start", dev, batch + 1)
    if tree_mask is not None:
        a.tree_mask = _i32(tree_mask, "tree_mask", dev, n, None)
        a.mask_words = tree_mask.shape[1]
    if out is None:
        out = torch.empty((n, hq, d), dtype=dt, device=dev)
    else:
        _need(out.shape == q.shape and out.dtype == dt and out.device == dev and out.is_contiguous(),
              "out must be a contiguous tensor like q")
    lse = torch.empty((n, hq), dtype=torch.float32, device=dev) if return_lse else None
    a.q, a.q_stride, a.q_head_stride = q.data_ptr(), q.stride(0), q.stride(1)
    a.k_cache, a.v_cache, a.page_table, a.table_stride = (k_cache.data_ptr(), v_cache.data_ptr(),
                                                          page_table.data_ptr(), page_table.stride(0))
    a.k_page_stride, a.k_head_stride, a.k_row_stride = k_cache.stride()[:3]
    a.v_page_stride, a.v_head_stride, a.v_row_stride = v_cache.stride()[:3]
    a.out, a.lse = out.data_ptr(), None if lse is None else lse.data_ptr()
    a.tokens, a.num_pages, a.alpha = n, k_cache.shape[0], float(alpha)
    a.batch, a.q_heads, a.kv_heads, a.d = batch, hq, k_cache.shape[1], d
    a.page_size, a.max_pages, a.dtype = k_cache.shape[2], page_table.shape[1], _TYPES[dt]
    a.max_new = n if max_new is None else int(max_new)
    lib = _lib.load()
    if n and batch:
        if dev.type != "cuda":
            raise RuntimeError("tree_attention needs CUDA tensors (there is no CPU path)")
        size = lib.ea_tree_attention_workspace(ctypes.byref(a))
        if size < 0:
            _check(-1, "tree_attention")
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        a.workspace = ws.data_ptr()
    _call(lib.ea_tree_attention_cuda, a, dev, "tree_attention")
    return (out, lse) if return_lse else out


def process_logits(logits, row_seq=None, *, history=None, history_lens=None, prompt_lens=None, repetition=None,
                   frequency=None, presence=None, bias_ids=None, bias_values=None, allowed_bits=None, mask_rows=None,
                   draft_tokens=None, q_start=None, tree_mask=None, out=None):
    """Penalties, biases and grammar masks (ea_process_logits_cuda) on logits (rows, vocab) of bf16, fp16 or
    fp32; row r belongs to sequence row_seq[r] (int32; None: r; outside the batch: the row is copied).
    history (batch, width) int32 holds each sequence's tokens, the first prompt_lens[b] of its
    history_lens[b] being the prompt; draft_tokens (rows,) int32 with q_start (batch + 1,) and tree_mask (as
    for tree_attention; None: a chain) add the drafted tokens on each row's path. Then, in 32 bits and
    rounded once: tokens that occurred are divided (positive logits) or multiplied by repetition[b]; minus
    frequency[b] times the generated occurrences, minus presence[b] if there is one; plus bias_values (batch,
    entries) at bias_ids (int32, negative: unused); -inf where the token's bit of allowed_bits[mask_rows[r]]
    ((states, words) int32, bit v % 32 of word v // 32; mask_rows None: r, negative: unrestricted) is clear.
    Steps whose tensors are None are left out. Returns `out` (may be logits), or a new tensor."""
    dev = logits.device
    _need(logits.dtype in _TYPES, "process_logits takes bfloat16, float16 or float32")
    _need(logits.dim() == 2 and (logits.stride(1) == 1 or logits.shape[1] <= 1),
          "logits must be (rows, vocab) with contiguous rows")
    rows, vocab = logits.shape
    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=dev)
    else:
        _need(out.shape == logits.shape and out.dtype == logits.dtype and out.device == dev
              and (out.stride(1) == 1 or vocab <= 1), "out must be a tensor like logits with contiguous rows")
    batch = None
    for t in (history, repetition, frequency, presence, bias_ids):
        if t is not None:
            _need(batch is None or t.shape[0] == batch, "the sequences' tensors differ in length")
            batch = t.shape[0]
    if batch is None:
        batch = rows if q_start is None else q_start.shape[0] - 1
    _need(row_seq is not None or batch == rows, "without row_seq there must be one row a sequence")
    a = _lib.ProcessLogitsArgs()
    a.row_seq = _i32(row_seq, "row_seq", dev, rows)
    if history is not None:
        _need(history_lens is not None, "history needs history_lens")
        a.history = _i32(history, "history", dev, batch, None)
        a.history_stride = a.max_history = history.shape[1]
        a.history_lens = _i32(history_lens, "history_lens", dev, batch)
        a.prompt_lens = _i32(prompt_lens, "prompt_lens", dev, batch)
    a.repetition = _f32(repetition, "repetition", dev, batch)
    a.frequency = _f32(frequency, "frequency", dev, batch)
    a.presence = _f32(presence, "presence", dev, batch)
    if bias_ids is not None:
        _need(bias_values is not None, "bias_ids needs bias_values")
        a.bias_ids = _i32(bias_ids, "bias_ids", dev, batch, None)
        a.num_biases = bias_ids.shape[1]
        a.bias_values = _f32(bias_values, "bias_values", dev, batch, a.num_biases)
    if allowed_bits is not None:
        words = (vocab + 31) // 32
        a.allowed_bits = _i32(allowed_bits, "allowed_bits", dev, None, None)
        _need(allowed_bits.shape[1] >= words, f"allowed_bits needs {words} words a row")
        a.num_masks, a.mask_stride = allowed_bits.shape
        _need(mask_rows is not None or a.num_masks >= rows, "without mask_rows there must be one mask a row")
        a.mask_rows = _i32(mask_rows, "mask_rows", dev, rows)
    if draft_tokens is not None:
        _need(q_start is not None, "draft_tokens needs q_start")
        a.draft_tokens = _i32(draft_tokens, "draft_tokens", dev, rows)
        a.q_start = _i32(q_start, "q_start", dev, batch + 1)
        if tree_mask is not None:
            a.tree_mask = _i32(tree_mask, "tree_mask", dev, rows, None)
            a.tree_words = tree_mask.shape[1]
    a.logits, a.out, a.logits_stride, a.out_stride = logits.data_ptr(), out.data_ptr(), logits.stride(0), out.stride(0)
    a.rows, a.vocab, a.batch, a.dtype = rows, vocab, batch, _TYPES[logits.dtype]
    _call(_lib.load().ea_process_logits_cuda, a, dev, "process_logits")
    return out
