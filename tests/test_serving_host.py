"""The serving operators' host side without a GPU: C ABI, struct layouts, refusals, helpers."""

import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from exactattention_b200 import _lib, serving

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
HEADER = os.path.join(ROOT, "include", "exactattn_serving.h")


def test_library_exports_the_serving_header(cuda_lib):
    src = open(HEADER).read()
    names = set(re.findall(r"^\s*(?:int|int64_t|const char\*)\s+(ea_\w+)\s*\(", src, re.M))
    assert names == set(_lib.SERVING_EXPORTS)
    for n in names:
        assert hasattr(cuda_lib, n), n


@pytest.mark.parametrize("ctype,mirror", [("ea_plan_step_t", _lib.PlanStepArgs), ("ea_rope_t", _lib.RopeArgs),
                                          ("ea_tree_attention_t", _lib.TreeAttentionArgs),
                                          ("ea_process_logits_t", _lib.ProcessLogitsArgs)])
def test_struct_layout_matches_header(tmp_path, ctype, mirror):
    fields = [f[0] for f in mirror._fields_]
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "exactattn_serving.h"\nint main(void){'
                   f'printf("%zu", sizeof({ctype}));'
                   + "".join(f'printf(" %zu", offsetof({ctype}, {f}));' for f in fields) + "return 0;}\n")
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    vals = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    assert vals[0] == ctypes.sizeof(mirror)
    assert vals[1:] == [getattr(mirror, f).offset for f in fields]


def test_tree_mask_and_rope_axes():
    m = serving.tree_mask([-1, 0, 0, 1, -1])
    assert m[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10000]
    m = serving.tree_mask([i - 1 for i in range(40)])
    assert m.shape == (40, 2) and m[39].tolist() == [-1, 0xFF] and m[31].tolist() == [-1, 0]
    assert serving.tree_mask([]).shape == (0, 1)
    for bad in ([0], [-2], [-1, 1]):
        with pytest.raises(ValueError):
            serving.tree_mask(bad)
    assert serving.rope_axes([2, 3]).tolist() == [0, 0, 1, 1, 1]
    assert serving.rope_axes([3, 1, 2], interleaved=True).tolist() == [0, 1, 2, 0, 2, 0]


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _plan(**kw):
    a = dict(context_lens=_i(2), new_lens=_i(2), page_table=_i(2, 4), free_pages=_i(5), page_size=16, max_tokens=8)
    return serving.plan_step(**{**a, **kw})


def _rope(**kw):
    a = dict(q=torch.zeros(3, 4, 64), k=torch.zeros(3, 2, 64), positions=_i(3), inv_freq=torch.zeros(32))
    return serving.rope(**{**a, **kw})


def _attention(**kw):
    b = torch.bfloat16
    a = dict(q=torch.zeros(3, 4, 64, dtype=b), k_cache=torch.zeros(5, 2, 16, 64, dtype=b),
             v_cache=torch.zeros(5, 2, 16, 64, dtype=b), page_table=_i(2, 4), seq_lens=_i(2), q_start=_i(3), alpha=0.1)
    return serving.tree_attention(**{**a, **kw})


def _logits(**kw):
    return serving.process_logits(**{**dict(logits=torch.zeros(3, 50)), **kw})


def test_cpu_tensors_are_refused(cuda_lib):
    for f in (_plan, _rope, _attention, _logits):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            f()


@pytest.mark.parametrize("call", [
    lambda: _plan(page_size=0), lambda: _plan(max_tokens=-1), lambda: _plan(new_lens=_i(3)),
    lambda: _plan(page_table=_i(3, 4)), lambda: _plan(context_lens=torch.zeros(2, dtype=torch.int64)),
    lambda: _plan(depths=_i(7)), lambda: _plan(free_head=_i(2)), lambda: _plan(page_table=_i(4, 2).T),
    lambda: _rope(pairs="other"), lambda: _rope(q=None, k=None), lambda: _rope(k=torch.zeros(4, 2, 64)),
    lambda: _rope(k=torch.zeros(3, 2, 64, dtype=torch.float16)), lambda: _rope(inv_freq=torch.zeros(33)),
    lambda: _rope(positions=torch.zeros(3)), lambda: _rope(axes=_i(31)), lambda: _rope(positions=_i(2)),
    lambda: serving.rope_append(torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), _i(3), torch.zeros(32),
                                _i(3), torch.zeros(2, 2, 16, 64), torch.zeros(2, 2, 16, 64)),
    lambda: serving.rope_append(torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), _i(3), torch.zeros(32),
                                _i(3).long(), torch.zeros(2, 1, 16, 64), torch.zeros(2, 2, 16, 64)),
    lambda: _attention(q=torch.zeros(3, 4, 64)), lambda: _attention(q_start=_i(4)), lambda: _attention(tree_mask=_i(2, 1)),
    lambda: _attention(v_cache=torch.zeros(5, 2, 16, 32, dtype=torch.bfloat16)), lambda: _attention(page_table=_i(3, 4)),
    lambda: _attention(k_cache=torch.zeros(5, 2, 16, 64)), lambda: _attention(out=torch.zeros(3, 4, 64)),
    lambda: _logits(logits=torch.zeros(3, 50, dtype=torch.float64)), lambda: _logits(history=_i(3, 4)),
    lambda: _logits(repetition=torch.zeros(4)), lambda: _logits(repetition=torch.zeros(3), presence=torch.zeros(2)),
    lambda: _logits(bias_ids=_i(3, 2)), lambda: _logits(allowed_bits=_i(3, 1)), lambda: _logits(allowed_bits=_i(2, 2)),
    lambda: _logits(draft_tokens=_i(3)), lambda: _logits(out=torch.zeros(2, 50)), lambda: _logits(row_seq=_i(2)),
])
def test_wrong_arguments_are_refused(cuda_lib, call):
    with pytest.raises(ValueError):
        call()


def test_c_entries_refuse_without_a_launch(cuda_lib):
    """Sizes and layouts that the C entries turn away before they touch the GPU."""
    lib = cuda_lib
    p = _lib.PlanStepArgs()
    assert lib.ea_plan_step_cuda(None, None) == -1
    p.page_size, p.batch = 0, 1
    assert lib.ea_plan_step_cuda(ctypes.byref(p), None) == -1
    p.page_size, p.batch = 16, 20000
    assert lib.ea_plan_step_cuda(ctypes.byref(p), None) == -1
    assert b"EA_PLAN_MAX_SEQS" in lib.ea_serving_last_error()
    r = _lib.RopeArgs()
    r.tokens, r.q_heads, r.d, r.rot, r.num_axes = 1, 1, 64, 63, 1
    assert lib.ea_rope_cuda(ctypes.byref(r), None) == -1
    r.rot, r.d = 64, 9000
    assert lib.ea_rope_cuda(ctypes.byref(r), None) == -9
    r.d = 64
    assert lib.ea_rope_cuda(ctypes.byref(r), None) == -1  # no pointers
    r.tokens = 0
    assert lib.ea_rope_cuda(ctypes.byref(r), None) == 0
    t = _lib.TreeAttentionArgs()
    t.tokens, t.batch, t.q_heads, t.kv_heads, t.d, t.page_size = 1, 1, 3, 2, 64, 16
    assert lib.ea_tree_attention_cuda(ctypes.byref(t), None) == -1
    t.q_heads = 4
    for d in (4, 132, 256):
        t.d = d
        assert lib.ea_tree_attention_cuda(ctypes.byref(t), None) == -9
    t.d, t.dtype = 64, 2
    assert lib.ea_tree_attention_cuda(ctypes.byref(t), None) == -9
    t.dtype, t.batch = 0, 10000
    assert lib.ea_tree_attention_cuda(ctypes.byref(t), None) == -1
    t.batch, t.max_pages = 1, 1 << 30
    assert lib.ea_tree_attention_cuda(ctypes.byref(t), None) == -1
    g = _lib.ProcessLogitsArgs()
    g.rows, g.vocab, g.num_biases = 1, 10, 2001
    assert lib.ea_process_logits_cuda(ctypes.byref(g), None) == -1
    g.num_biases, g.max_history = 0, 1000001
    assert lib.ea_process_logits_cuda(ctypes.byref(g), None) == -1
    g.max_history = 0
    assert lib.ea_process_logits_cuda(ctypes.byref(g), None) == -1
    g.rows = 0
    assert lib.ea_process_logits_cuda(ctypes.byref(g), None) == 0
    assert not np.any(np.frombuffer(bytes(_lib.RopeArgs()), np.uint8))
