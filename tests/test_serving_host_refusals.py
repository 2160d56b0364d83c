"""What the serving operators refuse on the host, before any launch, beyond test_serving_host.py."""

import ctypes
import os
import subprocess
import sys

import pytest
import torch

from exactattention_b200 import _lib, build, serving


@pytest.mark.parametrize("off", [2, 4, 8, 24])
@pytest.mark.parametrize("name", ["q", "k_cache", "v_cache", "out", "workspace"])
def test_tree_attention_refuses_rows_off_16_byte_boundaries(cuda_lib, name, off):
    """The kernels load and store rows 8 and 16 bytes at a time. The addresses are made up: the call has to come
    back without a launch."""
    t = _lib.TreeAttentionArgs()
    t.tokens, t.batch, t.q_heads, t.kv_heads, t.d, t.page_size, t.max_pages, t.num_pages, t.max_new = 40, 1, 4, 2, 64, 16, 4, 4, 40
    t.q_stride, t.q_head_stride = 256, 64
    t.k_page_stride, t.k_head_stride, t.k_row_stride = 2048, 1024, 64
    t.v_page_stride, t.v_head_stride, t.v_row_stride = 2048, 1024, 64
    for i, f in enumerate(("q", "k_cache", "v_cache", "page_table", "seq_lens", "q_start", "out", "workspace")):
        setattr(t, f, (i + 1) << 20)
    setattr(t, name, getattr(t, name) + off)
    assert cuda_lib.ea_tree_attention_cuda(ctypes.byref(t), None) == -9
    assert b"16-byte" in cuda_lib.ea_serving_last_error()


def test_tree_attention_counts_the_tiles_of_the_kernel_it_takes(cuda_lib):
    """A prompt's chunk over a table wide enough for a million keys is 2^32 tiles of 8 rows x 64 keys, of which the kernel for
    few rows would have more than it can count, but 2^26 of the ones that it runs in."""
    t = _lib.TreeAttentionArgs()
    t.tokens, t.batch, t.q_heads, t.kv_heads, t.d, t.page_size, t.max_pages, t.num_pages = 32768, 1, 64, 8, 128, 16, 65536, 4
    t.max_new = 32768
    assert cuda_lib.ea_tree_attention_workspace(ctypes.byref(t)) >= 0
    t.max_new = 1
    assert cuda_lib.ea_tree_attention_workspace(ctypes.byref(t)) == -1
    assert b"2^31 tiles" in cuda_lib.ea_serving_last_error()


@pytest.mark.parametrize("call", [
    lambda x: serving.rope(x, None, torch.zeros(3, dtype=torch.int32), torch.zeros(32)),
    lambda x: serving.rope(torch.zeros(3, 2, 64), x, torch.zeros(3, dtype=torch.int32), torch.zeros(32)),
    lambda x: serving.rope(torch.zeros(3, 2, 64), None, torch.zeros(3, dtype=torch.int32), x[0, 0, :32]),
    lambda x: serving.tree_attention(x, torch.zeros(5, 2, 16, 64), torch.zeros(5, 2, 16, 64), torch.zeros(2, 4, dtype=torch.int32),
                                     torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), 0.1),
    lambda x: serving.process_logits(x[0]),
])
def test_tensors_that_require_grad_are_refused(cuda_lib, call):
    """No graph is recorded, so a gradient would be lost silently; without grad mode there is none to lose."""
    x = torch.zeros(3, 2, 64, requires_grad=True)
    with pytest.raises(ValueError, match="requires grad"):
        call(x)
    with torch.no_grad():
        try:
            call(x)
        except (RuntimeError, ValueError) as e:  # CPU tensors, or a type that the operator does not take
            assert "requires grad" not in str(e)


def test_a_binding_of_another_torch_is_not_used(cuda_lib, monkeypatch):
    """The binding uses torch's C++ ABI: after a change of torch it counts as stale, and is refused until it is rebuilt."""
    assert build._serving_native_current(build.SERVING_NATIVE)
    monkeypatch.setattr(torch, "__version__", "2.99.0")
    assert not build._serving_native_current(build.SERVING_NATIVE)
    monkeypatch.setattr(serving, "_mod", None)
    with pytest.raises(RuntimeError, match="this is 2.99.0"):
        serving._native()


def test_the_library_builds_without_torch(cuda_lib):
    """The certified entry points take numpy arrays and need no torch, and neither does their build."""
    code = ("import sys; sys.modules['torch'] = None\n"
            "import exactattention_b200\nfrom exactattention_b200 import _lib, build\n"
            "assert build.build() == build.OUT and _lib.load()\n")
    root = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stderr[-2000:]
    assert "no torch" in run.stderr
