"""Calls that the operators on device tensors refuse where a result would be wrong without a word, without a GPU."""
import ctypes as C
import math
import os
import subprocess
import sys

import pytest
import torch

from test_device_ops_host import AT, pages, refused


@pytest.fixture(scope="module")
def D(b200):
    from llama_gguf_b200 import device_ops

    return device_ops


def test_forward_tangents_are_refused(b200, D):
    """Results carry no tangent either: dropping one would make a derivative zero."""
    import torch.autograd.forward_ad as fw

    x, w = torch.zeros(4, 64), torch.ones(64)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for args in ((dual, w), (x, fw.make_dual(w, w))):
            with pytest.raises(b200.Unsupported, match="tangent"):
                D.add_rms_norm_q8(*args, 1e-5)
        with pytest.raises(b200.InvalidArgument, match="CUDA"):
            D.add_rms_norm_q8(fw.unpack_dual(dual).primal, w, 1e-5)


def test_scales_that_are_no_f32_numbers_are_refused(b200, D):
    """The scale is f32: what is a number in 64 bits may be infinite there, and results NaN."""
    for scale in (math.inf, -math.inf, math.nan, 1e300):
        a = D.Q4Attention(device=0, type=0, q=AT, out=AT, q_token=256, q_head=64, out_token=256, out_head=64, kv_lens=AT, page_table=AT, table_stride=4, tokens=3, table_pages=4, seqs=3,
                          n_heads=4, scale=scale, cache=pages(D))
        refused(b200, D._lib().b200_dev_attention_paged_q4(C.byref(a)), b200.InvalidArgument, "scale")
        with pytest.raises(b200.InvalidArgument, match="scale"):
            D.attention_paged_q4(torch.zeros(3, 4, 64), D.q4_pages(4, 2, 64, 16, device="cpu"), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), scale)


def test_views_of_the_negative_are_refused(b200, D):
    """A view whose negative bit is set (imag of a conjugate, taken on) has the other sign in memory."""
    x = torch.randn(4, 64)
    view = torch._neg_view(x)
    assert view.is_neg() and torch.equal(view, -x)
    with pytest.raises(b200.Unsupported, match="negative"):
        D.add_rms_norm_q8(view, torch.ones(64), 1e-5)
    with pytest.raises(b200.InvalidArgument, match="CUDA"):
        D.add_rms_norm_q8(view.resolve_neg(), torch.ones(64), 1e-5)


def test_every_plan_of_products_is_tested(D):
    """The plans that calls of all sizes have are those of the tests' list."""
    import random

    from test_gpu_device_ops_edges import PLANS

    assert all(D.i8_plan(t, k, n) == plan for plan, t, k, n in PLANS)
    rng, seen = random.Random(1), set()
    for _ in range(20000):
        seen.add(D.i8_plan(*(int(2 ** rng.uniform(0, m)) for m in (13, 14, 15))))
    assert seen <= {p[0] for p in PLANS}


def test_the_library_builds_without_torch_and_the_calls_again_for_another_one(tmp_path):
    csrc = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "llama-gguf_b200", "csrc")

    def steps(*args):
        return subprocess.run(["make", "-n", "-C", csrc, "OBJDIR=" + str(tmp_path), *args], capture_output=True, text=True, check=True).stdout

    without = steps(f"PYTHON={sys.executable} -S")      # (no site-packages)
    assert "device_ops.cu" in without and "device_ops_py.cpp" not in without and "not built" in without
    built = os.path.join(csrc, "..", "_device_ops.so")
    known = tmp_path / "torch.txt"
    assert not known.exists()
    if "device_ops_py.cpp" not in steps(f"PYTHON={sys.executable}"):
        pytest.skip("torch without headers")
    assert torch.__version__ in known.read_text()
    if os.path.exists(built):
        os.utime(known, (0, 0))
        assert "device_ops_py.cpp" not in steps(f"PYTHON={sys.executable}")
        known.write_text("another one")
        assert "device_ops_py.cpp" in steps(f"PYTHON={sys.executable}")


def test_which_kernel_attention_takes(D):
    """By the rows of a call, the keys that its table or its window has room for, and what the host says of the longest sequence."""
    def blocks(tokens, seqs=1, keys=4096, nh=32, nkv=8, max_q=0, window=0, starts=1):
        a = D.Q4Attention(type=0, q_starts=starts, kv_lens=1, page_table=1, table_stride=keys // 16, tokens=tokens, table_pages=keys // 16, seqs=seqs, n_heads=nh, scale=1.0, max_q=max_q, window=window,
                          cache=D.Q4Pages(data=16, n_pages=4, page_size=16, n_kv_heads=nkv, head_dim=64))
        n = C.c_int64(-1)
        assert D._lib().b200_debug_q4_prompt_blocks(C.byref(a), C.byref(n)) == 0
        return n.value

    assert blocks(2048) == (2048 * 4 // 128 + 1) * 8
    assert not blocks(64) and blocks(96)
    assert not blocks(48, keys=2048) and blocks(48, keys=512)
    assert blocks(48, keys=65536, window=100) and not blocks(48, keys=65536)
    assert not blocks(2048, max_q=8) and not blocks(512, seqs=512, starts=None)
    assert not blocks(8)
