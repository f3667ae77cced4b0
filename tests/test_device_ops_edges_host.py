"""Calls that the operators on device tensors refuse where a result would be wrong without a word, without a GPU."""
import pytest
import torch


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
