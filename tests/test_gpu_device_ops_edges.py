"""Operators on device tensors where magnitudes, masks and sizes are far from ordinary, against plain forms in 64 bits."""
import pytest
import torch

from test_gpu_device_ops import D, check_norm, normal  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("dtype,magnitude", [(torch.bfloat16, 1e20), (torch.bfloat16, 1e30), (torch.bfloat16, 1e-25), (torch.bfloat16, 1e-30), (torch.float32, 1e20), (torch.float32, 1e-25),
                                             (torch.float16, 4096.0), (torch.float16, 2.0**-14)])
@pytest.mark.parametrize("rows,hidden", [(2, 256), (300, 4096), (2, 257)])
def test_norm_of_rows_of_any_magnitude(D, dtype, magnitude, rows, hidden):  # noqa: F811
    """Squares leave the range of f32 while the rows and their norms are well inside it: the same in whole words and by elements."""
    w, eps = (1 + 0.2 * normal(7, hidden)).cuda(), 0.0
    x = (magnitude * normal(rows, rows, hidden)).to(dtype).cuda()
    check_norm(D, x, w, eps, None)
    check_norm(D, x, w, eps, (2 * magnitude * normal(3, rows, hidden)).to(dtype).cuda())
    odd = torch.empty(rows, hidden + 1, dtype=dtype, device="cuda")[:, 1:]
    odd.copy_(x)
    assert all(torch.equal(a, b) for a, b in zip(D.add_rms_norm_q8(x, w, eps)[:2], D.add_rms_norm_q8(odd, w, eps)[:2]))
