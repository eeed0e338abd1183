"""Tables without columns: empty rows, and an empty gradient, as torch's embedding."""

import pytest
import torch

from redpanda_amd.embedding import hip_embedding

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(), (3,), (2, 0), (4, 5)])
def test_no_columns(gpu_lib, shape, t):
    w = torch.zeros(7, 0, dtype=t, device=dev, requires_grad=True)
    ids = torch.zeros(shape, dtype=torch.int64, device=dev)
    with torch.no_grad():
        assert hip_embedding(ids, w).shape == (*shape, 0)
    y = hip_embedding(ids, w, scale=2.0, out_dtype=torch.float16)
    assert y.shape == (*shape, 0) and y.dtype == torch.float16 and y.requires_grad
    (dw,) = torch.autograd.grad(y, (w,), torch.zeros_like(y))
    assert dw.shape == w.shape and dw.dtype == t
