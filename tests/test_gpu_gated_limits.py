"""More sequences than a launch holds are refused in the same words whether or not a
gradient is wanted."""

import pytest
import torch

from redpanda_amd.gated import hip_gated_scan

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.mark.parametrize("grad", [False, True])
def test_too_many_sequences(gpu_lib, grad):
    x = torch.zeros(2 ** 23 + 1, 1, 1, dtype=torch.bfloat16, device=dev, requires_grad=grad)
    with pytest.raises(RuntimeError, match="too many channels"):
        hip_gated_scan(x, x)
