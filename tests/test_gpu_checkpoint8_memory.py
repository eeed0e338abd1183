"""What checkpointed layers hold between the passes, by themselves: 33 bytes for 32
values of each layer's input, where a checkpoint of an fp32 stream holds 128."""

import torch
import torch.utils.checkpoint

import pytest

from redpanda_amd.checkpoint8 import hip_checkpoint8
from redpanda_amd.norm import hip_rmsnorm

pytestmark = pytest.mark.gpu
dev = "cuda"


def test_a_third_of_a_checkpoint_in_fp32(gpu_lib):
    rows, d, layers = 8192, 256, 6
    torch.manual_seed(0)
    mats = [torch.randn(d, d, device=dev, requires_grad=True) for _ in range(layers)]
    x = torch.randn(rows, d, device=dev, requires_grad=True)

    def plain(x):
        for m in mats:
            x = x + torch.utils.checkpoint.checkpoint(lambda t, m=m: hip_rmsnorm(t) @ m, x, use_reentrant=False)
        return x

    def own(x):
        out = None
        for m in mats:
            got = hip_checkpoint8(lambda n, m=m: n @ m, x, add=out, params=(m,))
            x, out = (x, got) if out is None else got
        return x + out

    def held(f):
        f(x)  # (workspaces of the library's products are there from here on)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = f(x)
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated() - before - y.numel() * 4

    stream = rows * d * 4
    a, b = held(plain), held(own)
    # (the first layer's input is x itself, which no checkpoint adds)
    assert a >= (layers - 1) * stream
    # 33 / 128 of a stream for every layer, and some kilobytes for what is rounded up
    assert b <= layers * stream * 33 / 128 + layers * 2 ** 16
    assert b / layers <= a / (layers - 1) / 3
