"""The embedding's gradient where a wave's share is 64 or 128 sorted places: more than 32
from 262144 places times kilobytes of a row on.  A row's gradient is a sum of n rows in
fp32 and one product, (n + 4) U sum |dy|, U = 2^-24, and the rounding to its type; the
expectation is summed in fp64."""

import pytest
import torch

from redpanda_amd.embedding import hip_embedding

pytestmark = pytest.mark.gpu
dev = "cuda"
U = 2.0 ** -24


def bordered(N, V, g):
    """Ids in V whose counts end shares of 64 and 128, pass them by one, or fill many; the
    last id of the table takes what is left."""
    counts = [64, 64, 128, 63, 1, 65, 127, 129, 1, 1, 126, 192, 320, 5, 59, 1000, 24, 3, 61]
    ids = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    rest = N - len(ids)
    some = torch.randint(len(counts), V, (rest // 3,), generator=g)
    ids = torch.cat((ids, some, torch.full((rest - len(some),), V - 1)))
    ids[torch.randperm(N, generator=g)[:N // 50]] = -1
    return ids[torch.randperm(N, generator=g)]


@pytest.mark.parametrize("N,d,t,share", [(70001, 1024, torch.float32, 64), (131072, 1024, torch.float32, 128),
                                         (9001, 16384, torch.bfloat16, 64), (20001, 16384, torch.float16, 128)])
def test_long_shares(gpu_lib, N, d, t, share):
    tiles = d * t.itemsize // 1024
    assert (share == 64) == (262144 <= N * tiles < 524288) and N * tiles >= 262144
    V = 150
    ids = bordered(N, V, torch.Generator().manual_seed(N)).to(dev)
    g = torch.Generator(device=dev).manual_seed(d)
    w = torch.randn(V, d, generator=g, device=dev).to(t).requires_grad_(True)
    dy = torch.randn(N, d, generator=g, device=dev).to(t)
    y = hip_embedding(ids, w)
    (dw,) = torch.autograd.grad(y, (w,), dy)
    assert torch.equal(y, torch.where((ids >= 0)[:, None], w.detach()[ids.clamp(min=0)], 0))
    fine = ids >= 0
    at, rows = ids[fine], dy[fine]
    n = torch.bincount(at, minlength=V)
    want = torch.zeros(V, d, dtype=torch.float64, device=dev).index_add_(0, at, rows.double())
    size = torch.zeros(V, d, dtype=torch.float64, device=dev).index_add_(0, at, rows.double().abs())
    tol = (n[:, None] + 4) * U * size
    tol = tol + torch.finfo(t).eps / 2 * (want.abs() + tol) + (2.0 ** -25 if t == torch.float16 else 0)
    assert bool(((dw.double() - want).abs() <= tol).all())
    assert torch.equal(dw, torch.autograd.grad(hip_embedding(ids, w), (w,), dy)[0])
