"""Rows in 8 bits at the top of each type's range: what was finite comes back finite.

A block whose largest magnitude m 2^k (1 <= m < 2) has m >= 127.5 / 64 is held in steps
of 2^(k - 5), in which that value is 64 (or 63.75 rounded up to it): 2^(k + 1), which is
beyond the type where k is its largest exponent.  Cut to the largest finite value, which
lies between the value and 2^(k + 1), it is nearer than half a step; everything else is
what the format holds, and has at most seven bits, so that no type rounds it again."""

import pytest
import torch

from oracle import train_ref as ref
from redpanda_amd.checkpoint8 import Packed8, hip_checkpoint8, hip_pack8, hip_unpack8
from redpanda_amd.norm import hip_rmsnorm

pytestmark = pytest.mark.gpu
dev = "cuda"
F, B, H = torch.float32, torch.bfloat16, torch.float16


def tops(rows, d, t, seed):
    """Rows whose blocks reach up to the type's largest value, of either sign."""
    g = torch.Generator(device=dev).manual_seed(seed)
    big = torch.finfo(t).max
    x = ((2 * torch.rand(rows, d, generator=g, device=dev) - 1).double() * big).to(t)
    x[:, 0], x[:, 1] = big, -big
    x[0, 2:] = 0
    if d > 34:
        x[:, 33] = -big
    return x


@pytest.mark.parametrize("t", [F, B, H])
@pytest.mark.parametrize("rows,d", [(1, 2), (5, 31), (4, 100), (3, 768)])
def test_finite_values_come_back_finite(gpu_lib, rows, d, t):
    x = tops(rows, d, t, rows + d)
    big = torch.finfo(t).max
    p = hip_pack8(x)
    q, e = ref.pack8(x.cpu())
    assert torch.equal(p.q.cpu(), q) and torch.equal(p.e.cpu(), e)
    back = hip_unpack8(p).cpu()
    assert bool(torch.isfinite(back).all())
    assert torch.equal(back.double(), ref.unpack8(q, e).clamp(-big, big))
    step = torch.pow(2.0, e.double() - 127).repeat_interleave(32, dim=1)[:, :d]
    assert bool(((back.double() - x.cpu().double()).abs() <= step / 2).all())
    # in another type: that value, rounded to it
    for out in (F, B, H):
        assert torch.equal(hip_unpack8(p, out).cpu(), back.to(out))


def test_infinities_and_nan_stay_nan(gpu_lib):
    x = tops(3, 64, H, 9)
    x[1, 40], x[2, 3] = float("inf"), float("nan")
    back = hip_unpack8(hip_pack8(x))
    assert torch.isnan(back[1, 32:]).all() and torch.isnan(back[2, :32]).all()
    assert torch.isfinite(back[0]).all() and torch.isfinite(back[1, :32]).all() and torch.isfinite(back[2, 32:]).all()


def test_packed_by_hand(gpu_lib):
    """Any q of any step below 255: finite in the type it says, and not cut in a wider one."""
    q = torch.tensor([[127, -127, 1, 0] * 8], dtype=torch.int8, device=dev)
    for e in (137, 138, 249, 254):
        p = Packed8(q, torch.tensor([[e]], dtype=torch.uint8, device=dev), H)
        value = q.double() * 2.0 ** (e - 127)
        for t in (H, B, F):
            big = torch.finfo(t).max
            p.dtype = t
            assert torch.equal(hip_unpack8(p).double(), value.clamp(-big, big).to(t).double())


@pytest.mark.parametrize("rows,d", [(7, 100), (3, 768), (2, 9000), (2, 20000)])
def test_the_gradient_at_kept_values(gpu_lib, rows, d):
    """fp16 rows clamped to the type's range: the gradient is that at the unpacked rows,
    which the kernels take with the same arithmetic."""
    x = tops(rows, d, H, d)
    g = torch.Generator(device=dev).manual_seed(1)
    w = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
    dy = torch.randn(rows, d, generator=g, device=dev).half()
    held = hip_unpack8(hip_pack8(x))
    got, want = [], []
    for rows_in, keep8, to in ((x, True, got), (held, False, want)):
        xl, wl = rows_in.clone().requires_grad_(True), w.clone().requires_grad_(True)
        to += torch.autograd.grad(hip_rmsnorm(xl, wl, keep8=keep8), (xl, wl), dy)
    assert all(bool(torch.isfinite(t).all()) for t in got)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a checkpointed layer's norm, computed again from 8 bits: its function's slope is
    # taken there
    xl, hl = x.clone().requires_grad_(True), held.clone().requires_grad_(True)
    a = torch.autograd.grad(hip_checkpoint8(lambda n: n * n, xl, w), (xl,), dy)[0]
    n = hip_rmsnorm(hl, w)
    b = torch.autograd.grad(n * n, (hl,), dy)[0]
    assert bool(torch.isfinite(a).all()) and torch.equal(a, b)
