"""Gated recurrences without a step, a sequence or a channel: they are part of the graph
like any other, and refuse tangents."""

import pytest
import torch

from redpanda_amd.gated import hip_gated_scan, hip_gated_step

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,D", [(0, 3, 6), (2, 0, 6), (2, 3, 0), (0, 0, 0)])
@pytest.mark.parametrize("state", [False, True])
def test_an_empty_batch_trains(gpu_lib, B, L, D, state, t):
    x, z = (torch.zeros(B, L, D, dtype=t, device=dev, requires_grad=True) for _ in range(2))
    h0 = torch.randn(B, D, device=dev, requires_grad=True) if state else None
    leaves = [v for v in (x, z, h0) if v is not None]
    y, last = hip_gated_scan(x, z, h0, torch.zeros(B, L, dtype=torch.bool, device=dev))
    assert y.shape == (B, L, D) and y.dtype == t and last.shape == (B, D) and last.dtype == torch.float32
    assert y.requires_grad and last.requires_grad
    assert torch.equal(last, torch.zeros(B, D, device=dev) if h0 is None else h0)
    dh = torch.randn(B, D, device=dev)
    grads = torch.autograd.grad((y, last), leaves, (torch.zeros_like(y), dh), retain_graph=True)
    assert all(g.shape == v.shape and g.dtype == v.dtype for g, v in zip(grads, leaves))
    if state and L == 0:
        assert torch.equal(grads[2], dh)
    (y.float().sum() + last.sum()).backward()
    assert x.grad.shape == x.shape and z.grad.shape == z.shape


def test_only_the_states_part(gpu_lib):
    x = torch.zeros(2, 0, 6, device=dev, requires_grad=True)
    h0 = torch.randn(2, 6, device=dev, requires_grad=True)
    y, _ = hip_gated_scan(x, x, h0)
    g = torch.autograd.grad(y.sum(), (x, h0), allow_unused=True)
    assert g[0].shape == x.shape and (g[1] is None or g[1].abs().max() == 0)


def test_a_step_of_no_rows(gpu_lib):
    x = torch.zeros(0, 5, device=dev, requires_grad=True)
    y, h = hip_gated_step(x, x)
    assert y.shape == (0, 5) and h.shape == (0, 5)
    y.sum().backward()
    assert x.grad.shape == (0, 5)
    with torch.no_grad():
        y, h = hip_gated_step(x, x)
    assert not y.requires_grad and not h.requires_grad


def test_tangents_are_refused(gpu_lib):
    e = torch.zeros(2, 0, 6, device=dev)
    h0 = torch.randn(2, 6, device=dev)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(h0, torch.ones_like(h0))
        with pytest.raises((RuntimeError, NotImplementedError)):
            hip_gated_scan(e, e, dual)
