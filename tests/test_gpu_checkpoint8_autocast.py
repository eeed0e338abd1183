"""A checkpointed function that turns autocast on by itself, inside another region of it:
the casts of its forward, which records nothing, must not be found by later uses."""

import pytest
import torch

from redpanda_amd.checkpoint8 import hip_checkpoint8

pytestmark = pytest.mark.gpu
dev = "cuda"


def cast(**kw):
    return torch.autocast("cuda", dtype=torch.bfloat16, **kw)


@pytest.mark.parametrize("inner", [{}, {"cache_enabled": True}, {"cache_enabled": False}])
def test_a_function_with_autocast_of_its_own(gpu_lib, inner):
    d = 64
    torch.manual_seed(1)
    lin = torch.nn.Linear(d, d).to(dev)
    params = list(lin.parameters())
    x, dy = torch.randn(70, d, device=dev), torch.randn(70, d, device=dev).bfloat16()

    def fn(n):
        with cast(**inner):
            return lin(n)

    def own():
        return hip_checkpoint8(fn, x.clone().requires_grad_(True), out_dtype=torch.bfloat16, params=params)

    with cast():
        want = torch.autograd.grad(lin(x), params, dy)
    want_own = torch.autograd.grad(own(), params, dy)
    with cast():
        first, second = own(), lin(x)
        assert second.requires_grad
        got = torch.autograd.grad(second, params, dy)
        got_own = torch.autograd.grad(first, params, dy)
    for a, b in zip((*got, *got_own), (*want, *want_own)):
        assert torch.equal(a, b)


def test_casts_made_before_it_are_not_used_up(gpu_lib):
    """A weight that has a recorded cast in the cache already: both uses have their
    gradients, in one backward."""
    d = 48
    torch.manual_seed(2)
    lin = torch.nn.Linear(d, d).to(dev)
    params = list(lin.parameters())
    x, dy = torch.randn(30, d, device=dev), torch.randn(30, d, device=dev).bfloat16()

    def own():
        return hip_checkpoint8(lin, x.clone().requires_grad_(True), out_dtype=torch.bfloat16, params=params)

    with cast():
        a = torch.autograd.grad(lin(x), params, dy)
    with cast():
        b = torch.autograd.grad(own(), params, dy)
    with cast():
        both = (lin(x), own(), lin(x))
    got = torch.autograd.grad(both, params, (dy, dy, dy))
    for g, p, q in zip(got, a, b):
        # (2 p + q, in fp32, each as it is)
        assert bool(((g - (2 * p + q)).abs() <= 2.0 ** -7 * (2 * p.abs() + q.abs())).all())
