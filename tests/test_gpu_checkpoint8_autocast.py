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


def test_captured_under_autocast(gpu_lib):
    d = 64
    torch.manual_seed(3)
    lin = torch.nn.Linear(d, d).to(dev)
    params = list(lin.parameters())
    x, dy = torch.randn(70, d, device=dev), torch.randn(70, d, device=dev).bfloat16()

    def step():
        with cast():
            leaf = x.detach().requires_grad_(True)
            first = hip_checkpoint8(lin, leaf, out_dtype=torch.bfloat16, params=params)
            out = first + lin(leaf)
        return [out.detach(), *torch.autograd.grad(out, (leaf, *params), dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(70, d, device=dev))
            dy.copy_(torch.randn(70, d, device=dev))
            lin.weight.mul_(1.01)
        graph.replay()
        torch.cuda.synchronize()
        held = [t.clone() for t in got]
        for a, b in zip(held, step()):
            # (the library's products in bf16 may be other ones in a graph: sums of 64 and 70
            # products in another order, rounded to bf16 at two places)
            assert float((a.double() - b.double()).norm() / b.double().norm()) <= 2 * 2.0 ** -8
