"""The head operators under forward-mode differentiation, which they do not have:
a call that would lose a tangent is refused."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from redpanda_amd.dropout import hip_dropout
from redpanda_amd.layernorm import hip_layernorm

pytestmark = pytest.mark.gpu
dev = "cuda"


def test_tangents_are_refused(gpu_lib):
    x, t = (torch.randn(6, 40, device=dev) for _ in range(2))
    w = torch.ones(40, device=dev)
    calls = [lambda v: hip_dropout(v, 0.1, 3), lambda v: hip_dropout(x, 0.1, 3, residual=v),
             lambda v: hip_layernorm(v, w, w), lambda v: hip_layernorm(v, gelu=True, p=0.1, seed=1),
             lambda v: hip_layernorm(x, v[0], w), lambda v: hip_layernorm(x, w, v[0])]
    for grad in (True, False):
        with torch.set_grad_enabled(grad), fwad.dual_level():
            for call in calls:
                with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
                    call(fwad.make_dual(x, t))
                # without a tangent the same call goes through
                assert torch.equal(call(x), call(x.clone()))


def test_calls_at_a_level_without_tangents(gpu_lib):
    x = torch.randn(6, 40, device=dev)
    want = hip_layernorm(x, gelu=True), hip_dropout(x, 0.3, 1)
    with fwad.dual_level():
        assert torch.equal(hip_layernorm(x, gelu=True), want[0])
        assert torch.equal(hip_dropout(x, 0.3, 1), want[1])
        v = x.clone().requires_grad_(True)
        hip_dropout(v, 0.3, 1).sum().backward()
        assert torch.equal(v.grad != 0, want[1] != 0)
