"""Mamba.forward(fused=True) and keep8=True take the settings of the modules that they
compute themselves into account."""

import pytest
import torch

from redpanda_amd.mamba import Mamba, MambaConfig

pytestmark = pytest.mark.gpu
dev = "cuda"


def make_model(seed=0, **kw):
    torch.manual_seed(seed)
    return Mamba(MambaConfig(d_model=64, n_layer=2, vocab_size=50, d_state=16, mimo_p=2, **kw)).to(dev)


def test_padding_idx_of_the_embedding(gpu_lib):
    m = make_model(1)
    m.embedding.padding_idx = 3
    ids = torch.randint(0, 50, (4, 12), device=dev)
    ids[:, :4] = 3
    dy = torch.randn(4, 12, 64, device=dev)
    for kw in ({}, dict(fused=True), dict(keep8=True)):
        m.zero_grad(set_to_none=True)
        m(ids, **kw).backward(dy)
        assert m.embedding.weight.grad[3].abs().max() == 0
        assert m.embedding.weight.grad.abs().max() > 0
