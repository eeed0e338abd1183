"""Mamba.forward(fused=True) and keep8=True compute the embedding and the norms from
their weights: what these modules would do beyond that is refused, not left out."""

import pytest
import torch
from torch import nn

from redpanda_amd.mamba import Mamba, MambaConfig, RMSNorm


def make_model():
    torch.manual_seed(0)
    return Mamba(MambaConfig(d_model=32, n_layer=2, vocab_size=50, d_state=16, mimo_p=2))


class Shifted(RMSNorm):
    def forward(self, x):
        return super().forward(x) + 1


def replaced_norm(m):
    m.layers[1]["norm"] = nn.LayerNorm(32)


def replaced_last(m):
    m.norm_f = nn.Identity()


def derived_norm(m):
    m.layers[0]["norm"] = Shifted(32)


def own_forward(m):
    m.layers[0]["norm"].forward = lambda x: x


def hooked_norm(m):
    m.layers[0]["norm"].register_forward_hook(lambda mod, a, out: out * 2)


def pre_hooked_norm(m):
    m.norm_f.register_forward_pre_hook(lambda mod, a: a)


def backward_hooked_norm(m):
    m.norm_f.register_full_backward_hook(lambda mod, a, b: None)


def hooked_embedding(m):
    m.embedding.register_forward_hook(lambda mod, a, out: out)


def replaced_embedding(m):
    m.embedding = nn.Sequential(nn.Embedding(50, 32))


def max_norm(m):
    m.embedding.max_norm = 1.0


def by_frequency(m):
    m.embedding.scale_grad_by_freq = True


def sparse(m):
    m.embedding.sparse = True


@pytest.mark.parametrize("kw", [dict(fused=True), dict(keep8=True)])
@pytest.mark.parametrize("change", [
    replaced_norm, replaced_last, derived_norm, own_forward, hooked_norm, pre_hooked_norm,
    backward_hooked_norm, hooked_embedding, replaced_embedding, max_norm, by_frequency, sparse])
def test_other_modules_are_refused(change, kw):
    m = make_model()
    change(m)
    ids = torch.zeros(1, 4, dtype=torch.int64)
    with pytest.raises(ValueError, match="fused"):
        m(ids, **kw)


@pytest.mark.parametrize("kw", [dict(fused=True), dict(keep8=True)])
@pytest.mark.parametrize("change", [hooked_embedding, replaced_embedding, max_norm])
def test_the_embedding_is_not_looked_at_where_none_is_made(change, kw):
    m = make_model()
    change(m)
    # (the kernels then refuse host tensors)
    with pytest.raises(RuntimeError, match="device"):
        m(None, input_embeds=torch.zeros(1, 4, 32), **kw)
