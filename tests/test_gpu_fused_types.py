"""Mamba.forward(fused=True) and keep8=True give a result of the plain path's type, for
streams of every type, with and without autocast."""

import pytest
import torch

from redpanda_amd.mamba import Mamba, MambaConfig

pytestmark = pytest.mark.gpu
dev = "cuda"


def make_model(seed=0, **kw):
    torch.manual_seed(seed)
    return Mamba(MambaConfig(d_model=64, n_layer=2, vocab_size=50, d_state=16, mimo_p=2, **kw)).to(dev)


@pytest.mark.parametrize("cast", [None, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", [dict(fused=True), dict(keep8=True), dict(fused=True, dropout=0.25, seed=5)])
def test_the_type_of_the_plain_path(gpu_lib, kw, t, cast):
    m = make_model()
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(2, 9, 64, generator=g, device=dev).to(t)
    plain = {k: v for k, v in kw.items() if k not in ("fused", "keep8")}
    with torch.no_grad(), torch.autocast("cuda", dtype=cast or torch.bfloat16, enabled=cast is not None):
        want = m(None, input_embeds=x, **plain)
        got = m(None, input_embeds=x, **kw)
    assert got.dtype == want.dtype
    # the streams' additions are rounded alike; norms in 16 bits are rounded in other places
    coarse = max(torch.finfo(v).eps for v in (t, cast or torch.float32))
    assert float((got.double() - want.double()).norm() / want.double().norm()) <= 16 * coarse
