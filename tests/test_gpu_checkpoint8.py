"""Checkpoints in 8 bits, and the backbone's fused training path.

A checkpointed layer's output is the plain layer's bit for bit; its gradients are those
of the plain layer on the values that 8 bits hold, for which the norm's kernels read
other bytes but do the same arithmetic."""

import pytest
import torch
import torch.utils.checkpoint

from redpanda_amd.checkpoint8 import hip_checkpoint8, hip_pack8, hip_unpack8
from redpanda_amd.mamba import Mamba, MambaConfig
from redpanda_amd.norm import hip_rmsnorm

pytestmark = pytest.mark.gpu
dev = "cuda"


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-30))


def branch(d, seed):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(d, 2 * d), torch.nn.GELU(), torch.nn.Linear(2 * d, d)).to(dev)


@pytest.mark.parametrize("with_add", [False, True])
@pytest.mark.parametrize("cast", [None, torch.bfloat16])
def test_layer_against_its_parts(gpu_lib, with_add, cast):
    d = 160
    fn = branch(d, 1)
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(5, 30, d, generator=g, device=dev)
    add = torch.randn(5, 30, d, generator=g, device=dev).to(cast or torch.float32) if with_add else None
    w = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
    ds, dy = torch.randn(5, 30, d, generator=g, device=dev), torch.randn(5, 30, d, generator=g, device=dev)
    params = list(fn.parameters())
    leaves = [t.clone().requires_grad_(True) for t in (x, add, w) if t is not None]

    def call(f, x, w, add, *rest):
        with torch.autocast("cuda", dtype=cast or torch.bfloat16, enabled=cast is not None):
            return f(x, w, add, *rest)

    def own(x, w, add):
        out = hip_checkpoint8(fn, x, w, add=add, out_dtype=cast or torch.float32, params=params)
        return out if add is not None else (None, out)

    lx, lw, la = leaves[0], leaves[-1], leaves[1] if with_add else None
    total, out = call(own, lx, lw, la)
    outs = (out,) if add is None else (total, out)
    dys = (dy.to(out.dtype),) if add is None else (ds, dy.to(out.dtype))
    got = torch.autograd.grad(outs, (*leaves, *params), dys)
    # the outputs: the plain layer's
    s = x if add is None else x + add
    plain = call(lambda s, w, _: fn(hip_rmsnorm(s, w, out_dtype=cast or torch.float32)), s, w, None)
    assert torch.equal(out, plain)
    if with_add:
        assert torch.equal(total, s)
    # the gradients: the plain layer's at the kept values
    held = hip_unpack8(hip_pack8(s)).requires_grad_(True)
    wl = w.clone().requires_grad_(True)
    at = call(lambda s, w, _: fn(hip_rmsnorm(s, w, out_dtype=cast or torch.float32)), held, wl, None)
    dh, dw, *dp = torch.autograd.grad(at, (held, wl, *params), dys[-1])
    full = dh if add is None else dh + ds
    # (the sum with ds is rounded inside in one, and outside in the other)
    assert rel(got[0], full) <= 2e-7
    if with_add:
        assert got[1].dtype == add.dtype and rel(got[1], full) <= (2e-7 if cast is None else 2 ** -8)
    assert torch.equal(got[len(leaves) - 1], dw)
    assert all(torch.equal(a, b) for a, b in zip(got[len(leaves):], dp))


def test_part_of_the_gradients_and_none(gpu_lib):
    d = 96
    fn = branch(d, 3)
    params = list(fn.parameters())
    x = torch.randn(20, d, device=dev)
    w = torch.ones(d, device=dev)
    out = hip_checkpoint8(fn, x, w, params=params)
    assert out.requires_grad
    full = torch.autograd.grad(out, params, torch.ones_like(out))
    params[0].requires_grad_(False)
    out = hip_checkpoint8(fn, x, w, params=params)
    got = torch.autograd.grad(out, params[1:], torch.ones_like(out))
    assert all(torch.equal(a, b) for a, b in zip(got, full[1:]))
    with torch.no_grad():
        assert not hip_checkpoint8(fn, x, w, params=params).requires_grad
    # only the sum is used: the branch is not run again
    xl = x.clone().requires_grad_(True)
    total, out = hip_checkpoint8(fn, xl, w, add=x, params=params)
    assert torch.equal(torch.autograd.grad(total, (xl,), torch.ones_like(total))[0], torch.ones_like(x))


def test_a_parameter_changed_in_between_is_refused(gpu_lib):
    d = 64
    fn = branch(d, 4)
    x = torch.randn(8, d, device=dev, requires_grad=True)
    out = hip_checkpoint8(fn, x, params=fn.parameters())
    with torch.no_grad():
        fn[0].weight.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


def make_model(seed=0, **kw):
    torch.manual_seed(seed)
    cfg = MambaConfig(d_model=96, n_layer=3, vocab_size=200, d_state=16, mimo_p=2, **kw)
    m = Mamba(cfg).to(dev)
    for layer in m.layers:
        layer["norm"].weight.data.add_(0.1 * torch.randn_like(layer["norm"].weight))
    return m


def grads(m, ids, dy, cast=None, **kw):
    m.zero_grad(set_to_none=True)
    with torch.autocast("cuda", dtype=cast or torch.bfloat16, enabled=cast is not None):
        y = m(ids, **kw)
    y.backward(dy)
    return y.detach(), {n: p.grad.clone() for n, p in m.named_parameters()}


@pytest.mark.parametrize("bidirectional", [False, True])
def test_fused_forward_is_the_plain_one(gpu_lib, bidirectional):
    """fp32: the same mathematics with the norm's and the table's sums in another order."""
    m = make_model(bidirectional=bidirectional)
    g = torch.Generator(device=dev).manual_seed(5)
    ids = torch.randint(0, 200, (4, 33), generator=g, device=dev)
    dy = torch.randn(4, 33, 96, generator=g, device=dev)
    y0, g0 = grads(m, ids, dy)
    y1, g1 = grads(m, ids, dy, fused=True)
    assert rel(y1, y0) <= 2e-6
    worst = max(rel(g1[n], g0[n]) for n in g0)
    assert worst <= 2e-5, worst
    with torch.no_grad():
        assert rel(m(ids, fused=True), y0) <= 2e-6
        x = torch.randn(2, 9, 96, generator=g, device=dev)
        assert rel(m(None, input_embeds=x, fused=True), m(None, input_embeds=x)) <= 2e-6


@pytest.mark.parametrize("cast", [None, torch.bfloat16])
@pytest.mark.parametrize("dropout", [0.0, 0.2])
def test_keep8_in_the_backbone(gpu_lib, cast, dropout):
    """The output is the fused path's bit for bit.  Each value kept is off by 1/128 of the
    largest of its 32 at most, a few thousandths of the rows' size, and so are the
    gradients: 8 roundings of that size may meet in one (three layers' input and norm,
    and what they pass on)."""
    m = make_model(1)
    g = torch.Generator(device=dev).manual_seed(6)
    ids = torch.randint(0, 200, (4, 40), generator=g, device=dev)
    dy = torch.randn(4, 40, 96, generator=g, device=dev)
    kw = dict(dropout=dropout, seed=3) if dropout else {}
    y0, g0 = grads(m, ids, dy, cast, fused=True, **kw)
    y1, g1 = grads(m, ids, dy, cast, keep8=True, **kw)
    assert torch.equal(y0, y1)
    worst = max(rel(g1[n], g0[n]) for n in g0)
    assert worst <= 8 / 128, worst


def test_fused_with_grad_checkpoint(gpu_lib):
    m = make_model(2)
    g = torch.Generator(device=dev).manual_seed(7)
    ids = torch.randint(0, 200, (3, 20), generator=g, device=dev)
    dy = torch.randn(3, 20, 96, generator=g, device=dev)
    y0, g0 = grads(m, ids, dy, fused=True)
    m.grad_checkpoint = True
    y1, g1 = grads(m, ids, dy, fused=True)
    assert torch.equal(y0, y1) and all(torch.equal(g0[n], g1[n]) for n in g0)


def test_embed_scale(gpu_lib):
    m = make_model(3)
    ids = torch.randint(0, 200, (2, 15), device=dev)
    x = (m.embedding(ids) * 3.0).detach()
    with torch.no_grad():
        assert rel(m(ids, fused=True, embed_scale=3.0), m(None, input_embeds=x, fused=True)) <= 1e-7
    with pytest.raises(ValueError, match="embed_scale"):
        m(ids, embed_scale=3.0)


def test_keep8_keeps_less(gpu_lib):
    """What is held between the passes: under a third of what fp32 checkpoints hold."""
    m = make_model(4)
    m.grad_checkpoint = True
    ids = torch.randint(0, 200, (64, 64), device=dev)

    def held(**kw):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = m(ids, **kw)
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated() - before - y.numel() * 4

    stream = 64 * 64 * 96 * 4
    plain, kept = held(), held(keep8=True)
    # plain: each layer's input, and norm_f's; kept: those in 8 bits, and norm_f's
    assert kept <= plain - 3 * stream * 0.7, (kept / stream, plain / stream)


def test_training_step_captured(gpu_lib):
    m = make_model(5)
    ids = torch.randint(0, 200, (4, 24), device=dev)
    dy = torch.randn(4, 24, 96, device=dev)
    params = list(m.parameters())

    def step():
        y = m(ids, keep8=True)
        return (y, *torch.autograd.grad(y, params, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [t.detach() for t in step()]
    for k in range(3):
        ids.copy_(torch.randint(0, 200, (4, 24), device=dev))
        dy.copy_(torch.randn(4, 24, 96, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        held = [t.detach().clone() for t in got]
        want = step()
        assert all(rel(a, b) <= 1e-5 for a, b in zip(held, want))


def test_weights_used_again_under_autocast(gpu_lib):
    """A weight that a checkpointed layer has cast for its forward, which records
    nothing, is cast anew where it is used with a graph, in a second layer or when the
    backward itself runs under autocast."""
    d = 64
    fn = branch(d, 3)
    g = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(70, d, generator=g, device=dev)
    dy = torch.randn(70, d, generator=g, device=dev).bfloat16()
    params = list(fn.parameters())

    def own():
        leaf = x.clone().requires_grad_(True)
        return hip_checkpoint8(fn, leaf, out_dtype=torch.bfloat16, params=params)

    def cast():
        return torch.autocast("cuda", dtype=torch.bfloat16)

    with cast():
        alone = own()
    want = torch.autograd.grad(alone, params, dy)
    with cast():
        plain = fn(x)
    want_plain = torch.autograd.grad(plain, params, dy)
    with cast():
        first, second = own(), fn(x)
        assert second.requires_grad
        got = torch.autograd.grad(first, params, dy)
        got_plain = torch.autograd.grad(second, params, dy)
    for a, b in zip((*got, *got_plain), (*want, *want_plain)):
        assert torch.equal(a, b)


def test_a_parameter_given_twice(gpu_lib):
    fn = branch(32, 5)
    x = torch.randn(9, 32, device=dev, requires_grad=True)
    params = list(fn.parameters())
    dy = torch.randn(9, 32, device=dev)
    want = torch.autograd.grad(hip_checkpoint8(fn, x, params=params), (x, *params), dy)
    got = torch.autograd.grad(hip_checkpoint8(fn, x, params=params + params[:2]), (x, *params), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_function_of_several_results_is_refused(gpu_lib):
    x = torch.randn(9, 32, device=dev)
    for leaf in (x, x.clone().requires_grad_(True)):
        with pytest.raises(TypeError, match="one tensor"):
            hip_checkpoint8(lambda n: (n, n * 2), leaf)


def test_embed_scale_of_given_embeddings_is_refused(gpu_lib):
    m = make_model(6)
    x = torch.randn(2, 15, 96, device=dev)
    for kw in ({}, {"fused": True}, {"keep8": True}):
        with pytest.raises(ValueError, match="embed_scale"):
            m(None, input_embeds=x, embed_scale=2.0, **kw)


def test_hooks_on_saved_tensors(gpu_lib):
    """Another checkpoint around it, or saved tensors kept on the host: the parameters'
    gradients are still found."""
    fn = branch(32, 7)
    x = torch.randn(9, 32, device=dev, requires_grad=True)
    params = list(fn.parameters())
    dy = torch.randn(9, 32, device=dev)

    def own(x):
        return hip_checkpoint8(fn, x, params=params)

    want = torch.autograd.grad(own(x), (x, *params), dy)
    y = torch.utils.checkpoint.checkpoint(own, x, use_reentrant=False)
    got = torch.autograd.grad(y, (x, *params), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.autograd.graph.save_on_cpu():
        y = own(x)
    got = torch.autograd.grad(y, (x, *params), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
