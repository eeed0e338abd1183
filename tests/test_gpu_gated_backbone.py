"""The training operators as one backbone: ids of packed sequences through the embedding,
layers of a norm, a projection, the gated recurrence and a projection back, and a last
norm; trained, checkpointed in 8 bits, and walked token by token.

Tolerances, relative in the 2-norm, in units of U = 2^-24: a layer rounds about 200 times
its own size at worst (two products over 48 and 40 terms, a mean over 48 squares, the
gate's exp and reciprocal, a recurrence whose errors its own gates average), so that two
layers, embedding and last norm stay below 512, and the gradients, which go over the
forward's results and back, below 2048."""

import pytest
import torch

from redpanda_amd.checkpoint8 import hip_checkpoint8
from redpanda_amd.embedding import hip_embedding
from redpanda_amd.gated import hip_gated_scan, hip_gated_step
from redpanda_amd.norm import hip_rmsnorm

pytestmark = pytest.mark.gpu
dev = "cuda"
U = 2.0 ** -24
V, D, H, B, L = 30, 48, 40, 3, 70
SCALE = D ** 0.5


def rel(a, b):
    return float((a.detach().double() - b.detach().double()).norm() / b.detach().double().norm())


def weights(layers=2):
    g = torch.Generator(device=dev).manual_seed(1)
    w = [torch.randn(V, D, generator=g, device=dev) * 0.2]
    for _ in range(layers):
        w += [1 + 0.1 * torch.randn(D, generator=g, device=dev),
              torch.randn(D, 2 * H, generator=g, device=dev) / D ** 0.5,
              torch.randn(H, D, generator=g, device=dev) / H ** 0.5]
    return w + [1 + 0.1 * torch.randn(D, generator=g, device=dev)]


def data():
    g = torch.Generator(device=dev).manual_seed(2)
    ids = torch.randint(0, V, (B, L), generator=g, device=dev)
    ids[0, 60:] = -1  # padding
    starts = torch.rand(B, L, generator=g, device=dev) < 0.05
    starts[0] = False
    return ids, starts, torch.randn(B, L, D, generator=g, device=dev)


def own(w, ids, starts, keep8):
    x, branch = hip_embedding(ids, w[0], scale=SCALE), None
    for k in range(1, len(w) - 1, 3):
        nw, w_in, w_out = w[k:k + 3]

        def mix(normed, w_in=w_in, w_out=w_out):
            v, gate = (normed @ w_in).split(H, -1)
            return hip_gated_scan(v, gate, starts=starts)[0] @ w_out

        if keep8:
            got = hip_checkpoint8(mix, x, nw, add=branch, params=(w_in, w_out))
            x, branch = (x, got) if branch is None else got
        else:
            got = hip_rmsnorm(x, nw, add=branch)
            x, normed = (x, got) if branch is None else got
            branch = mix(normed)
    return hip_rmsnorm(x, w[-1], add=branch)[1]


def plain(w, ids, starts):
    """The same in torch operations, in the weights' type."""
    def norm(x, nw):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * nw

    x = torch.where((ids >= 0)[..., None], w[0][ids.clamp(min=0)] * SCALE, 0.0)
    for k in range(1, len(w) - 1, 3):
        v, gate = (norm(x, w[k]) @ w[k + 1]).split(H, -1)
        a, h, ys = torch.sigmoid(gate), torch.zeros_like(v[:, 0]), []
        for t in range(L):
            h = torch.where(starts[:, t, None], 0.0, h)
            h = a[:, t] * h + (1 - a[:, t]) * v[:, t]
            ys.append(h)
        x = x + torch.stack(ys, 1) @ w[k + 2]
    return norm(x, w[-1])


def test_trained(gpu_lib):
    ids, starts, dy = data()
    w = [t.requires_grad_(True) for t in weights()]
    w64 = [t.detach().cpu().double().requires_grad_(True) for t in w]
    want = plain(w64, ids.cpu(), starts.cpu())
    want_g = torch.autograd.grad(want, w64, dy.cpu().double())
    y = own(w, ids, starts, False)
    got_g = torch.autograd.grad(y, w, dy)
    assert rel(y.cpu(), want) <= 512 * U
    for a, b in zip(got_g, want_g):
        assert rel(a.cpu(), b) <= 2048 * U
    # in 8 bits: the same results, and gradients at values off by up to 1/128 of the largest
    # of 32, which may meet in each of two layers twice, and in the norms
    y8 = own(w, ids, starts, True)
    got8 = torch.autograd.grad(y8, w, dy)
    assert torch.equal(y8, y)
    for a, b in zip(got8, got_g):
        assert rel(a, b) <= 6 / 128


def test_trained_in_a_graph(gpu_lib):
    ids, starts, dy = data()
    w = [t.requires_grad_(True) for t in weights()]

    def step():
        y = own(w, ids, starts, True)
        return [t.detach() for t in (y, *torch.autograd.grad(y, w, dy))]

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
        dy.copy_(torch.randn(B, L, D, device=dev))
        ids.copy_(torch.randint(-1, V, (B, L), device=dev))
        graph.replay()
        torch.cuda.synchronize()
        held = [t.clone() for t in got]
        for a, b in zip(held, step()):
            assert rel(a, b) <= 64 * U  # (the library's products may be others in a graph)


def test_walked_token_by_token(gpu_lib):
    ids, _, _ = data()
    w = weights()
    none = torch.zeros(B, L, dtype=torch.bool, device=dev)
    with torch.no_grad():
        want = own(w, ids, none, False)
        states = [None] * ((len(w) - 2) // 3)
        for t in range(L):
            x, branch = hip_embedding(ids[:, t], w[0], scale=SCALE), None
            for i, k in enumerate(range(1, len(w) - 1, 3)):
                got = hip_rmsnorm(x, w[k], add=branch)
                x, normed = (x, got) if branch is None else got
                v, gate = (normed @ w[k + 1]).split(H, -1)
                y, states[i] = hip_gated_step(v, gate, states[i])
                branch = y @ w[k + 2]
            out = hip_rmsnorm(x, w[-1], add=branch)[1]
            live = ids[:, t] >= 0
            assert rel(out[live], want[live, t]) <= 1024 * U
