"""The training operators on buffers whose offsets pass 32 bits, in elements and in
bytes: the same bits as on compact copies."""

import pytest
import torch

from redpanda_amd.checkpoint8 import hip_pack8, hip_unpack8
from redpanda_amd.embedding import hip_embedding
from redpanda_amd.gated import hip_gated_scan
from redpanda_amd.norm import hip_rmsnorm

pytestmark = pytest.mark.gpu
dev = "cuda"
FAR = 2 ** 31 + 64  # elements between rows


def spread(t, far=FAR):
    """The rows of t (2-D) `far` elements apart in one buffer."""
    rows, d = t.shape
    buf = torch.empty((rows - 1) * far + d, dtype=t.dtype, device=dev)
    v = torch.as_strided(buf, (rows, d), (far, 1))
    v.copy_(t)
    return v


def test_rows_far_apart(gpu_lib):
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(3, 200, generator=g, device=dev).bfloat16()
    add, dy = (torch.randn(3, 200, generator=g, device=dev).bfloat16() for _ in range(2))
    w = torch.randn(200, generator=g, device=dev)
    far = spread(x)
    a, b = x.clone().requires_grad_(True), far.detach().requires_grad_(True)
    (s0, o0), (s1, o1) = hip_rmsnorm(a, w, add=add), hip_rmsnorm(b, w, add=spread(add))
    assert torch.equal(s0, s1) and torch.equal(o0, o1)
    g0, = torch.autograd.grad((s0, o0), (a,), (dy, dy))
    g1, = torch.autograd.grad((s1, o1), (b,), (spread(dy), spread(dy)))
    assert torch.equal(g0, g1)
    p0, p1 = hip_pack8(x), hip_pack8(far)
    assert torch.equal(p0.q, p1.q) and torch.equal(p0.e, p1.e)


def test_tables_and_gradients_far_apart(gpu_lib):
    g = torch.Generator(device=dev).manual_seed(2)
    w = torch.randn(3, 40, generator=g, device=dev).half()
    ids = torch.tensor([2, 0, 1], device=dev)
    dy = torch.randn(3, 40, generator=g, device=dev).half()
    a, b = w.clone().requires_grad_(True), spread(w).detach().requires_grad_(True)
    y0, y1 = hip_embedding(ids, a, scale=2.0), hip_embedding(ids, b, scale=2.0)
    assert torch.equal(y0, y1)
    assert torch.equal(torch.autograd.grad(y0, (a,), dy)[0], torch.autograd.grad(y1, (b,), spread(dy))[0])


def test_a_table_of_more_than_four_gigabytes(gpu_lib):
    V, d = 70000, 32768  # 2.3e9 elements
    w = torch.zeros(V, d, dtype=torch.bfloat16, device=dev)
    w[V - 1] = 1.5
    w[3] = -2.0
    w.requires_grad_(True)
    ids = torch.tensor([V - 1, 3, V - 1], device=dev)
    y = hip_embedding(ids, w)
    assert bool((y[0] == 1.5).all()) and bool((y[1] == -2.0).all()) and torch.equal(y[0], y[2])
    (dw,) = torch.autograd.grad(y, (w,), torch.ones_like(y))
    assert bool((dw[V - 1] == 2).all()) and bool((dw[3] == 1).all())
    assert int(torch.count_nonzero(dw[:3])) == 0 and int(torch.count_nonzero(dw[4:V - 1])) == 0


def test_rows_in_8_bits_beyond_four_gigabytes(gpu_lib):
    rows, d = 70000, 65537  # 4.6e9 elements, an odd width
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device=dev)
    x[-1, -1], x[-1, 0], x[40000, 7] = 3.0, -1.0, 0.5
    p = hip_pack8(x)
    back = hip_unpack8(p)
    del x
    assert back[-1, -1] == 3.0 and back[-1, 0] == -1.0 and back[40000, 7] == 0.5
    back[-1, -1] = back[-1, 0] = back[40000, 7] = 0
    assert not bool(back.any())


def test_states_far_apart(gpu_lib):
    g = torch.Generator(device=dev).manual_seed(3)

    def far(t):
        B, L, D = t.shape
        buf = torch.empty((B - 1) * FAR + L * D, dtype=t.dtype, device=dev)
        v = torch.as_strided(buf, (B, L, D), (FAR, D, 1))
        v.copy_(t)
        return v

    x, z, dy = (torch.randn(3, 40, 70, generator=g, device=dev).bfloat16() for _ in range(3))
    a = [t.clone().requires_grad_(True) for t in (x, z)]
    b = [far(t).detach().requires_grad_(True) for t in (x, z)]
    (y0, l0), (y1, l1) = hip_gated_scan(*a), hip_gated_scan(*b)
    assert torch.equal(y0, y1) and torch.equal(l0, l1)
    dl = torch.randn(3, 70, generator=g, device=dev)
    for p, q in zip(torch.autograd.grad((y0, l0), a, (dy, dl)), torch.autograd.grad((y1, l1), b, (far(dy), dl))):
        assert torch.equal(p, q)


def test_a_long_sequence_of_more_than_four_gigabytes(gpu_lib):
    L, D = 70000, 32768
    x = torch.zeros(1, L, D, dtype=torch.bfloat16, device=dev)
    z = torch.full((1, 1, D), float("inf"), dtype=torch.bfloat16, device=dev).repeat(1, L, 1)  # keeps
    x[0, 10], z[0, 10] = 2.0, float("-inf")  # takes
    x[0, L - 5], z[0, L - 5] = -3.0, float("-inf")
    y, last = hip_gated_scan(x, z)
    assert not bool(y[0, :10].any()) and bool((y[0, 10] == 2).all()) and bool((y[0, L - 6] == 2).all())
    assert bool((y[0, L - 5:] == -3).all()) and bool((last == -3).all())
