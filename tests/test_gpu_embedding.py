"""GPU parity of the embedding and its gradient against the restatement in 64 bits
(oracle/train_ref.py).

With U = 2^-24: a row is one fp32 product (the scale itself is rounded to fp32), 2 U
|y|, and the rounding to its type; an id's gradient is a sum of n rows in fp32 and one
product by the scale, (n + 4) U |scale| sum |dy|, and the rounding to the table's
type."""

import pytest
import torch

from oracle import train_ref as ref
from redpanda_amd.embedding import hip_embedding

pytestmark = pytest.mark.gpu
dev = "cuda"
U = 2.0 ** -24
PAIRS = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float16)]


def to_type(v, t, bound):
    bound = bound + torch.finfo(t).eps / 2 * (v.abs() + bound)
    return bound + 2.0 ** -25 if t == torch.float16 else bound


def check(ids, w, scale, out_dtype, dy, padding_idx=None):
    w = w.detach().requires_grad_(True)
    y = hip_embedding(ids, w, scale=scale, out_dtype=out_dtype, padding_idx=padding_idx)
    assert y.shape == (*ids.shape, w.shape[1]) and y.dtype == out_dtype
    (dw,) = torch.autograd.grad(y, (w,), dy)
    d = w.shape[1]
    flat = ids.cpu().reshape(-1)
    want = ref.embedding(flat, w.detach().cpu(), scale)
    err = (y.detach().cpu().double().reshape(-1, d) - want).abs()
    assert bool((err <= to_type(want, out_dtype, 2 * U * want.abs())).all())
    dyc = dy.cpu().reshape(-1, d)
    want = ref.embedding(flat, w.detach().cpu(), scale, dyc, padding_idx)
    size = ref.embedding(flat, w.detach().cpu(), abs(scale), dyc.abs(), padding_idx)
    n = torch.zeros(w.shape[0], dtype=torch.float64)
    for v in flat.tolist():
        if 0 <= v < w.shape[0]:
            n[v] += 1
    tol = to_type(want, w.dtype, (n[:, None] + 4) * U * size)
    err = (dw.cpu().double() - want).abs()
    assert dw.dtype == w.dtype and bool((err <= tol).all()), float((err - tol).max())
    return y, dw


def make(N, V, d, tw, tout, seed, skew=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    w = torch.randn(V, d, generator=g, device=dev).to(tw)
    r = torch.rand(N, generator=g, device=dev)
    ids = (V * (r ** 4 if skew else r)).long().clamp(max=V - 1)
    ids = torch.where(torch.rand(N, generator=g, device=dev) < 0.05, -1, ids)
    return ids, w, torch.randn(N, d, generator=g, device=dev).to(tout)


@pytest.mark.parametrize("tw,tout", PAIRS)
@pytest.mark.parametrize("N,V,d", [(1, 1, 1), (5, 3, 7), (31, 40, 64), (32, 40, 100), (33, 7, 257),
                                   (64, 5, 33), (300, 50, 384), (700, 1000, 1001), (65, 4, 1030), (4097, 70, 6),
                                   (33000, 300, 12)])
def test_rows_and_gradient(gpu_lib, N, V, d, tw, tout):
    ids, w, dy = make(N, V, d, tw, tout, N * 100 + d)
    check(ids, w, 1.0, tout, dy)
    check(ids.to(torch.int32), w, 3.3, tout, dy)


def test_one_id_over_many_shares(gpu_lib):
    for N in (32, 33, 64, 1000, 4096):
        ids, w, dy = make(N, 9, 40, torch.float32, torch.float32, N)
        check(torch.full_like(ids, 4), w, 1.0, torch.float32, dy)
        two = torch.where(torch.arange(N, device=dev) < N // 2, 8, 0)
        check(two, w, 1.0, torch.float32, dy)


def test_borders_of_shares(gpu_lib):
    """Ids whose places end with a share, begin with one, or fill one."""
    for counts in ([32, 32, 32], [31, 1, 32, 33, 5], [64, 32, 1], [1] * 70, [96, 4], [16, 48, 31, 2, 31]):
        ids = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
        ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(1))].to(dev)
        g = torch.Generator(device=dev).manual_seed(len(counts))
        w = torch.randn(len(counts) + 3, 20, generator=g, device=dev)
        check(ids, w, 1.0, torch.float32, torch.randn(len(ids), 20, generator=g, device=dev))


@pytest.mark.parametrize("N", [3000, 50000])
def test_many_ids(gpu_lib, N):
    """More ids than 256 buckets have counters for."""
    g = torch.Generator(device=dev).manual_seed(5)
    V, d = 200003, 8
    w = torch.randn(V, d, generator=g, device=dev)
    ids = torch.randint(0, V, (N,), generator=g, device=dev)
    ids[::7] = V - 1
    dy = torch.randn(N, d, generator=g, device=dev)
    w.requires_grad_(True)
    (dw,) = torch.autograd.grad(hip_embedding(ids, w), (w,), dy)
    want = torch.zeros(V, d, dtype=torch.float64, device=dev).index_add_(0, ids, dy.double())
    size = torch.zeros(V, d, dtype=torch.float64, device=dev).index_add_(0, ids, dy.double().abs())
    assert bool(((dw.double() - want).abs() <= (N / 7 + 20) * U * size).all())


def test_ids_outside_the_table(gpu_lib):
    ids, w, dy = make(200, 30, 48, torch.float32, torch.float32, 8)
    ids[3], ids[50], ids[51], ids[199] = 30, 2 ** 40, -2 ** 40, 2 ** 32 + 5
    y, dw = check(ids, w, 2.0, torch.float32, dy)
    assert y.detach()[[3, 50, 51, 199]].abs().max() == 0
    none = torch.full((70,), -1, device=dev)
    y, dw = check(none, w, 1.0, torch.float32, dy[:70])
    assert dw.abs().max() == 0


def test_padding_idx(gpu_lib):
    ids, w, dy = make(500, 20, 33, torch.bfloat16, torch.bfloat16, 9)
    _, dw = check(ids, w, 1.0, torch.bfloat16, dy, padding_idx=0)
    assert dw[0].abs().max() == 0
    w = w.detach().requires_grad_(True)
    y = hip_embedding(ids, w, padding_idx=-20)
    assert torch.equal(torch.autograd.grad(y, (w,), dy)[0], dw)


def test_no_ids_and_shapes(gpu_lib):
    w = torch.randn(6, 10, device=dev, requires_grad=True)
    y = hip_embedding(torch.zeros(2, 0, dtype=torch.int64, device=dev), w)
    assert y.shape == (2, 0, 10)
    assert torch.autograd.grad(y, (w,), torch.zeros(2, 0, 10, device=dev))[0].abs().max() == 0
    assert hip_embedding(torch.tensor(3, device=dev), w).shape == (10,)
    ids = torch.randint(0, 6, (4, 5), device=dev)
    assert torch.equal(hip_embedding(ids.t(), w), w[ids.t()])
    assert torch.equal(hip_embedding(ids, w[:, ::2]), w[:, ::2][ids])


def test_strided_gradient_and_table(gpu_lib):
    g = torch.Generator(device=dev).manual_seed(11)
    big = torch.randn(40, 100, generator=g, device=dev)
    w = big[:, 3:70]
    ids = torch.randint(0, 40, (90,), generator=g, device=dev)
    dy = torch.randn(90, 201, generator=g, device=dev)[:, 7:74]
    check(ids, w, 1.0, torch.float32, dy)
    wl = w.detach().requires_grad_(True)
    y = hip_embedding(ids, wl)
    (dw,) = torch.autograd.grad(y, (wl,), torch.ones((), device=dev).expand(90, 67))
    n = torch.bincount(ids, minlength=40).float()
    assert torch.equal(dw, n[:, None].expand(40, 67))


def test_the_same_bits_each_time(gpu_lib):
    ids, w, dy = make(20000, 64, 256, torch.float32, torch.float32, 12)
    w.requires_grad_(True)
    got = [torch.autograd.grad(hip_embedding(ids, w), (w,), dy)[0] for _ in range(4)]
    assert all(torch.equal(got[0], g) for g in got[1:])


def test_captured_and_on_another_stream(gpu_lib):
    ids, w, dy = make(3000, 100, 128, torch.float32, torch.float32, 13)
    w = w.detach().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(hip_embedding(ids, w), (w,), dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = hip_embedding(ids, w)
        (dw,) = torch.autograd.grad(y, (w,), dy)
    for seed in range(3):
        new = make(3000, 100, 128, torch.float32, torch.float32, 20 + seed)
        ids.copy_(new[0])
        dy.copy_(new[2])
        graph.replay()
        torch.cuda.synchronize()
        we = w.detach().clone().requires_grad_(True)
        ye = hip_embedding(ids, we)
        assert torch.equal(y, ye)
        assert torch.equal(dw, torch.autograd.grad(ye, (we,), dy)[0])


def test_refusals(gpu_lib):
    w = torch.randn(6, 10, device=dev)
    ids = torch.zeros(3, dtype=torch.int64, device=dev)
    with pytest.raises(TypeError, match="ids"):
        hip_embedding(ids.float(), w)
    with pytest.raises(TypeError, match="ids"):
        hip_embedding(ids.to(torch.int16), w)
    with pytest.raises(ValueError, match="ids on cpu"):
        hip_embedding(ids.cpu(), w)
    with pytest.raises(ValueError, match="V, d"):
        hip_embedding(ids, w[0])
    with pytest.raises(ValueError, match="V, d"):
        hip_embedding(ids, w[:0])
    with pytest.raises(TypeError, match="dtype"):
        hip_embedding(ids, w.double())
    with pytest.raises(TypeError, match="dtype"):
        hip_embedding(ids, w, out_dtype=torch.int32)
    with pytest.raises(ValueError, match="padding_idx"):
        hip_embedding(ids, w, padding_idx=6)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(w, torch.ones_like(w))
        with pytest.raises((RuntimeError, NotImplementedError)):
            hip_embedding(ids, dual)


@pytest.mark.parametrize("V", [2 ** 22 + 3, 2 ** 27])
@pytest.mark.parametrize("N", [3000, 40000])
def test_tables_of_millions_of_rows(gpu_lib, V, N):
    """Buckets of up to 19 bits, of which many share the low eight."""
    g = torch.Generator(device=dev).manual_seed(8)
    d = 1
    w = torch.randn(V, d, generator=g, device=dev).bfloat16().requires_grad_(True)
    ids = torch.randint(0, V, (N,), generator=g, device=dev)
    ids[::5] = V - 1 - 256 * torch.randint(0, 40, (len(ids[::5]),), generator=g, device=dev)
    dy = torch.randint(-8, 9, (N, d), generator=g, device=dev).bfloat16()
    y = hip_embedding(ids, w)
    assert torch.equal(y, w[ids])
    (dw,) = torch.autograd.grad(y, (w,), dy)
    # (sums of small integers: exact in fp32, and rounded to bf16 once)
    want = torch.zeros(V, d, device=dev).index_add_(0, ids, dy.float()).bfloat16()
    assert torch.equal(dw, want)
