"""GPU parity of dropout with a recomputed mask, against the restatement in 64
bits (oracle/heads_ref.py): the mask element for element, the values within the
roundings of s x and of the sum."""

import pytest
import torch

from oracle import heads_ref as ref
from redpanda_amd.dropout import hip_dropout

pytestmark = pytest.mark.gpu
dev = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24  # half a step of fp32


def half_step(t):
    return torch.finfo(t).eps / 2


def check(y, x, res, keep, p):
    """y within the roundings of [res +] keep * s * x: s itself, s x and the sum
    in fp32, and the result's own."""
    dx = x.detach().cpu().double()
    prod = ref.drop(dx, p, keep)
    want = prod if res is None else prod + res.detach().cpu().double()
    tol = 3 * U * prod.abs() + U * want.abs() + half_step(y.dtype) * (1 + 8 * U) * want.abs()
    if y.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step below the normal range
    err = (y.detach().cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def make(rows, d, t, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (scale * torch.randn(rows, d, generator=g, device=dev)).to(t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("res_t", [None, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,d,p", [(5, 64, 0.1), (3, 1, 0.5), (37, 33, 0.2), (2, 1001, 0.05),
                                      (130, 384, 0.9)])
def test_values_mask_and_gradients(gpu_lib, rows, d, p, t, res_t):
    x = make(rows, d, t, rows + d).requires_grad_(True)
    res = None if res_t is None else make(rows, d, res_t, 7, 2.0).requires_grad_(True)
    seed = 0x1234567 * rows + (d << 40)
    keep = ref.keep_mask(range(rows), d, p, seed, stream=3)
    y = hip_dropout(x, p, seed, residual=res, stream=3)
    assert y.dtype == (t if res is None else torch.promote_types(t, res_t))
    check(y, x, res, keep, p)
    dy = make(rows, d, y.dtype, 9)
    y.backward(dy)
    assert x.grad.dtype == t
    check(x.grad, dy, None, keep, p)
    if res is not None:
        assert torch.equal(res.grad, dy.to(res_t))


@pytest.mark.parametrize("p", [0.0, 1e-6, 1.0])
def test_ends_of_p(gpu_lib, p):
    x, res = make(9, 40, torch.bfloat16, 1), make(9, 40, torch.float32, 2)
    check(hip_dropout(x, p, 5), x, None, ref.keep_mask(range(9), 40, p, 5), p)
    check(hip_dropout(x, p, 5, residual=res), x, res, ref.keep_mask(range(9), 40, p, 5), p)


def test_dropped_places_hide_inf_and_nan(gpu_lib):
    x = torch.full((4, 200), float("nan"), device=dev)
    x[1] = float("inf")
    keep = ref.keep_mask(range(4), 200, 0.5, 3)
    y = hip_dropout(x, 0.5, 3).cpu()
    assert bool((y[~keep] == 0).all()) and bool(torch.isnan(y[0][keep[0]]).all())
    assert bool(torch.isinf(y[1][keep[1]]).all())


def test_the_mask_is_the_seeds_streams_and_places(gpu_lib):
    """One mask for every dtype, stride, alignment and shape; another for another
    seed or stream, whether the seed comes by value or from the device."""
    ones = torch.ones(24, 6, 67, device=dev)
    a = hip_dropout(ones, 0.3, -77) != 0
    assert torch.equal(a.view(144, 67).cpu(), ref.keep_mask(range(144), 67, 0.3, -77))
    seed = torch.tensor([-77], device=dev)
    wide = torch.ones(144, 131, device=dev, dtype=torch.float16)
    for v in (wide[:, 1:68], wide[:, 64:], torch.ones(67, 144, device=dev).t(),
              torch.ones(1, 67, device=dev).expand(144, 67)):
        assert torch.equal(hip_dropout(v, 0.3, seed) != 0, a.view(144, 67))
    assert torch.equal(hip_dropout(torch.ones(67, device=dev), 0.3, seed) != 0, a[0, 0])
    assert not torch.equal(hip_dropout(ones, 0.3, -78) != 0, a)
    assert not torch.equal(hip_dropout(ones, 0.3, -77, stream=1) != 0, a)
    assert hip_dropout(torch.ones(0, 5, device=dev), 0.3, 1).shape == (0, 5)
    assert hip_dropout(torch.ones(5, 0, device=dev), 0.3, 1).shape == (5, 0)


def test_offsets_past_32_bits(gpu_lib):
    rows, d = (1 << 21) + 5, 1029  # 2.16e9 elements: offsets past 2^31, bytes past 2^32
    x = torch.ones(rows, d, dtype=torch.bfloat16, device=dev)
    y = hip_dropout(x, 0.5, 99)
    last = range(rows - 4, rows)
    keep = ref.keep_mask(last, d, 0.5, 99)
    assert torch.equal(y[-4:].cpu().double(), keep.double() * 2)
    share = float((y[::4099] != 0).double().mean())
    assert abs(share - 0.5) < 5 * 0.5 / (y[::4099].numel()) ** 0.5


def test_on_a_stream_of_its_own(gpu_lib):
    x = make(300, 768, torch.float32, 4)
    want = hip_dropout(x, 0.2, 8)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = hip_dropout(x, 0.2, 8)
    st.synchronize()
    assert torch.equal(got, want)


def test_captured_graph_draws_by_its_seed(gpu_lib):
    """Forward and backward in one graph; every replay against the eager result
    of the seed on the device, with eager work between the replays."""
    x = make(65, 200, torch.bfloat16, 4).requires_grad_(True)
    res, dy = make(65, 200, torch.float32, 5), make(65, 200, torch.float32, 6)
    seed = torch.tensor([1], device=dev)

    def step():
        y = hip_dropout(x, 0.3, seed, residual=res)
        return y, torch.autograd.grad(y, x, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for value in (1, 2, 3, 2):
        seed.fill_(value)
        graph.replay()
        got = [t.detach().clone() for t in out]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_a_seed_that_changes_before_the_backward_is_refused(gpu_lib):
    x = make(4, 16, torch.float32, 1).requires_grad_(True)
    seed = torch.tensor([5], device=dev)
    y = hip_dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def test_refusals(gpu_lib):
    x = make(4, 16, torch.float32, 1)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="p must"):
            hip_dropout(x, p, 1)
    with pytest.raises(ValueError, match="needs a seed"):
        hip_dropout(x, 0.1, None)
    for seed in (torch.tensor([1]), torch.tensor([1, 2], device=dev),
                 torch.tensor([1], device=dev, dtype=torch.int32)):
        with pytest.raises(ValueError, match="seed tensor"):
            hip_dropout(x, 0.1, seed)
    with pytest.raises(ValueError, match="residual"):
        hip_dropout(x, 0.1, 1, residual=x[:1])
    with pytest.raises(ValueError, match="residual"):
        hip_dropout(x, 0.1, 1, residual=x.cpu())
    with pytest.raises(TypeError, match="dtype"):
        hip_dropout(x.double(), 0.1, 1)
    with pytest.raises(TypeError, match="dtype"):
        hip_dropout(x, 0.1, 1, residual=x.double())
    with pytest.raises(ValueError, match="stream"):
        hip_dropout(x, 0.1, 1, stream=-1)
    with pytest.raises(ValueError, match="dimension"):
        hip_dropout(x[0, 0], 0.1, 1)
    y = hip_dropout(x.requires_grad_(True), 0.5, 1)
    (gx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), x)
