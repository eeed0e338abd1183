"""GPU parity of layer norm (with GELU and dropout) and its backward pass against
the restatement in 64 bits (oracle/heads_ref.py).

Tolerances count the kernels' fp32 roundings, U = 2^-24 each.  A row's sums are
chains of at most CHAIN additions.  With h the normalised input's source (GELU(x)
or x), its error eh = 10 U |x| with GELU (the fit's 2e-8, an exponential whose
argument x^2/2 is rounded, a polynomial of degree 6) and 0 without, r the inverse
standard deviation:
    mean:   em = CHAIN U mean|h| + max eh
    xh:     ex = r (eh + em + 2 U |h - mean|) + |xh| (CHAIN U + r max eh)
    out:    (ex + 3 U |xh|) |w| + 2 U |y|, times the dropout's scale, and the
            rounding to the output's type
and for the gradient, q = g w, with m1 = mean q and m2 = mean(q xh):
    m2:     e2 = mean(|q| ex) + CHAIN U mean|q xh|
    dx:     r (CHAIN U (|q| + mean|q|) + ex |m2| + |xh| e2) slope
            + |dx| (CHAIN U + r max eh) + r |..| 10 U (1 + |x|), and its rounding
    dw:     sum |g| ex + (rows + 4) U sum |g xh|;  db: (rows + 4) U sum |g|
"""

import pytest
import torch
import torch.nn.functional as F

from oracle import heads_ref as ref
from redpanda_amd.layernorm import hip_layernorm

pytestmark = pytest.mark.gpu
dev = "cuda"
U = 2.0 ** -24
CHAIN = 64
PAIRS = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
         (torch.float16, torch.float32), (torch.float32, torch.bfloat16)]


def make(rows, d, tx, tout, seed, mean=0.3):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, d, generator=g, device=dev) + mean * torch.randn(rows, 1, generator=g, device=dev)
    w = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
    b = 0.1 * torch.randn(d, generator=g, device=dev)
    dy = torch.randn(rows, d, generator=g, device=dev).to(tout)
    return x.to(tx), w, b, dy


def to_type(v, t, bound):
    """The tolerance of v with its rounding to type t."""
    bound = bound + torch.finfo(t).eps / 2 * (v.abs() + bound)
    return bound + 2.0 ** -25 if t == torch.float16 else bound


def check_all(x, w, b, dy, out, grads, eps, gelu, p, keep):
    """out and (dx, dw, db) (any may be None) within the bounds above."""
    rows, d = x.shape
    x64 = x.detach().cpu().double().requires_grad_(True)
    w64 = (torch.ones(d) if w is None else w.detach().cpu()).double().requires_grad_(True)
    b64 = (torch.zeros(d) if b is None else b.detach().cpu()).double().requires_grad_(True)
    y64 = ref.layernorm(x64, w64, b64, eps, gelu, p, keep)
    s = 1.0 if keep is None else ref.drop_scale(p)
    with torch.no_grad():
        h = ref.gelu(x64) if gelu else x64
        eh = 10 * U * x64.abs() if gelu else torch.zeros_like(h)
        ehm = eh.amax(-1, keepdim=True)
        c = h - h.mean(-1, keepdim=True)
        r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
        xh = c * r
        em = CHAIN * U * h.abs().mean(-1, keepdim=True) + ehm
        er = CHAIN * U + r * ehm
        ex = r * (eh + em + 2 * U * c.abs()) + xh.abs() * er
        full = s * (xh * w64 + b64)
        tol = s * (ex + 3 * U * xh.abs()) * w64.abs() + 3 * U * full.abs()
        tol = tol if keep is None else torch.where(keep, tol, 0.0)
        err = (out.detach().cpu().double() - y64).abs()
        tol = to_type(y64, out.dtype, tol)
        assert bool((err <= tol).all()), ("out", float((err / (tol + 1e-300)).max()))
    if grads is None:
        return
    dx64, dw64, db64 = torch.autograd.grad(y64, (x64, w64, b64), dy.detach().cpu().double())
    with torch.no_grad():
        g = dy.detach().cpu().double()
        g = g if keep is None else ref.drop(g, p, keep)
        q = g * w64
        m2 = (q * xh).mean(-1, keepdim=True)
        e2 = (q.abs() * ex).mean(-1, keepdim=True) + CHAIN * U * (q * xh).abs().mean(-1, keepdim=True)
        slope, es = torch.ones_like(x64), torch.zeros_like(x64)
        if gelu:
            slope = 0.5 * torch.erfc(-x64 / 2 ** 0.5) + x64 * torch.exp(-x64 * x64 / 2) / (2 * torch.pi) ** 0.5
            es = 10 * U * (1 + x64.abs())
        inner = q - q.mean(-1, keepdim=True) - xh * m2
        tx = r * (CHAIN * U * (q.abs() + q.abs().mean(-1, keepdim=True)) + ex * m2.abs() + xh.abs() * e2)
        tx = tx * slope.abs() + dx64.abs() * er + r * inner.abs() * es
        tw = (g.abs() * ex).sum(0) + (rows + 4) * U * (g * xh).abs().sum(0)
        tb = (rows + 4) * U * g.abs().sum(0)
        for name, got, want, tol in (("dx", grads[0], dx64, tx), ("dw", grads[1], dw64, tw),
                                     ("db", grads[2], db64, tb)):
            if got is None:
                continue
            err = (got.detach().cpu().double() - want).abs()
            tol = to_type(want, got.dtype, tol + 1e-30)
            assert bool((err <= tol).all()), (name, float((err / tol).max()))


def run(x, w, b, dy, gelu, p, seed, tout, eps=1e-5, stream=0):
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = hip_layernorm(x, w, b, eps, gelu=gelu, p=p, seed=seed, out_dtype=tout, stream=stream)
    assert y.dtype == tout and y.shape == x.shape
    g = dict(zip(map(id, leaves), torch.autograd.grad(y, leaves, dy)))
    return y, [g.get(id(t)) for t in (x, w, b)]


@pytest.mark.parametrize("tx,tout", PAIRS)
@pytest.mark.parametrize("gelu,p", [(False, 0.0), (True, 0.0), (True, 0.2)])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 5), (2, 64), (33, 100), (17, 384), (5, 768), (9, 1001),
                                    (130, 257)])
def test_forward_and_gradients(gpu_lib, rows, d, gelu, p, tx, tout):
    x, w, b, dy = make(rows, d, tx, tout, rows * 1000 + d)
    y, grads = run(x, w, b, dy, gelu, p, 42, tout)
    keep = ref.keep_mask(range(rows), d, p, 42) if p else None
    check_all(x, w, b, dy, y, grads, 1e-5, gelu, p, keep)
    with torch.no_grad():  # the call without a graph gives the same bits
        assert torch.equal(hip_layernorm(x, w, b, gelu=gelu, p=p, seed=42, out_dtype=tout), y)


@pytest.mark.parametrize("d", [8, 63, 64, 65, 127, 129, 256, 511, 512, 513, 1023, 1024, 1025, 1536, 1537,
                               2047, 2048, 2049, 2560, 4095, 4097, 8191, 8192, 8193, 9000, 16391])
@pytest.mark.parametrize("tx", [torch.float32, torch.bfloat16])
def test_every_width_of_a_row(gpu_lib, d, tx):
    x, w, b, dy = make(21, d, tx, tx, d)
    y, grads = run(x, w, b, dy, True, 0.1, 7, tx)
    check_all(x, w, b, dy, y, grads, 1e-5, True, 0.1, ref.keep_mask(range(21), d, 0.1, 7))


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 63, 65, 257, 1031, 4099])
@pytest.mark.parametrize("d", [40, 384, 1000])
def test_every_number_of_rows(gpu_lib, rows, d):
    x, w, b, dy = make(rows, d, torch.bfloat16, torch.float32, rows)
    y, grads = run(x, w, b, dy, True, 0.1, 7, torch.float32)
    check_all(x, w, b, dy, y, grads, 1e-5, True, 0.1, ref.keep_mask(range(rows), d, 0.1, 7))


def test_rows_far_from_zero(gpu_lib):
    """A mean of 1000 standard deviations: a variance from squares would be lost."""
    x, w, b, dy = make(6, 768, torch.float32, torch.float32, 5, mean=0.0)
    x = x + 1000.0
    y, grads = run(x, w, b, dy, False, 0.0, None, torch.float32)
    check_all(x, w, b, dy, y, grads, 1e-5, False, 0.0, None)


def test_constant_rows(gpu_lib):
    x = torch.zeros(4, 96, device=dev)
    x[1] = 3.0
    w, b = torch.full((96,), 2.0, device=dev), torch.full((96,), 0.5, device=dev)
    y = hip_layernorm(x, w, b)
    assert torch.equal(y, torch.full_like(y, 0.5))


def test_rows_with_inf_or_nan_stay_by_themselves(gpu_lib):
    x, w, b, dy = make(9, 300, torch.float32, torch.float32, 3)
    clean, grads = run(x, w, b, dy, True, 0.0, None, torch.float32)
    x2 = x.detach().clone()
    x2[2, 7], x2[5, 0], x2[6, 299] = float("nan"), float("inf"), -float("inf")
    y, g2 = run(x2, w, b, dy, True, 0.0, None, torch.float32)
    ok = [0, 1, 3, 4, 7, 8]
    assert torch.equal(y[ok], clean[ok]) and torch.equal(g2[0][ok], grads[0][ok])
    assert bool(torch.isnan(y[[2, 5, 6]]).all()) and bool(torch.isnan(g2[0][[2, 5, 6]]).all())


@pytest.mark.parametrize("which", ["none", "w", "b"])
def test_without_weights(gpu_lib, which):
    x, w, b, dy = make(12, 200, torch.float32, torch.float32, 5)
    w, b = (w if which == "w" else None), (b if which == "b" else None)
    y, grads = run(x, w, b, dy, True, 0.1, 3, torch.float32)
    check_all(x, w, b, dy, y, grads, 1e-5, True, 0.1, ref.keep_mask(range(12), 200, 0.1, 3))


def test_weights_in_16_bits_and_frozen_leaves(gpu_lib):
    x, w, b, dy = make(12, 200, torch.bfloat16, torch.bfloat16, 5)
    wh, bh = w.bfloat16(), b.bfloat16()
    y, grads = run(x, wh, bh, dy, True, 0.0, None, torch.bfloat16)
    assert grads[1].dtype == torch.bfloat16
    check_all(x, wh, bh, dy, y, grads, 1e-5, True, 0.0, None)
    xf = x.detach()
    yf = hip_layernorm(xf, wh, bh.detach(), gelu=True)
    assert torch.equal(torch.autograd.grad(yf, wh, dy)[0], grads[1])
    yf = hip_layernorm(x, wh.detach(), bh.detach(), gelu=True)
    assert torch.equal(torch.autograd.grad(yf, x, dy)[0], grads[0])


def test_strides_offsets_and_shapes(gpu_lib):
    """Column slices off every vector boundary, transposed and expanded inputs and
    gradients, leading dimensions: the bits of the contiguous call."""
    g = torch.Generator(device=dev).manual_seed(0)
    for t in (torch.float32, torch.bfloat16):
        wide = torch.randn(40, 415, generator=g, device=dev).to(t)
        w, b = torch.randn(201, generator=g, device=dev), torch.randn(201, generator=g, device=dev)
        dyw = torch.randn(40, 415, generator=g, device=dev).to(t)
        for off in (0, 1, 3, 8, 13):
            x, dy = wide[:, off:off + 201], dyw[:, off + 1:off + 202]
            ya, ga = run(x.clone(), w, b, dy.clone(), True, 0.1, 5, t)
            yb, gb = run(x.detach(), w, b, dy, True, 0.1, 5, t)
            assert torch.equal(ya, yb) and all(torch.equal(m, n) for m, n in zip(ga, gb))
        xt = wide[:, :201].t().contiguous().t()
        yb, gb = run(xt, w, b, dyw[:, :201].t().contiguous().t(), True, 0.1, 5, t)
        ya, ga = run(wide[:, :201].clone(), w, b, dyw[:, :201].clone(), True, 0.1, 5, t)
        assert torch.equal(ya, yb) and all(torch.equal(m, n) for m, n in zip(ga, gb))
        y3, g3 = run(wide[:, :201].reshape(5, 8, 201), w, b, dyw[:, :201].reshape(5, 8, 201), True, 0.1,
                     5, t)
        assert torch.equal(y3.view(40, 201), ya) and torch.equal(g3[0].view(40, 201), ga[0])
        assert torch.equal(hip_layernorm(wide[0, :201], w, b, gelu=True, p=0.1, seed=5), ya[0])
        x = wide[:, :201].clone().requires_grad_(True)
        hip_layernorm(x, w, b, gelu=True).sum().backward()  # an expanded gradient
        x2 = x.detach().clone().requires_grad_(True)
        hip_layernorm(x2, w, b, gelu=True).backward(torch.ones(40, 201, device=dev, dtype=t))
        assert torch.equal(x.grad, x2.grad)


def test_no_rows(gpu_lib):
    x = torch.zeros(0, 64, device=dev, requires_grad=True)
    w, b = (torch.ones(64, device=dev, requires_grad=True) for _ in range(2))
    y = hip_layernorm(x, w, b, gelu=True, p=0.5, seed=1)
    assert y.shape == (0, 64)
    y.sum().backward()
    assert x.grad.shape == (0, 64) and bool((w.grad == 0).all()) and bool((b.grad == 0).all())


def test_gradient_against_differences(gpu_lib):
    """The kernel's gradients along random directions against central differences
    of the loss in 64 bits: the step's own error is of order h^2 = 1e-8 of the
    loss's third derivative, the gradient's about 100 U of its size."""
    x, w, b, dy = make(7, 129, torch.float32, torch.float32, 11)
    y, grads = run(x, w, b, dy, True, 0.2, 3, torch.float32)
    keep = ref.keep_mask(range(7), 129, 0.2, 3)
    base = [t.detach().cpu().double() for t in (x, w, b)]

    def loss(ts):
        return float((ref.layernorm(*ts, 1e-5, True, 0.2, keep) * dy.cpu().double()).sum())

    g = torch.Generator().manual_seed(2)
    for i in range(3):
        for _ in range(4):
            v = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
            v /= v.norm()
            hi, lo = list(base), list(base)
            hi[i], lo[i] = base[i] + 1e-4 * v, base[i] - 1e-4 * v
            diff = (loss(hi) - loss(lo)) / 2e-4
            got = float((grads[i].cpu().double() * v).sum())
            assert abs(got - diff) <= 1e-5 * float(grads[i].norm()), (i, got, diff)


def test_deterministic(gpu_lib):
    x, w, b, dy = make(5000, 384, torch.bfloat16, torch.float32, 4)
    a = run(x, w, b, dy, True, 0.1, 9, torch.float32)
    for _ in range(3):
        c = run(x, w, b, dy, True, 0.1, 9, torch.float32)
        assert torch.equal(a[0], c[0]) and all(torch.equal(m, n) for m, n in zip(a[1], c[1]))


def test_offsets_past_32_bits(gpu_lib):
    rows, d = (1 << 21) + 5, 1029
    g = torch.Generator(device=dev).manual_seed(0)
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device=dev)
    some = [0, 1 << 20, rows - 2, rows - 1]
    x[some] = torch.randn(4, d, generator=g, device=dev).bfloat16()
    w, b = torch.randn(d, generator=g, device=dev), torch.randn(d, generator=g, device=dev)
    xs = x.requires_grad_(True)
    w.requires_grad_(True)
    y = hip_layernorm(xs, w, b, gelu=True, p=0.2, seed=6)
    dy = torch.zeros_like(y)
    dys = torch.randn(4, d, generator=g, device=dev).bfloat16()
    dy[some] = dys
    dx, dw = torch.autograd.grad(y, (xs, w), dy)
    keep = ref.keep_mask(some, d, 0.2, 6)
    check_all(x.detach()[some], w, b, dys, y.detach()[some], (dx[some], dw, None), 1e-5, True, 0.2, keep)


def test_on_a_stream_of_its_own(gpu_lib):
    x, w, b, dy = make(400, 768, torch.float32, torch.float32, 4)
    a = run(x, w, b, dy, True, 0.1, 9, torch.float32)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        c = run(x, w, b, dy, True, 0.1, 9, torch.float32)
    st.synchronize()
    assert torch.equal(a[0], c[0]) and all(torch.equal(m, n) for m, n in zip(a[1], c[1]))


def test_captured_training_step(gpu_lib):
    x, w, b, dy = make(300, 384, torch.bfloat16, torch.float32, 4)
    seed = torch.tensor([1], device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x, w, b, dy, True, 0.1, seed, torch.float32)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, grads = run(x, w, b, dy, True, 0.1, seed, torch.float32)
        outs = [y.detach(), *grads]
        del y
    for value in (1, 5, 2, 5):
        seed.fill_(value)
        graph.replay()
        got = [t.clone() for t in outs]
        torch.cuda.synchronize()
        ye, ge = run(x, w, b, dy, True, 0.1, seed, torch.float32)
        for m, n in zip(got, [ye.detach(), *ge]):
            assert torch.equal(m, n)
        del ye, ge


def test_close_to_torchs_own(gpu_lib):
    """The plain norm beside torch's on the device, in fp32."""
    x, w, b, _ = make(64, 512, torch.float32, torch.float32, 2)
    y = hip_layernorm(x, w, b)
    z = F.layer_norm(x, (512,), w, b)
    assert float((y - z).abs().max()) <= 256 * U * float(z.abs().max())


def test_refusals(gpu_lib):
    x, w, b, _ = make(4, 64, torch.float32, torch.float32, 1)
    with pytest.raises(ValueError, match="weight"):
        hip_layernorm(x, w[:-1], b)
    with pytest.raises(ValueError, match="bias"):
        hip_layernorm(x, w, b.cpu())
    with pytest.raises(ValueError, match="last dimension"):
        hip_layernorm(torch.zeros(3, 0, device=dev))
    with pytest.raises(TypeError, match="dtype"):
        hip_layernorm(x.double())
    with pytest.raises(TypeError, match="dtype"):
        hip_layernorm(x, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="eps"):
        hip_layernorm(x, eps=-1e-5)
    with pytest.raises(ValueError, match="p must"):
        hip_layernorm(x, p=2.0, seed=1)
    with pytest.raises(ValueError, match="needs a seed"):
        hip_layernorm(x, p=0.1)
    with pytest.raises(ValueError, match="stream"):
        hip_layernorm(x, p=0.1, seed=1, stream=1 << 32)
