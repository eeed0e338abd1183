"""Sampling by every kernel shape that the launch rule picks, against the
restatement in 64 bits (oracle/heads_ref.py) and against the same rows in small
calls: a row's token and log-probability are sums of whole numbers, so they do
not depend on the kernel that takes it."""

import numpy as np
import pytest
import torch

from oracle import heads_ref as ref
from redpanda_amd.sampling import hip_sample

pytestmark = pytest.mark.gpu
dev = "cuda"
INF = float("inf")

SETTINGS = [dict(), dict(T=0.0), dict(T=0.7), dict(k=1), dict(k=8), dict(k=40, tp=0.95), dict(tp=0.9),
            dict(tp=0.5, T=1.3), dict(mp=0.05), dict(tp=0.9, mp=0.02), dict(k=100, tp=0.9, mp=0.02),
            dict(k=128), dict(k=129), dict(k=191, tp=0.9), dict(k=192), dict(k=1000, T=1.3), dict(mp=1.0),
            dict(tp=0.999, T=2.0)]

# (rows, vocabulary): a wave a row in registers; a wave a row, short and long rows;
# four waves a row beyond their registers; sixteen waves a row; few long rows
# shared by workgroups
SHAPES = [(600, 500), (600, 1001), (1300, 5003), (70, 9001), (330, 16400), (130, 40001), (40, 16400)]


def rows_of_all_kinds(R, V, t, seed):
    """Random rows, and among the first ones equal, masked, infinite, NaN and
    outlying values."""
    g = torch.Generator(device=dev).manual_seed(seed)
    lg = 2.5 * torch.randn(R, V, generator=g, device=dev)
    lg[1] = 0.5
    lg[2] = torch.arange(V, device=dev) % 7 * 0.25
    lg[3] = -INF
    lg[4, ::2] = float("nan")
    lg[5, [V // 5, V // 3, V - 1]] = INF
    lg[6, 10:] = torch.finfo(torch.float32).min
    lg[7, 17] = -1e9
    lg[8, 5] = 40.0
    lg[9] *= 1e-3
    lg[10, V // 2:] = -INF
    lg[11] = float("nan")
    return lg.to(t), torch.rand(R, generator=g, device=dev)


def check(lg, u, tokens=None, T=1.0, k=0, tp=1.0, mp=0.0):
    def call(at):
        s = [v[at].contiguous() if torch.is_tensor(v) else v for v in (T, k, tp, mp)]
        return hip_sample(lg[at], u[at], temperature=s[0], top_k=s[1], top_p=s[2], min_p=s[3],
                          tokens=None if tokens is None else tokens[at], logprob=True)

    R = lg.shape[0]
    ids, logp = call(slice(None))
    step = 33  # a call of few rows takes another shape
    for i in range(0, R, step):
        a, b = call(slice(i, i + step))
        assert torch.equal(a, ids[i:i + step]) and torch.equal(b, logp[i:i + step]), i
    some = sorted({*range(12), *np.random.default_rng(R).integers(0, R, 24).tolist(), R - 1})

    def host(v):
        return v[some].cpu().double().numpy() if torch.is_tensor(v) else v

    want, wlogp = ref.sample(host(lg), host(u), host(T), host(k), host(tp), host(mp),
                             None if tokens is None else tokens[some].cpu().numpy())
    assert ids[some].tolist() == want
    for a, b in zip(logp[some].tolist(), wlogp):
        assert a == b or abs(a - b) <= 2.0 ** -24 * abs(b) + 1e-9, (a, b)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", SHAPES)
def test_every_shape(gpu_lib, R, V, t):
    lg, u = rows_of_all_kinds(R, V, t, V)
    for s in SETTINGS:
        check(lg, u, **s)


@pytest.mark.parametrize("R,V", SHAPES)
def test_every_shape_with_settings_of_their_own(gpu_lib, R, V):
    lg, u = rows_of_all_kinds(R, V, torch.float32, V + 1)
    g = torch.Generator(device=dev).manual_seed(2)

    def r():
        return torch.rand(R, generator=g, device=dev)

    T = torch.where(r() < 0.2, 0.0, 0.3 + r())
    k = ((r() * 300) * (r() < 0.7)).to(torch.int32)
    tp = torch.where(r() < 0.3, 1.0, r())
    mp = torch.where(r() < 0.5, 0.0, 0.1 * r())
    check(lg, u, T=T, k=k, tp=tp, mp=mp)
    check(lg, u, k=k)
    check(lg, u, tp=tp)
    check(lg, u, T=T)
    check(lg, u, mp=mp)


@pytest.mark.parametrize("R,M", [(600, 400), (600, 1000), (1300, 2500), (100, 9000)])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_lists_of_every_shape(gpu_lib, R, M, t):
    V = 10007
    lg, u = rows_of_all_kinds(R, V, t, M)
    g = torch.Generator(device=dev).manual_seed(M)
    tok = torch.argsort(torch.rand(R, V, generator=g, device=dev), dim=1)[:, :M].to(torch.int32)
    n = torch.randint(0, M + 1, (R, 1), generator=g, device=dev)
    tok = torch.where(torch.arange(M, device=dev) < n, tok, -1)
    for s in (dict(), dict(tp=0.9), dict(k=40, tp=0.95), dict(mp=0.05, T=0.7), dict(k=150), dict(T=0.0)):
        check(lg, u, tokens=tok, **s)


@pytest.mark.parametrize("R,V", [(1300, 1500), (1300, 7001), (1300, 9001), (600, 17001), (1400, 17001)])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_top_k_around_what_a_shape_lists(gpu_lib, R, V, t):
    lg, u = rows_of_all_kinds(R, V, t, V)
    for k in (127, 128, 129, 191, 192, 511, 512, 513, V - 1, V, V + 1):
        check(lg, u, k=k)
    k = torch.arange(R, device=dev, dtype=torch.int32) % 7 * 40
    check(lg, u, k=k, tp=0.95)
