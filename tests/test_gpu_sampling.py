"""GPU parity of sampling against the restatement in 64 bits: the tokens have to be
equal, the log-probabilities within their rounding to fp32.  (The kernel misses a
border between two tokens by about 1e-13 of the total; the inputs' borders are no
closer.)"""

import math

import numpy as np
import pytest
import torch

from oracle import heads_ref as ref
from redpanda_amd.sampling import hip_sample

pytestmark = pytest.mark.gpu
dev = "cuda"


def check(logits, u, tokens=None, T=1.0, k=0, tp=1.0, mp=0.0):
    def host(v):
        return v.cpu().double().numpy() if torch.is_tensor(v) else v

    ids, logp = hip_sample(logits, u, temperature=T, top_k=k, top_p=tp, min_p=mp, tokens=tokens,
                           logprob=True)
    want, wlogp = ref.sample(host(logits), host(u), host(T), host(k), host(tp), host(mp),
                             None if tokens is None else tokens.cpu().numpy())
    assert ids.dtype == torch.int64 and ids.tolist() == want
    for a, b in zip(logp.tolist(), wlogp):
        assert a == b or abs(a - b) <= 2.0 ** -24 * abs(b) + 1e-9, (a, b)
    only = hip_sample(logits, u, temperature=T, top_k=k, top_p=tp, min_p=mp, tokens=tokens)
    assert torch.equal(only, ids)
    return ids


def make(R, V, t=torch.float32, seed=0, std=2.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    lg = (std * torch.randn(R, V, generator=g, device=dev)).to(t)
    return lg, torch.rand(R, generator=g, device=dev)


SETTINGS = [dict(), dict(T=0.0), dict(T=0.7), dict(k=1), dict(k=8), dict(k=40, tp=0.95), dict(tp=0.9),
            dict(tp=0.5, T=1.3), dict(mp=0.05), dict(k=200, tp=0.9, mp=0.02), dict(k=1000, T=1.3),
            dict(tp=0.0), dict(mp=1.0), dict(tp=0.999, T=2.0)]


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("s", SETTINGS)
def test_settings(gpu_lib, s, t):
    lg, u = make(33, 1000, t, 5)
    check(lg, u, **s)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 255, 256, 257, 2047, 2049, 8191, 8192, 8193, 16385, 40001,
                               131072])
@pytest.mark.parametrize("s", [dict(tp=0.9), dict(k=50, tp=0.95), dict(mp=0.1, T=0.8), dict()])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_sizes_of_the_vocabulary(gpu_lib, V, s, t):
    lg, u = make(3, V, t, V)
    check(lg, u, **s)


@pytest.mark.parametrize("R", [1, 2, 600, 1500])
@pytest.mark.parametrize("V", [100, 5000])
def test_numbers_of_rows(gpu_lib, R, V):
    lg, u = make(R, V, torch.bfloat16, R)
    check(lg, u, tp=0.9, k=300)


def test_every_row_its_own_settings(gpu_lib):
    R = 257
    lg, u = make(R, 3001, seed=1)
    g = torch.Generator(device=dev).manual_seed(2)

    def r():
        return torch.rand(R, generator=g, device=dev)

    T = torch.where(r() < 0.2, torch.zeros(R, device=dev), 0.3 + r())
    k = (r() * 100).to(torch.int32) * (r() < 0.7)
    tp = torch.where(r() < 0.3, torch.ones(R, device=dev), r())
    mp = torch.where(r() < 0.5, torch.zeros(R, device=dev), 0.1 * r())
    check(lg, u, T=T, k=k.to(torch.int32), tp=tp, mp=mp)
    check(lg, u, T=T.double(), k=k.long(), tp=0.9, mp=mp)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [700, 9000])
@pytest.mark.parametrize("s", [dict(k=300), dict(tp=0.3), dict(k=500, tp=0.4), dict(), dict(mp=0.5)])
def test_equal_logits(gpu_lib, V, t, s):
    """Whole rows of one value, and of few: the cut falls between equal logits,
    where the first places stay."""
    lg = torch.zeros(4, V, device=dev)
    lg[1] = -3.25
    lg[2, ::2] = 1.0
    lg[3] = torch.arange(V, device=dev) % 7 * 0.25
    lg[3, 5] = -1e30
    u = torch.tensor([0.1, 0.77, 0.5, 0.999], device=dev)
    check(lg.to(t), u, **s)


def test_a_range_stretched_by_outliers(gpu_lib):
    """One very low value, masked places of the type's lowest value, and nearly
    equal logits: most elements fall into one step of the histogram."""
    lg, u = make(6, 6000, seed=4, std=0.001)
    lg[0, 17] = -1e9
    lg[1, ::3] = torch.finfo(torch.float32).min
    lg[2, 5] = 30.0
    lg[3] *= 1e-30
    lg[4] += 1000.0
    lg[5, 100:] = torch.finfo(torch.float32).min
    for s in (dict(tp=0.9), dict(k=2000), dict(k=1500, tp=0.5), dict(), dict(T=100.0, tp=0.7),
              dict(T=1e-4, tp=0.9, k=77)):
        check(lg, u, **s)


def test_masked_rows_inf_and_nan(gpu_lib):
    lg, u = make(9, 5000, seed=8)
    inf = float("inf")
    lg[0] = -inf
    lg[1] = float("nan")
    lg[2, :] = -inf
    lg[2, 4321] = -50.0
    lg[3, ::2] = float("nan")
    lg[4, [10, 3000, 4999]] = inf
    lg[5, 1:] = -inf
    lg[6, 7], lg[6, 8] = -0.0, 0.0
    lg[6, 9:] = -1.0
    lg[6, :7] = -1.0
    lg[7] = torch.finfo(torch.float32).min
    for s in (dict(), dict(tp=0.9), dict(k=2), dict(k=100, tp=0.8, mp=0.1), dict(T=0.0)):
        for t in (torch.float32, torch.bfloat16):
            check(lg.to(t), u, **s)
    ids, logp = hip_sample(lg, u, logprob=True)
    assert ids[0] == -1 and ids[1] == -1 and ids[2] == 4321 and float(logp[0]) == -inf
    assert float(logp[2]) == 0.0


@pytest.mark.parametrize("M", [1, 5, 64, 200, 256, 257, 1000])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_lists_of_ids(gpu_lib, M, t):
    R, V = 41, 4001
    lg, u = make(R, V, t, M)
    g = torch.Generator().manual_seed(M)
    tok = torch.stack([torch.randperm(V, generator=g)[:M] for _ in range(R)]).to(torch.int32)
    n = torch.randint(0, M + 1, (R, 1), generator=g)
    tok = torch.where(torch.arange(M) < n, tok, -1).to(dev)
    for s in (dict(), dict(mp=0.05, T=0.7), dict(k=4), dict(tp=0.8), dict(T=0.0), dict(k=100, tp=0.9)):
        ids = check(lg, u, tokens=tok, **s)
        assert bool(((ids < 0) == (n.view(-1).to(dev) == 0)).all())
    assert torch.equal(hip_sample(lg, u, tokens=tok.long()), hip_sample(lg, u, tokens=tok))


def test_bad_ids_are_padding(gpu_lib):
    lg, u = make(3, 100, seed=1)
    tok = torch.tensor([[100, 2**31 - 1, 7, -5], [-2**31, -1, 100, 101], [3, 3, 3, 99]],
                       dtype=torch.int32, device=dev)
    assert check(lg, u, tokens=tok).tolist()[:2] == [7, -1]
    assert hip_sample(lg, u, tokens=torch.zeros(3, 0, dtype=torch.int32, device=dev)).tolist() == [-1] * 3


def test_the_ends_of_u(gpu_lib):
    lg, _ = make(1, 5000, seed=3)
    for u in (0.0, 1.0 - 2.0 ** -24):
        for s in (dict(), dict(k=30), dict(tp=0.9)):
            check(lg, torch.tensor([u], device=dev), **s)
    kept = set(torch.topk(lg, 30).indices[0].tolist())
    for u in (1.0, 2.0, float("inf"), -1.0, float("nan")):  # outside [0, 1): still a kept token
        assert int(hip_sample(lg, torch.tensor([u], device=dev), top_k=30)) in kept


def test_shares_of_many_draws(gpu_lib):
    """100,000 rows of the same logits: each token's share within five standard
    deviations of its probability among the kept."""
    n = 100000
    lg = torch.tensor([1.0, 0.0, 2.0, -1.0, 0.5, 2.0], device=dev).expand(n, 6)
    u = torch.rand(n, generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    ids = hip_sample(lg, u, temperature=0.8, top_k=4)
    w = torch.exp(torch.tensor([1.0, 0.0, 2.0, -1.0, 0.5, 2.0], dtype=torch.float64) / 0.8)
    w[[1, 3]] = 0
    for i, q in enumerate((w / w.sum()).tolist()):
        assert abs(float((ids == i).double().mean()) - q) <= 5 * math.sqrt(q * (1 - q) / n)


def test_strides_and_offsets(gpu_lib):
    lg, u = make(12, 9100, torch.bfloat16, 6)
    for off in (0, 1, 5, 8):
        v = lg[:, off:off + 8192]
        a = hip_sample(v, u, top_p=0.9)
        assert torch.equal(a, hip_sample(v.clone(), u, top_p=0.9))
        check(v, u, tp=0.9)
    assert torch.equal(hip_sample(lg.t().contiguous().t(), u, top_k=9), hip_sample(lg, u, top_k=9))
    u2 = torch.stack((u, u), 1)[:, 0]
    assert torch.equal(hip_sample(lg, u2, top_k=9), hip_sample(lg, u.double(), top_k=9))


def test_offsets_past_32_bits(gpu_lib):
    store = torch.zeros(3 * (1 << 30) + 9000, dtype=torch.bfloat16, device=dev)
    lg, u = make(3, 8192, torch.bfloat16, 9)
    v = store.as_strided((3, 8192), (3 << 29, 1))
    v.copy_(lg)
    assert torch.equal(hip_sample(v, u, top_p=0.9), hip_sample(lg, u, top_p=0.9))


def test_streams_graphs_and_repeats(gpu_lib):
    lg, u = make(600, 4096, torch.bfloat16, 2)
    want = hip_sample(lg, u, top_p=0.9, logprob=True)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = hip_sample(lg, u, top_p=0.9, logprob=True)
    st.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hip_sample(lg, u, top_p=0.9, logprob=True)
    for i in range(4):
        u.copy_(torch.rand(600, generator=torch.Generator(device=dev).manual_seed(i), device=dev))
        graph.replay()
        a = [t.clone() for t in out]
        torch.cuda.synchronize()
        b = hip_sample(lg, u, top_p=0.9, logprob=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_refusals(gpu_lib):
    lg, u = make(4, 100)
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
                dict(top_p=-0.1), dict(top_p=float("nan")), dict(min_p=1.1), dict(min_p=-0.1)):
        with pytest.raises(ValueError):
            hip_sample(lg, u, **bad)
    for bad in (dict(top_k=torch.ones(3, dtype=torch.int32, device=dev)), dict(min_p=torch.zeros(4)),
                dict(temperature=torch.ones(4, 1, device=dev))):
        with pytest.raises(ValueError, match="must be a number or"):
            hip_sample(lg, u, **bad)
    with pytest.raises(ValueError, match="u "):
        hip_sample(lg, u[:3])
    with pytest.raises(ValueError, match="logits"):
        hip_sample(lg[0], u)
    with pytest.raises(ValueError, match="empty"):
        hip_sample(lg[:, :0], u)
    with pytest.raises(TypeError, match="dtype"):
        hip_sample(lg.double(), u)
    with pytest.raises(TypeError, match="tokens"):
        hip_sample(lg, u, tokens=torch.zeros(4, 2, device=dev))
    with pytest.raises(ValueError, match="tokens"):
        hip_sample(lg, u, tokens=torch.zeros(3, 2, dtype=torch.int32, device=dev))
    assert hip_sample(lg[:0], u[:0]).shape == (0,)
    assert np.array_equal(hip_sample(lg[:1], u[:1]).cpu().numpy(),
                          hip_sample(lg, u)[:1].cpu().numpy())


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", [(1, 16385), (2, 20000), (5, 32769), (3, 70001), (2, 131073)])
def test_rows_that_workgroups_share(gpu_lib, R, V, t):
    """Few long rows: each plan, masked and equal values, and what the shared looks
    do not hold."""
    lg, u = make(R, V, t, V)
    lg[0, V // 3:] = -float("inf")  # whole stretches without a candidate
    for s in SETTINGS + [dict(k=191), dict(k=192, tp=0.5), dict(k=3000, mp=0.001), dict(tp=0.99, mp=0.01)]:
        check(lg, u, **s)
    flat = torch.zeros(R, V, device=dev)
    flat[0, 7::5] = 0.5
    for s in (dict(tp=0.3), dict(k=150), dict(), dict(T=0.0), dict(mp=0.9, tp=0.8)):
        check(flat.to(t), u, **s)
    odd = lg.clone()
    odd[0] = -float("inf")
    odd[-1, V - 1] = float("inf")
    if R > 2:
        odd[1] = float("nan")
    for s in (dict(tp=0.9), dict(k=5), dict(), dict(T=0.0)):
        check(odd, u, **s)


def test_shared_rows_with_settings_of_their_own(gpu_lib):
    R, V = 60, 30011
    lg, u = make(R, V, seed=5)
    g = torch.Generator(device=dev).manual_seed(2)

    def r():
        return torch.rand(R, generator=g, device=dev)

    T = torch.where(r() < 0.2, torch.zeros(R, device=dev), 0.3 + r())
    k = (r() * 300).to(torch.int32) * (r() < 0.6)
    tp = torch.where(r() < 0.3, torch.ones(R, device=dev), r())
    mp = torch.where(r() < 0.5, torch.zeros(R, device=dev), 0.1 * r())
    check(lg, u, T=T, k=k.to(torch.int32), tp=tp, mp=mp)
    for _ in range(3):  # the same bits each time
        a = hip_sample(lg, u, temperature=T, top_p=tp, logprob=True)
        b = hip_sample(lg, u, temperature=T, top_p=tp, logprob=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_shared_rows_in_a_graph(gpu_lib):
    lg, u = make(9, 20001, torch.bfloat16, 2)
    hip_sample(lg, u, top_p=0.9, logprob=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hip_sample(lg, u, top_p=0.9, logprob=True)
    for i in range(4):
        u.copy_(torch.rand(9, generator=torch.Generator(device=dev).manual_seed(i), device=dev))
        graph.replay()
        a = [t.clone() for t in out]
        torch.cuda.synchronize()
        b = hip_sample(lg, u, top_p=0.9, logprob=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
