"""Sampling with settings a row at the ends of their ranges, against the
restatement in 64 bits (oracle/heads_ref.py)."""

import pytest
import torch

from redpanda_amd.sampling import hip_sample
from tests.test_gpu_sampling import check, make

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.mark.parametrize("R,V", [(6, 20001), (129, 20001), (6, 3000), (1500, 3000)])
def test_one_setting_a_row(gpu_lib, R, V):
    """One setting is a tensor and the others numbers: a row's first place alone is
    kept from a min-p above 1 or a NaN on, whichever kernel takes the row."""
    lg, u = make(R, V, seed=V)

    def rows(*v):
        return torch.tensor(v, device=dev).repeat(-(-R // len(v)))[:R]

    nan = float("nan")
    mp = rows(0.02, 1.0, 1.5, nan, 0.0, 2.0)
    some = slice(0, 12)
    for name, v, more in (("min_p", mp, {}), ("min_p", mp, dict(temperature=0.7)),
                          ("min_p", mp, dict(top_p=0.9)), ("min_p", mp, dict(top_k=30)),
                          ("top_k", rows(0, 1, 5, -3, 300).int(), {}),
                          ("top_p", rows(1.0, 0.0, 0.5, nan, 2.0), {}),
                          ("temperature", rows(1.0, 0.0, -1.0, nan, 0.3), {})):
        ids, logp = hip_sample(lg, u, logprob=True, **{name: v}, **more)
        short = {"temperature": "T", "top_k": "k", "top_p": "tp", "min_p": "mp"}
        want = check(lg[some], u[some], **{short[name]: v[some]}, **{short[k]: x for k, x in more.items()})
        assert torch.equal(ids[some], want), name
        first = lg.argmax(1)
        alone = {"min_p": ~(v <= 1), "top_k": v == 1, "top_p": ~(v > 0), "temperature": ~(v > 0)}[name]
        assert torch.equal(ids[alone], first[alone]) and bool((logp[alone] == 0).all()), name


@pytest.mark.parametrize("V", [300, 3000, 9001, 20001])
def test_the_smallest_temperatures(gpu_lib, V):
    """Only the largest logits have a weight, equal ones the same, down to the least
    positive number."""
    lg, u = make(5, V, seed=V)
    lg[1, [3, V // 2, V - 1]] = 30.0
    lg[2] = 0.25
    lg[3, [V // 3, V - 2]] = float("inf")
    lg[4, 5:] = -float("inf")
    u[1], u[2], u[3] = 0.5, 0.75, 0.9
    for T in (5e-324, 1e-310, 8e-309, 1e-300, 1e-45):
        for s in (dict(), dict(k=2), dict(tp=0.9), dict(mp=1.0), dict(k=200, tp=0.5)):
            check(lg, u, T=T, **s)
    check(lg, u, T=torch.full((5,), 1e-45, device=dev), tp=0.9)


@pytest.mark.parametrize("R,V", [(8, 300), (8, 3000), (8, 9001), (8, 20001), (1300, 3000), (400, 17000)])
def test_infinite_temperatures_a_row(gpu_lib, R, V):
    """Every candidate weighs the same, whatever min-p asks for."""
    lg, u = make(R, V, seed=V)
    lg[1, ::3] = -float("inf")
    lg[2, 7:9] = float("inf")
    lg[4] = 0.0
    T = torch.tensor([float("inf"), float("inf"), float("inf"), 1.0, float("inf"), 0.0, 3e38, 1e30],
                     device=dev).repeat(-(-R // 8))[:R]
    some = slice(0, 8)
    for s in (dict(mp=1.0), dict(mp=0.5), dict(), dict(tp=0.3), dict(k=7), dict(k=7, mp=1.0),
              dict(tp=0.5, mp=1.0), dict(k=200, tp=0.9)):
        want = check(lg[some], u[some], T=T[some], **s)
        ids = hip_sample(lg, u, temperature=T, top_k=s.get("k", 0), top_p=s.get("tp", 1.0),
                         min_p=s.get("mp", 0.0))
        assert torch.equal(ids[some], want)
    check(lg[some], u[some], T=T[some], mp=torch.ones(8, device=dev))


@pytest.mark.parametrize("R,V", [(6, 20001), (6, 9001), (1300, 6000), (6, 600)])
def test_temperatures_that_even_out_all_values(gpu_lib, R, V):
    """A temperature at which even the type's lowest value has a weight: masked
    places of that value count, and the cut falls among them."""
    lg, u = make(R, V, seed=V + 1)
    lg[:, 100:] = torch.finfo(torch.float32).min
    lg[1, 50:100] = torch.finfo(torch.float32).max
    some = slice(0, 6)
    u[:6] = torch.tensor([0.999, 0.2, 0.5, 0.9, 1e-4, 0.97], device=dev)
    for T in (1e38, 3e37, 1e300):
        for s in (dict(tp=0.9), dict(tp=0.99), dict(k=500), dict(k=300, tp=0.5), dict(), dict(mp=0.01)):
            want = check(lg[some], u[some], T=T, **s)
            ids = hip_sample(lg, u, temperature=T, top_k=s.get("k", 0), top_p=s.get("tp", 1.0),
                             min_p=s.get("mp", 0.0))
            assert torch.equal(ids[some], want)
