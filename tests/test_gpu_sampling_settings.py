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
