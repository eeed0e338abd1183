"""Rollouts drawn on the device at their ends."""

import pytest
import torch

from tests.test_gpu_search_heads import model

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.mark.parametrize("compact", [True, False])
def test_a_rollout_without_a_first_move_has_the_boards_value(gpu_lib, compact):
    m = model(4)
    board = torch.arange(9)
    u = torch.rand(3, 5, generator=torch.Generator().manual_seed(2)).to(dev)
    legal = torch.arange(20, dtype=torch.int32, device=dev).expand(5, 20).clone()
    legal[[1, 3]] = -1
    tok, logp, val = m.sample_rollout(board, u, legal=lambda t, last: legal, compact=compact)
    assert bool((tok[:, [1, 3]] == -1).all()) and bool((logp[:, [1, 3]] == -float("inf")).all())
    with torch.no_grad():
        hidden, _ = m.prime_board(board.to(dev), compact=compact)
        want = float(torch.tanh(m.value_head(hidden)))
    # a head's GELU and norm are a few hundred fp32 roundings either way
    assert float((val[:, [1, 3]] - want).abs().max()) <= 1e-5 * max(abs(want), 1e-2)
    # the others are as without the ended ones
    live = [0, 2, 4]
    tok2, logp2, val2 = m.sample_rollout(board, u[:, live].contiguous(), legal=lambda t, last: legal[live],
                                         compact=compact)
    assert torch.equal(tok[:, live], tok2)
    assert float((val[:, live] - val2).abs().max()) <= 1e-5


def test_no_plies(gpu_lib):
    m = model(4)
    tok, logp, val = m.sample_rollout(torch.arange(9), torch.rand(0, 5, device=dev))
    assert tok.shape == logp.shape == val.shape == (0, 5)
    assert tok.dtype == torch.int64 and logp.dtype == val.dtype == torch.float32
    with torch.autocast("cuda", torch.bfloat16):
        a = m.sample_rollout(torch.arange(9), torch.rand(0, 5, device=dev))
        b = m.sample_rollout(torch.arange(9), torch.rand(1, 5, device=dev))
    assert [t.dtype for t in a] == [t.dtype for t in b]
