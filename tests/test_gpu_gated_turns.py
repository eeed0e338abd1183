"""Gated recurrences whose workgroups take several turns of steps: the state and the
gradient carried from turn to turn, both halves of the LDS, the steps loaded ahead in the
sums of a split, and more chunks than the fold's waves take at once.  The bounds are those
of tests/test_gpu_gated.py."""

import pytest
import torch

from tests.test_gpu_gated import TYPES, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B,L,D,starts", [
    (200, 2501, 3, 0.0),    # split into chunks of 256 steps, four turns each, the last of them cut
    (200, 2501, 3, 0.004),
    (300, 203, 66, 0.0),    # whole sequences by four waves: four turns, the last of them cut
    (300, 203, 66, 0.02),
    (1, 20000, 5, 0.0005),  # 313 chunks: a wave of the fold takes 20
])
def test_several_turns(gpu_lib, B, L, D, starts, t):
    check(*make(B, L, D, t, L + D, True, starts))


def test_several_turns_of_wide_rows(gpu_lib):
    check(*make(60, 2500, 130, torch.bfloat16, 3, True, 0.002))


def test_long_memory_over_turns(gpu_lib):
    """Gates near 1: what enters a turn matters to the end."""
    for B, L, D in ((200, 1203, 5), (300, 203, 66)):
        x, z, h0, _, dy, dh = make(B, L, D, torch.float32, 5)
        check(x, (z.abs() + 5).detach(), 100 * h0, None, dy, dh)
