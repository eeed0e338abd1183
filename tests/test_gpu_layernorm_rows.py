"""Layer norm where every group of lanes walks several rows: the buffers that a
row's sums share, the rows loaded ahead and the weights' gradients over several
rows, at one width of each kernel shape, within the bounds of
tests/test_gpu_layernorm.py."""

import pytest
import torch

from oracle import heads_ref as ref
from tests.test_gpu_layernorm import check_all, make, run

pytestmark = pytest.mark.gpu
F, B, H = torch.float32, torch.bfloat16, torch.float16


# widths of each shape (8 lanes to 1024, one to three blocks a lane), rows for two
# to four a group and a remainder
@pytest.mark.parametrize("rows,d,tx,tout", [
    (115003, 60, B, F), (58001, 120, F, F), (50021, 190, B, B), (29009, 250, F, B), (25013, 384, F, F),
    (25013, 380, B, B), (14407, 500, H, H), (13001, 768, F, F), (13001, 700, B, F), (10303, 1000, F, F),
    (10303, 1001, B, B), (6501, 1500, F, F), (6501, 1500, B, F), (5407, 2000, F, F), (5407, 2000, B, B),
    (2603, 4001, F, F), (2603, 4001, B, F), (1103, 8000, F, F), (1103, 8000, B, B), (803, 9001, F, F),
    (803, 9001, B, B), (67, 17000, B, F),
])
def test_groups_that_walk_rows(gpu_lib, rows, d, tx, tout):
    x, w, b, dy = make(rows, d, tx, tout, rows + d)
    y, grads = run(x, w, b, dy, True, 0.1, 7, tout)
    check_all(x, w, b, dy, y, grads, 1e-5, True, 0.1, ref.keep_mask(range(rows), d, 0.1, 7))


@pytest.mark.parametrize("rows,d,tx", [(13001, 768, F), (5407, 2000, F), (1103, 8000, B), (803, 9001, F)])
def test_plain_norm_of_groups_that_walk_rows(gpu_lib, rows, d, tx):
    x, w, b, dy = make(rows, d, tx, tx, rows)
    y, grads = run(x, w, b, dy, False, 0.0, None, tx)
    check_all(x, w, b, dy, y, grads, 1e-5, False, 0.0, None)
