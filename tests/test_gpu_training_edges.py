"""Edges of the training operators: calls and values that their other tests leave out."""
import math

import pytest
import torch

from test_gpu_training_operators import BF16, check, check_linear, linear_inputs, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k,n,act", [(256, 128, "silu"), (200, 256, "gelu"), (128, 384, None), (128, 512, "silu"), (72, 264, "relu")])
@pytest.mark.parametrize("tiles", [148, 149, 222, 223, 300])
def test_paired_backward_ends_after_any_number_of_tiles(k, n, act, tiles):
    """Two CTAs share a layer's k, and each waits at its end for the other's last arrivals at the slots that were used: slots used
    once, twice, an even and an odd number of times, and not at all.  A wait for a phase that never comes would be in the status."""
    from bioemu2_b200 import training as t

    rows = tiles * 128 - 5
    g, x, w = linear_inputs(rows, k, n, BF16)
    dy = (randn(g, rows, n) / math.sqrt(rows)).bfloat16()
    check_linear(x, w, randn(g, n), act, None, dy)
    pre = None if act is None else randn(g, rows, n).bfloat16()
    first = t.linear_backward(dy, x, w, pre, act)
    for _ in range(20):  # one launch behind the other: what one leaves on its way would land in the next one's
        last = t.linear_backward(dy, x, w, pre, act)
    check("status", first[2], first[2].double(), torch.zeros_like(first[2], dtype=torch.float64))
    assert all(torch.equal(a, b) for a, b in zip(first, last))
