"""That the bounds on fp32 attention over an eight-bit cache (tests/test_gpu_fp8_edges.py) tell a kernel that holds q or the weights in fewer than fp32's 24 bits
from one that holds all: on the CPU, the definition with q or the weights cut to their first bf16 numbers."""
import pytest
import torch

from test_gpu_fp8_edges import PINNED, pinned_scores


def first(parts):
    """x as the sum of that many bf16 numbers, each the nearest to what those before leave."""
    def cut(x):
        left, total = x.float(), torch.zeros_like(x, dtype=torch.float64)
        for _ in range(parts):
            part = left.to(torch.bfloat16).float()
            left, total = left - part, total + part.double()
        return total
    return cut


@pytest.mark.parametrize("make,a", PINNED)
def test_bounds_tell_lost_bits(make, a):
    c = make(*a)
    assert c.holds(c.result(first(3), first(3)))  # three hold them all
    for parts in (1, 2):
        if make is pinned_scores:
            assert not c.holds(c.result(cut_q=first(parts)))
        else:
            assert not c.holds(c.result(cut_weights=first(parts)))
