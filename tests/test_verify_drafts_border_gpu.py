"""Draws at the border of a CTA's part of the vocabulary, on the GPU, against exact sums."""
from __future__ import annotations

from fractions import Fraction

import pytest
import torch

from test_verify_drafts_gpu import _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tiny", [2.0 ** -53, 2.0 ** -54, 1.5 * 2.0 ** -54])
@pytest.mark.parametrize("every", [1, 37, 393])
def test_draw_at_a_border_that_rounding_moves(cuda, tiny, every):
    """Half of the weight in front, then many weights too small to move a sum of 1 one at a time but not together,
    and the other half in two tokens far behind.  The draw is half of the total: it lies among the small ones, whatever
    the order of the sums."""
    V = 50257
    p = torch.zeros(1, V)
    p[0, 10] = 1.0
    p[0, 6283:12566:every] = tiny
    p[0, 45000] = p[0, 50000] = 0.5
    got, taken = _run(torch.zeros(1), p, None, [0, 1], torch.zeros(1), torch.tensor([0.5]), 1)
    pick = got[0][0]
    w = [Fraction(float(x)) for x in p[0, :pick + 1]]
    total, below = sum(Fraction(float(x)) for x in p[0] if x), sum(w[:-1])
    # a sum of n weights in 64 bits, in any order, is off by n 2^-53 of it at most; n: weights, and the parts' sums
    n = int((p > 0).sum()) + 8 * 16
    slack = total * n / 2 ** 53 if every == 1 else total * 64 / 2 ** 53
    assert w[-1] > 0 and taken == [0]
    assert below <= total / 2 + slack and below + w[-1] >= total / 2 - slack
