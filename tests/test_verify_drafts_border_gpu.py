"""Draws at the border of a CTA's part of the vocabulary, on the GPU, against exact sums."""
from __future__ import annotations

from fractions import Fraction

import pytest
import torch

import paged_w4_plain as plain
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


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("u", [0.0, 0.3, 1.0, 2.0 ** -140])
def test_subnormal_probabilities_count(cuda, certain, u):
    """Probabilities below FP32's normal range: they are accepted against 0, are what is left of a target, and are drawn."""
    V = 300
    p, q = torch.zeros(8, V), torch.zeros(8, V)
    p[0, 7] = 2.0 ** -140                         # a draft as likely as nothing else: accepted at u 0
    p[1, 5:9] = torch.tensor([1.0, 2, 3, 4]) * 2.0 ** -149  # a row of subnormals alone
    p[2, 40], q[2, 40] = 0.5, 0.5                 # all that is left of the target is subnormal
    p[2, 90] = p[2, 200] = 2.0 ** -135
    p[3, 1] = 1.0
    p[4, 11], q[4, 11] = 2.0 ** -130, 2.0 ** -131
    p[5, 250] = 2.0 ** -127
    p[6, 0] = p[6, 299] = 2.0 ** -128
    tokens = torch.tensor([0, 7, 0, 40, 0, 11, 0, 0])
    args = (tokens, p, None if certain else q, [0, 2, 4, 6, 7], torch.full((8,), u), torch.full((4,), u), 3)
    assert _run(*args) == plain.verify(*args)


@pytest.mark.parametrize("rows,V", [(1, 40), (3, 50257)])
def test_greedy_among_subnormal_logits(cuda, rows, V):
    """Logits that differ by a subnormal are no tie."""
    from cuda_gpt2_inference_b200 import ops
    x = torch.zeros(rows, V)
    x[:, V // 3], x[:, V // 2], x[:, V - 2] = 2.0 ** -149, 3 * 2.0 ** -149, 3 * 2.0 ** -149
    x[0] -= 0.0
    x[-1, 5] = -(2.0 ** -140)
    out = torch.full((rows, V), -7.0, device="cuda")
    ops.softmax_probs(out, x.cuda(), 0.0)
    want = torch.zeros(rows, V)
    want[:, V // 2] = 1
    assert torch.equal(out.cpu(), want)
