"""Probabilities and verification of drafted tokens on the GPU, against plain 64-bit forms."""
from __future__ import annotations

import math

import pytest
import torch

import paged_w4_plain as plain

pytestmark = pytest.mark.gpu
I32 = torch.int32


# ------------------------------------------------------------- probabilities ----
def _probs(x, T, V=None, inplace=False):
    from cuda_gpt2_inference_b200 import ops
    d = x.cuda()
    out = d if inplace else torch.full_like(d, -7.0)
    ops.softmax_probs(out, d, T, V=V)
    return out.cpu()


@pytest.mark.parametrize("rows,V", [(1, 1), (1, 2), (3, 31), (2, 1000), (5, 4097), (3, 50257), (2, 131072), (1, 300001), (400, 63)])
@pytest.mark.parametrize("T", [1.0, 0.3, 5.0])
@pytest.mark.parametrize("spread", [3.0, 60.0])
def test_probs(cuda, rows, V, T, spread):
    x = torch.randn(rows, V, generator=torch.Generator().manual_seed(V)) * spread
    x[:, V // 3] = torch.finfo(torch.float32).min  # a masked token
    x[:, V // 2] = -math.inf
    if V < 3:
        x = torch.zeros(rows, V)
    got = _probs(x, T).double()
    z = x.double() / T
    z = z - z.amax(-1, keepdim=True)
    want = torch.exp(z)
    total = want.sum(-1, keepdim=True)
    want = want / total
    # (x - max)/T: two roundings of its value, an e^x of 2^-21, the sum's (pairwise over threads) and the quotient's
    rel = 2.0 ** -24 * 3 * z.abs().clamp(max=104) + 2.0 ** -21 + 2.0 ** -24 * (V / 256 + 40)
    assert ((got - want).abs() <= rel * want + 2.0 ** -126).all()
    assert torch.equal(_probs(x, T, inplace=True).double(), got)


def test_probs_greedy_ties_masks_and_columns(cuda):
    x = torch.randn(4, 999, generator=torch.Generator().manual_seed(1))
    x[0, 500] = x[0, 77] = 9.0
    x[1] = -math.inf
    x[2, 3] = math.nan
    x[3, 998] = 50.0
    got = _probs(x, 0.0)
    want = torch.zeros(4, 999)
    want[0, 77] = want[3, 998] = 1
    want[2, int(torch.nan_to_num(x[2], nan=-9.0).argmax())] = 1
    assert torch.equal(got, want)
    got = _probs(x, 1.0)
    assert not got[1].any() and got[2].isnan().all() and torch.isfinite(got[[0, 3]]).all()
    x[0, 5] = math.inf
    assert _probs(x, 1.0)[0].isnan().all()
    # columns behind V are neither read nor written
    x = torch.randn(3, 700, generator=torch.Generator().manual_seed(2))
    ref = torch.softmax(x[:, :601].double(), -1)
    x[:, 601:] = math.nan
    got = _probs(x, 1.0, V=601)
    assert (got[:, 601:] == -7).all()
    assert ((got[:, :601].double() - ref).abs() <= 2.0 ** -19 * ref).all()
    # rows of a wider buffer at an odd pitch and offset
    from cuda_gpt2_inference_b200 import ops
    wide = torch.full((3, 907), math.nan, device="cuda")
    wide[:, 3:604] = x[:, :601].cuda()
    out = torch.full((3, 613), -7.0, device="cuda")
    ops.softmax_probs(out[:, 1:602], wide[:, 3:604])
    assert torch.equal(out[:, 1:602].cpu(), got[:, :601]) and (out[:, 602:] == -7).all() and (out[:, 0] == -7).all()


# -------------------------------------------------------------- verification ----
def _run(tokens, p, q, start, ua, us, max_out):
    from cuda_gpt2_inference_b200 import ops
    B = len(start) - 1
    out = torch.full((B, max_out), -7, dtype=I32, device="cuda")
    n = torch.full((B,), -7, dtype=I32, device="cuda")
    ops.verify_draft_tokens(out, n, tokens.to(I32).cuda(), p.cuda(), None if q is None else q.cuda(),
                            torch.tensor(start, dtype=I32, device="cuda"), ua.cuda(), us.cuda())
    return out.tolist(), n.tolist()


def _state(rows, V, seed, spread=2.0, near=0.5):
    g = torch.Generator().manual_seed(seed)
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    R = start[-1] + 2  # padding rows
    x = torch.randn(R, V, generator=g) * spread
    p = torch.softmax(x, -1)
    q = torch.softmax(x + near * torch.randn(R, V, generator=g), -1)
    tokens = torch.multinomial(q, 1, generator=g)[:, 0].roll(1)
    return tokens, p, q, start, torch.rand(R, generator=g), torch.rand(len(rows), generator=g)


@pytest.mark.parametrize("V", [1, 2, 33, 1000, 4099, 50257, 131072])
@pytest.mark.parametrize("rows", [[1], [5], [1, 2, 9, 1, 4], [0, 3, 0, 2], [40]])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(cuda, gpt2b, V, rows, certain):
    for seed in range(3):
        tokens, p, q, start, ua, us = _state(rows, V, seed + V, near=0.2 if seed else 3.0)
        args = (tokens, p, None if certain else q, start, ua * (0.05 if seed == 2 else 1.0), us, max(rows) + 1)
        got = _run(*args)
        assert got == plain.verify(*args)
    assert gpt2b.device_error() == 0


@pytest.mark.parametrize("u", [0.0, 1.0, 0.5, math.nan, -1.0, 2.0])
def test_verify_borders(cuda, u):
    """Weights of zero at both ends, a draw at the border of a token, random numbers at and beyond their range."""
    V = 2000
    p = torch.zeros(6, V)
    p[:, 100], p[:, 1500] = 0.5, 0.5
    p[2] = 0  # no weight at all
    p[3, 3] = math.nan  # counts as nothing
    q = torch.zeros(6, V)
    q[0, 1500] = 1.0
    q[4] = p[4]
    q[4, 100] = 0.75  # draft above target everywhere: refused, and nothing is left of the target
    tokens = torch.tensor([0, 1500, 0, 0, 0, 100])
    ua = torch.tensor([0.6, 0, 0, 0, 0.9, 0])
    for qq in (q, None):
        args = (tokens, p, qq, [0, 2, 3, 4, 6], ua, torch.full((4,), u), 3)
        got, taken = _run(*args)
        assert (got, taken) == plain.verify(*args)
        assert got[1][0] == -1


def test_verify_greedy_by_one_hot_probabilities(cuda):
    """Temperature 0: the longest run of drafts that are the target's own picks, then its next pick."""
    from cuda_gpt2_inference_b200 import ops
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(6, 5000, generator=g)
    best = logits.argmax(-1)
    p = torch.empty(6, 5000, device="cuda")
    ops.softmax_probs(p, logits.cuda(), 0.0)
    tokens = torch.tensor([9, int(best[0]), int(best[1]), 17, int(best[3]), 5])
    got = _run(tokens, p.cpu(), None, [0, 6], torch.rand(6, generator=g), torch.rand(1, generator=g), 7)
    assert got == ([[int(best[0]), int(best[1]), int(best[2]), -1, -1, -1, -1]], [2])


def test_verify_short_outputs_bad_drafts_and_offsets(cuda, gpt2b):
    tokens, p, q, start, ua, us = _state([9, 6], 700, 5, near=0.01)
    ua = ua * 0.5
    for max_out in (1, 2, 4):
        args = (tokens, p, q, start, ua, us, max_out)
        assert _run(*args) == plain.verify(*args)
    for bad in (-1, 700, 2 ** 31 - 1, -2 ** 31):
        t = tokens.clone()
        t[3] = bad
        args = (t, p, q, start, ua, us, 9)
        assert _run(*args) == plain.verify(*args)
    torch.cuda.synchronize()
    assert gpt2b.device_error() == 0
    got = _run(tokens, p, q, [0, 9, 99], ua, us, 20)
    assert gpt2b.device_error() == gpt2b.DEVERR_BAD_POS
    assert got == plain.verify(tokens, p, q, [0, 9, 17], ua, us, 20)
    got = _run(tokens, p, q, [5, 3, 2], ua, us, 20)
    assert gpt2b.device_error() == gpt2b.DEVERR_BAD_POS
    assert got == plain.verify(tokens, p, q, [5, 5, 5], ua, us, 20)[0:2]


def test_verify_draws_from_the_target(cuda):
    """Accepted or redrawn, the first token's frequencies are the target's (64-bit probabilities of 6 tokens,
    40000 requests: five standard deviations of a count)."""
    g = torch.Generator().manual_seed(6)
    V, B = 6, 40000
    p1, q1 = torch.softmax(torch.randn(V, generator=g), 0), torch.softmax(torch.randn(V, generator=g), 0)
    p, q = p1.repeat(2 * B, 1), q1.repeat(2 * B, 1)
    tokens = torch.multinomial(q1, 2 * B, replacement=True, generator=g)
    got, _ = _run(tokens, p, q, list(range(0, 2 * B + 1, 2)), torch.rand(2 * B, generator=g), torch.rand(B, generator=g), 2)
    count = torch.bincount(torch.tensor([r[0] for r in got]), minlength=V).double()
    sd = (B * p1.double() * (1 - p1.double())).sqrt()
    assert ((count - B * p1.double()).abs() <= 5 * sd).all()


def test_verify_in_a_graph(cuda):
    from cuda_gpt2_inference_b200 import ops
    tokens, p, q, start, ua, us = _state([4, 1, 6], 5000, 7)
    d = [t.cuda() for t in (tokens.to(I32), p, q, torch.tensor(start, dtype=I32), ua, us)]
    probs = torch.empty_like(d[1])
    logits = torch.log(d[1])
    out, n = torch.full((3, 7), -7, dtype=I32, device="cuda"), torch.full((3,), -7, dtype=I32, device="cuda")

    def step():
        ops.softmax_probs(probs, logits)
        ops.verify_draft_tokens(out, n, d[0], probs, d[2], d[3], d[4], d[5])

    step()
    want = out.clone(), n.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
        step()
    out.fill_(-7), n.fill_(-7), probs.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(n, want[1])
    ua2 = torch.rand_like(d[4])
    d[4].copy_(ua2)  # new numbers, same graph
    graph.replay()
    torch.cuda.synchronize()
    assert (out.tolist(), n.tolist()) == plain.verify(tokens, probs.cpu(), q, start, ua2.cpu(), us, 7)


def test_probs_beside_their_logits(cuda):
    """Logits and probabilities as columns of one buffer."""
    from cuda_gpt2_inference_b200 import ops
    both = torch.zeros(7, 2 * 333 + 5, device="cuda")
    x = torch.randn(7, 333, generator=torch.Generator().manual_seed(3))
    both[:, :333] = x.cuda()
    ops.softmax_probs(both[:, 336:669], both[:, :333])
    want = torch.softmax(x.double(), -1)
    assert ((both[:, 336:669].cpu().double() - want).abs() <= 2.0 ** -20 * want).all()
    assert torch.equal(both[:, :333].cpu(), x) and not both[:, 333:336].any() and not both[:, 669:].any()


def test_sizes_beyond_32_bits_are_refused(cuda, gpt2b):
    """Empty tensors hold no memory and may have any size; the refusal is an error of the call, which the next
    call does not see."""
    from cuda_gpt2_inference_b200 import ops
    many = torch.empty(2 ** 31, 0, device=cuda)
    with pytest.raises(gpt2b.Gpt2bError, match="32 bits"):
        ops.softmax_probs(many, many, V=0)
    one = torch.empty(0, dtype=torch.int32, device=cuda)
    with pytest.raises(gpt2b.Gpt2bError, match="32 bits"):
        ops.verify_draft_tokens(torch.empty(0, 2 ** 31, dtype=torch.int32, device=cuda), one, one,
                                torch.empty(0, 8, device=cuda), None, torch.zeros(1, dtype=torch.int32, device=cuda),
                                one.float(), one.float())
    logits = torch.zeros(1, 4, device=cuda)
    ops.softmax_probs(logits, logits)
    assert logits.tolist() == [[0.25] * 4]
