"""Values at the ends of FP32's range, hidden outliers and subnormals in the paged 4-bit cache, on the GPU."""
from __future__ import annotations

import math

import pytest
import torch

import paged_w4_plain as plain
from test_paged_w4_gpu import _attend, _attention_state, _check_attention

pytestmark = pytest.mark.gpu
I32, I64, BF = torch.int32, torch.int64, torch.bfloat16


@pytest.mark.parametrize("NKV,ratio,hs", [(2, 1, 64), (1, 8, 128), (2, 4, 128), (1, 16, 64)])
def test_attention_of_flat_groups_beside_tiny_steps(cuda, NKV, ratio, hs):
    """Half of V's positions hold one large value a group (step 0), the others values and steps near 2^-112."""
    NH, qkv, codes, scales, table, lens, start = _attention_state(NKV, ratio, hs, 16, [200, 33], [2, 1], 71)
    flat = torch.rand(scales.shape[0], 1, 16, 1, generator=torch.Generator().manual_seed(1)) < 0.5
    step, low = scales[:, 1, ..., 0].float(), scales[:, 1, ..., 1].float()
    scales[:, 1, ..., 0] = torch.where(flat, step * 0, step * 2.0 ** -112).to(BF)
    scales[:, 1, ..., 1] = torch.where(flat, low * 2.0 ** 40, low * 2.0 ** -112).to(BF)
    st = (NH, qkv, codes, scales, table, lens, start)
    _check_attention(st, _attend(st, 2))


@pytest.mark.parametrize("NKV,ratio,hs", [(2, 1, 64), (1, 8, 128), (2, 4, 128), (1, 16, 64)])
@pytest.mark.parametrize("length", [200, 20011])
def test_attention_of_values_near_the_largest(cuda, NKV, ratio, hs, length):
    """Steps near 2^123, values near 2^126: small weights still count, and sums over many positions do not overflow."""
    st = _attention_state(NKV, ratio, hs, 16, [length, 33], [2, 1], 72, q_scale=2.0)
    st[3][:, 1] = (st[3][:, 1].float() * 2.0 ** 124).to(BF)
    _check_attention(st, _attend(st, 2))


@pytest.mark.parametrize("NKV,ratio,hs,bs", [(2, 1, 64, 16), (1, 8, 128, 32), (2, 4, 64, 16), (2, 4, 128, 64), (3, 1, 128, 16)])
@pytest.mark.parametrize("power", [20, 24, 30, 40, 60])
def test_attention_does_not_feel_hidden_outliers(cuda, NKV, ratio, hs, bs, power):
    """V at a draft's own position is 2^power larger: the rows before it, which do not see it, have the same bits as
    with nothing there; the row that sees it has its own values."""
    lens, rows = [70, 45, 300], [5, 3, 2]
    NH, qkv, codes, scales, table, lens, start = _attention_state(NKV, ratio, hs, bs, lens, rows, 73)
    large, none = scales.clone(), scales.clone()
    for b, n in enumerate(lens.tolist()):
        at = (int(table[b, (n - 1) // bs]), 1, slice(None), (n - 1) % bs)
        large[at] = (scales[at].float() * 2.0 ** power).to(BF)
        none[at] = 0
    hidden = [0, 1, 2, 3, 5, 6, 8]
    st = (NH, qkv, codes, large, table, lens, start)
    out = _attend(st, 5)
    clean = (NH, qkv, codes, none, table, lens, start)
    without = _attend(clean, 5)
    assert torch.equal(out[hidden], without[hidden])
    _check_attention(clean, without)
    _check_attention(st, out)


def _append(x, hs):
    """x [rows, 2 NKV hs] appended to a fresh cache, one row a slot: (codes, scales) [rows, 2, NKV, ...]."""
    from cuda_gpt2_inference_b200 import ops
    rows, NKV = x.shape[0], x.shape[1] // (2 * hs)
    nb = -(-rows // 16)
    codes = torch.zeros(nb, 2, NKV, 16, hs // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(nb, 2, NKV, 16, hs // 64, 2, dtype=BF, device="cuda")
    qkv = torch.cat([torch.zeros(rows, NKV * hs, dtype=BF), x], 1).cuda()
    ops.kv_cache_write_w4(codes, scales, qkv, torch.arange(rows, device="cuda"), NKV)
    return [t.cpu().transpose(2, 3).transpose(1, 2).flatten(0, 1)[:rows] for t in (codes, scales)]


def _check_codes(x, hs, codes, scales):
    """Steps and low ends as defined, to the bit; a code differs from its 64-bit form only where the quotient is near
    a half: within 2^-17 (those are ties) and what its arithmetic is off by, 2^-18 (a reciprocal of 2 units in the
    last place at most, 2^-22 of a quotient below 15.5)."""
    want_c, want_s = plain.quantise(x.view(x.shape[0], 2, -1, hs))
    assert torch.equal(scales.view(torch.int16), want_s.view(torch.int16))
    g = x.view(x.shape[0], 2, -1, hs // 64, 64).double()
    step, low = want_s[..., 0:1].double(), want_s[..., 1:2].double()
    q = torch.where(step > 0, (g - low) / step, torch.zeros_like(g)).clamp(0, 15)
    got, want = (torch.stack([c & 15, c >> 4], -1).flatten(-2).view(g.shape).double() for c in (codes, want_c))
    near = (q - q.floor() - 0.5).abs() <= 2.0 ** -17 + 2.0 ** -18
    assert ((got == want) | near).all()
    assert ((got - q).abs() <= 0.5 + 2.0 ** -17 + 2.0 ** -18).all()


@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("power", [0, -60, -112, 100])
@pytest.mark.parametrize("offset", [0.0, 3.0, 100.0])
def test_codes_differ_only_at_ties(cuda, hs, power, offset):
    x = ((torch.randn(500, 4 * hs, generator=torch.Generator().manual_seed(hs)) + offset) * 2.0 ** power).to(BF)
    _check_codes(x, hs, *_append(x, hs))


def test_append_of_subnormal_values(cuda):
    """BF16 subnormals count: beside a step of 2^-119 they decide a quotient's half, and as an end of their group the step."""
    g = torch.Generator().manual_seed(5)
    tiny = torch.randint(-127, 128, (300, 128), generator=g) * 2.0 ** -133
    x = tiny.clone()
    x[:, 0::64], x[:, 1::64] = -15 * 2.0 ** -120, 15 * 2.0 ** -120  # quotients of the others: 7.5 +- up to 2^-7
    x = x.to(BF)
    _check_codes(x, 64, *_append(x, 64))
    low = -(1 + torch.rand(300, 128, generator=g)) * 2.0 ** -116
    x = torch.where(torch.arange(128) % 64 < 40, low, tiny).to(BF)  # the largest of a group is subnormal
    _check_codes(x, 64, *_append(x, 64))


@pytest.mark.parametrize("power", [-119, -125, -130, -133])
def test_read_back_of_subnormal_values(cuda, power):
    """Values of a flat group, and low ends below a step, are read back as they are held."""
    from cuda_gpt2_inference_b200 import ops
    g = torch.Generator().manual_seed(6)
    codes = torch.randint(0, 256, (2, 2, 1, 16, 32), generator=g, dtype=torch.uint8)
    scales = torch.zeros(2, 2, 1, 16, 1, 2)
    scales[..., 1] = torch.randint(-127, 128, scales.shape[:-1], generator=g) * 2.0 ** power
    scales[1, ..., 0] = 2.0 ** -120
    scales = scales.to(BF)
    out = torch.zeros(32, 2, 1, 64, dtype=BF, device="cuda")
    ops.kv_cache_read_w4(out, codes.cuda(), scales.cuda(), torch.arange(32, device="cuda"))
    want = plain.values(codes, scales).transpose(2, 3).transpose(1, 2).flatten(0, 1)
    # one rounding in 32 bits and one in BF16, of a value or of the smallest subnormals
    assert ((out.cpu().double() - want).abs() <= plain.BF16 * (1 + 2.0 ** -15) * want.abs() + 2.0 ** -134 + 2.0 ** -149).all()


@pytest.mark.parametrize("NKV,ratio,hs,bs", [(2, 1, 64, 16), (1, 8, 128, 32), (2, 4, 64, 16), (2, 4, 128, 64), (3, 1, 128, 16)])
@pytest.mark.parametrize("factor", [0.0, 5.0, 100.0, -1e6])
@pytest.mark.parametrize("lens,rows", [([70, 45, 300, 33], [5, 3, 4, 3]), (list(range(290, 322)), [4] * 32)])
def test_attention_rows_do_not_depend_on_later_drafts(cuda, monkeypatch, NKV, ratio, hs, bs, factor, lens, rows):
    """Keys and values at the last two drafts' own positions change: the rows before them keep their bits."""
    values = plain.values

    def with_negative_steps(codes, scales, magnitude=False):  # (what bounds the errors is |code * step| + |low end|)
        return values(codes, torch.stack([scales[..., 0].abs(), scales[..., 1]], -1) if magnitude else scales, magnitude)

    monkeypatch.setattr(plain, "values", with_negative_steps)
    NH, qkv, codes, scales, table, lens, start = _attention_state(NKV, ratio, hs, bs, lens, rows, 74)
    other = scales.clone()
    for b, n in enumerate(lens.tolist()):
        for p in (n - 1, n - 2):
            at = (int(table[b, p // bs]), slice(None), slice(None), p % bs)
            other[at] = (scales[at].float() * factor).to(BF)
    outs = [_attend((NH, qkv, codes, s, table, lens, start), 5) for s in (scales, other)]
    before = torch.cat([torch.arange(int(start[b]), int(start[b + 1]) - 2) for b in range(len(rows))])
    assert torch.equal(outs[0][before], outs[1][before])
    _check_attention((NH, qkv, codes, other, table, lens, start), outs[1])


@pytest.mark.parametrize("NKV,ratio,hs", [(2, 1, 64), (1, 8, 128), (2, 4, 128)])
@pytest.mark.parametrize("at", [0, 5, 290])
def test_attention_of_a_key_of_minus_infinity(cuda, NKV, ratio, hs, at):
    """A score of -infinity is a weight of 0, not a hidden position: V counts there as 0 times what it holds, in a step
    that all rows see and in one that they do not."""
    lens, rows = [300], [3]
    NH, qkv, codes, scales, table, lens, start = _attention_state(NKV, ratio, hs, 16, lens, rows, 75)
    qkv = qkv.abs()
    place = (int(table[0, at // 16]), 0, slice(None), at % 16)
    codes[place] = 0
    scales[place] = torch.tensor([0.0, -math.inf]).to(BF)
    st = (NH, qkv, codes, scales, table, lens, start)
    out = _attend(st, 3)
    want = plain.attention(qkv, codes, scales, table, lens, start, NH)[0]
    err = plain.attention(qkv, codes, torch.nan_to_num(scales, neginf=0.0), table, lens, start, NH)[1]  # (no infinite bound)
    off = (out[:3].cpu().double() - want[:3]).abs()
    assert (off <= plain.BF16 * want[:3].abs() + 1.01 * err[:3] + 2.0 ** -126).all()
    scales[(place[0], 1, *place[2:])] = math.nan
    assert _attend(st, 3)[:3].isnan().all()


@pytest.mark.parametrize("NKV,ratio,hs,bs", [(2, 4, 128, 32), (3, 1, 64, 16)])
def test_attention_of_prompt_pieces(cuda, NKV, ratio, hs, bs):
    """Hundreds of rows a request, with and without a past, beside a decoding request and one with nothing."""
    st = _attention_state(NKV, ratio, hs, bs, [700, 512, 130, 0, 333], [512, 512, 101, 0, 1], 76)
    _check_attention(st, _attend(st, 512))
