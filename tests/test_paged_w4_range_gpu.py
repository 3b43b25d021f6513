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
