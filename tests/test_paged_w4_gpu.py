"""Batches of requests over the paged 4-bit KV cache, on the GPU, against plain 64-bit forms."""
from __future__ import annotations

import math

import pytest
import torch

import paged_w4_plain as plain

pytestmark = pytest.mark.gpu
I32, I64, BF = torch.int32, torch.int64, torch.bfloat16


def i32(v):
    return torch.tensor(v, dtype=I32, device="cuda")


@pytest.fixture(autouse=True)
def _no_device_error(cuda, gpt2b):
    gpt2b.device_error()
    yield
    torch.cuda.synchronize()


# ------------------------------------------------------ append and read-back ----
def _rows(rows, width, seed, kind):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g)
    if kind == "large":
        x = x * 1e30
    elif kind == "small":
        x = x * 2.0 ** -118
    elif kind == "flat":
        x = torch.full_like(x, -2.5)
    elif kind == "range":  # the range of a group passes FP32's
        x = torch.where(x > 0, 3.3e38, -3.3e38) * (0.25 + 0.75 * torch.rand(rows, width, generator=g))
    elif kind == "shifted":
        x = x * 0.125 + 100
    return x.to(BF)


@pytest.mark.parametrize("NKV,ratio,hs,bs", [(12, 1, 64, 16), (1, 1, 64, 16), (3, 4, 64, 48), (2, 8, 128, 16), (5, 1, 128, 32)])
@pytest.mark.parametrize("rows", [1, 7, 100])
@pytest.mark.parametrize("kind", ["normal", "large", "small", "flat", "range", "shifted"])
def test_append_holds_the_defined_codes(cuda, gpt2b, NKV, ratio, hs, bs, rows, kind):
    from cuda_gpt2_inference_b200 import ops
    NH, nb = NKV * ratio, -(-rows // bs) + 2
    x = _rows(rows, (NH + 2 * NKV) * hs, rows + hs, kind)
    g = torch.Generator().manual_seed(rows)
    slots = torch.randperm(nb * bs, generator=g)[:rows]
    if rows > 3:
        slots[3] = -1
    codes = torch.full((nb, 2, NKV, bs, hs // 2), 0xA5, dtype=torch.uint8)
    scales = torch.full((nb, 2, NKV, bs, hs // 64, 2), 7.0, dtype=BF)
    dc, ds = codes.cuda(), scales.cuda()
    ops.kv_cache_write_w4(dc, ds, x.cuda(), slots.cuda(), NH)
    kv = x[:, NH * hs:].view(rows, 2, NKV, hs)
    want_c, want_s = plain.quantise(kv)
    keep = slots >= 0
    codes[slots[keep] // bs, :, :, slots[keep] % bs] = want_c[keep]
    scales[slots[keep] // bs, :, :, slots[keep] % bs] = want_s[keep]
    # the step of subnormal-range groups may differ where the products underflow; there the values are compared below
    got_c, got_s = dc.cpu(), ds.cpu()
    assert torch.equal(got_s.view(torch.int16), scales.view(torch.int16)) or kind == "small"
    # quotients within 2^-17 of a half count as one: codes differ from the 64-bit form's only there, by one
    diff = torch.stack([got_c & 15, got_c >> 4]).int() - torch.stack([codes & 15, codes >> 4]).int()
    assert diff.abs().max() <= 1
    assert (diff != 0).float().mean() < 1e-3
    # read-back: one rounding of code * step + low end
    out = torch.full((rows, 2, NKV, hs), 9.0, dtype=BF, device="cuda")
    ops.kv_cache_read_w4(out, dc, ds, slots.cuda())
    safe = slots.clamp(min=0)
    v = plain.values(got_c[safe // bs, :, :, safe % bs], got_s[safe // bs, :, :, safe % bs])
    v[~keep] = 0
    want = v.to(torch.float32).to(BF)
    got = out.cpu()
    assert torch.isfinite(got.float()).all()
    assert ((got.double() - v).abs() <= plain.BF16 * v.abs() * (1 + 2.0 ** -14) + 2.0 ** -126).all()
    assert (got != want).float().mean() < 1e-2
    # and it is near what was appended: half a step, and at the top what the rounded step misses
    step = got_s[safe // bs, :, :, safe % bs][..., 0].double().repeat_interleave(64, -1)
    bound = step * (0.5 + 15 * plain.BF16 + 2.0 ** -10) + plain.BF16 * v.abs() + 2.0 ** -116
    assert ((got.double() - kv.double()).abs() <= bound)[keep].all()
    assert gpt2b.device_error() == 0


def test_append_of_non_finite_groups_and_bad_slots(cuda, gpt2b):
    from cuda_gpt2_inference_b200 import ops
    NH, hs, bs, nb = 2, 128, 16, 2
    x = torch.randn(4, 3 * NH * hs)
    x[0, NH * hs + 5] = math.nan
    x[1, NH * hs + 70] = math.inf
    x[2, 2 * NH * hs + 1] = -math.inf
    x = x.to(BF).cuda()
    dc = torch.zeros(nb, 2, NH, bs, hs // 2, dtype=torch.uint8, device="cuda")
    ds = torch.zeros(nb, 2, NH, bs, hs // 64, 2, dtype=BF, device="cuda")
    slots = torch.tensor([3, 4, 5, nb * bs], device="cuda")  # the last one is outside
    ops.kv_cache_write_w4(dc, ds, x, slots, NH)
    torch.cuda.synchronize()
    assert gpt2b.device_error() == gpt2b.DEVERR_BAD_BLOCK
    out = torch.zeros(4, 2, NH, hs, dtype=BF, device="cuda")
    ops.kv_cache_read_w4(out, dc, ds, slots)
    torch.cuda.synchronize()
    assert gpt2b.device_error() == gpt2b.DEVERR_BAD_BLOCK
    bad = torch.zeros(4, 2, NH, hs, dtype=torch.bool)
    bad[0, 0, 0, :64] = bad[1, 0, 0, 64:] = bad[2, 1, 0, :64] = True  # the group alone
    assert torch.equal(out.cpu().isnan(), bad)
    assert not out[3].any() and not dc[:, :, :, 6:].any()


# ---------------------------------------------------------------- tables ----
def _run_tables(table, ctx, new, have, free, count, bs, max_rows):
    from cuda_gpt2_inference_b200 import ops
    B = len(ctx)
    t = i32(table)
    slot = torch.full((max_rows,), -7, dtype=I64, device="cuda")
    pos, start, lens, blocks, left = (torch.full((n,), -7, dtype=I32, device="cuda") for n in (max_rows, B + 1, B, B, 1))
    args = (t, slot, pos, start, lens, blocks, left, i32(ctx), i32(new), i32(have),
            i32(free) if free else torch.empty(0, dtype=I32, device="cuda"), i32([count]), bs)
    ops.kv_block_tables(*args)
    ops.kv_block_tables(*args)  # again: the same result
    return [x.tolist() for x in (t, slot, pos, start, lens, blocks)] + [int(left)]


@pytest.mark.parametrize("B", [1, 2, 31, 257, 1000, 4096])
@pytest.mark.parametrize("bs,mb,most,short", [(16, 8, 1, 0), (16, 40, 60, 0), (32, 4, 40, 5), (1, 9, 4, 30), (48, 3, 150, 0)])
def test_block_tables(cuda, B, bs, mb, most, short):
    import random
    rng = random.Random(B * 100 + bs)
    ctx = [rng.randint(0, mb * bs) for _ in range(B)]
    new = [rng.choice([0, 1, rng.randint(0, most)]) for _ in range(B)]
    have = [min(mb, -(-c // bs) + rng.randint(0, 1)) for c in ctx]
    need = sum(max(0, min(mb, -(-(c + n) // bs)) - h) for c, n, h in zip(ctx, new, have))
    ids = list(range(sum(have) + need + 3))
    rng.shuffle(ids)
    table, at = [], 0
    for h in have:
        table.append(ids[at:at + h] + [-1] * (mb - h))
        at += h
    free = ids[at:]
    count = max(0, len(free) - 3 - short)
    max_rows = max(0, sum(new) + rng.choice([3, 0, -2]))
    got = _run_tables(table, ctx, new, have, free, count, bs, max_rows)
    want = plain.tables(table, ctx, new, have, free, count, bs, max_rows)
    assert got == list(want)


def test_block_tables_of_odd_inputs(cuda):
    # negative lengths count as 0, more blocks than the table has as its width, a count beyond the list as
    # its length; a context far beyond the table is refused
    table = [[5, 6, 7], [8, -1, -1], [-1, -1, -1], [9, -1, -1]]
    args = ([-3, 2 ** 31 - 1, 0, 4], [5, 2 ** 31 - 1, 17, -9], [99, 1, -4, 1], [1, 2, 3], 50, 16, 40)
    assert _run_tables(table, *args) == list(plain.tables(table, *args))
    args = ([0, 0, 0, 0], [1, 1, 1, 1], [0, 0, 0, 0], [], 4, 16, 4)  # nothing free
    got = _run_tables([[-1]] * 4, *args)
    assert got == list(plain.tables([[-1]] * 4, *args)) and got[4] == [0, 0, 0, 0]


# -------------------------------------------------------------- attention ----
CASES = [  # NKV, ratio, hs, bs, lens, rows
    (12, 1, 64, 16, [1], [1]),
    (12, 1, 64, 16, [1000], [1]),
    (2, 1, 64, 16, [15, 16, 17, 31, 32, 33, 127, 128, 129], [1] * 9),
    (2, 1, 128, 16, [1, 63, 64, 65, 257, 511], [1] * 6),
    (1, 8, 128, 32, [300, 0, 5, 77], [4, 1, 5, 0]),
    (5, 3, 64, 48, [200, 2, 0, 600], [5, 4, 3, 1]),        # rows that see nothing
    (2, 4, 128, 16, [130, 700], [8, 3]),
    (3, 1, 64, 64, [100, 640], [20, 33]),
    (1, 16, 64, 16, [333], [3]),
    (2, 1, 128, 16, [40, 90], [40, 17]),                    # a prompt without a past
    (1, 1, 64, 16, [5000], [2]),
    (1, 4, 128, 32, [9001], [1]),
    (2, 1, 64, 96, [500, 97, 96, 95], [2, 1, 1, 3]),
    (1, 3, 128, 160, [1000, 161, 31], [7, 1, 2]),
    (1, 1, 64, 16, list(range(0, 300)), [1] * 300),         # more requests than a pass of the CTA's scan
]


def _attention_state(NKV, ratio, hs, bs, lens, rows, seed, spread=None, q_scale=1.0, pad=3):
    g = torch.Generator().manual_seed(seed)
    NH, held = NKV * ratio, [-(-n // bs) for n in lens]
    nb = sum(held) + 2
    x = torch.randn(nb, 2, NKV, bs, hs, generator=g)
    if spread is not None:
        x = x * 2.0 ** torch.randint(-spread, spread + 1, (nb, 2, NKV, bs, 1), generator=g)
    codes, scales = plain.quantise(x.to(BF))
    order = torch.randperm(nb, generator=g).tolist()
    mb = max(held + [1]) + 2
    # entries behind a request's blocks are never read
    table = torch.randint(-2 ** 31, 2 ** 31 - 1, (len(lens), mb), generator=g).to(I32)
    used = torch.zeros(nb, bs, dtype=torch.bool)
    at = 0
    for b, (n, h) in enumerate(zip(lens, held)):
        table[b, :h] = torch.tensor(order[at:at + h], dtype=I32)
        for j in range(h):
            used[order[at + j], :min(bs, n - j * bs)] = True
        at += h
    # what no request holds is garbage: NaN steps and ends, or infinities
    dead = ~used[:, None, None, :].expand(nb, 2, NKV, bs)
    scales[dead] = torch.where(torch.rand(int(dead.sum()), hs // 64, 2, generator=g) < 0.5, math.nan, math.inf).to(BF)
    R = sum(rows)
    qkv = (torch.randn(R + pad, (NH + 2 * NKV) * hs, generator=g) * q_scale).to(BF)
    start = torch.tensor([0] + rows).cumsum(0).to(I32)
    return NH, qkv, codes, scales, table, torch.tensor(lens, dtype=I32), start


def _attend(st, max_q, scale=None, stream=None, out=None):
    from cuda_gpt2_inference_b200 import ops
    NH, qkv, codes, scales, table, lens, start = st
    NKV, hs = codes.shape[2], codes.shape[4] * 2
    d = [t.cuda() for t in st[1:]]
    out = torch.full((qkv.shape[0], NH * hs), 123.0, dtype=BF, device="cuda") if out is None else out
    ws = torch.full((ops.attention_paged_w4_workspace(NH, NKV, hs, max_q),), 0xFF, dtype=torch.uint8, device="cuda")
    ops.attention_forward_paged_w4(out, *d[:3], d[3], d[4], d[5], NH, max_q, ws, scale=scale, stream=stream)
    return out


def _check_attention(st, out, scale=None):
    NH, qkv, codes, scales, table, lens, start = st
    want, err = plain.attention(qkv, codes, scales, table, lens, start, NH, scale)
    got, R = out.cpu().double(), int(start[-1])
    assert (got[R:] == 123.0).all()  # rows behind the last request
    off = (got[:R] - want[:R]).abs()
    assert torch.isfinite(got[:R]).all()
    tol = plain.BF16 * want[:R].abs() + (1 + plain.BF16) * err[:R] + 2.0 ** -126
    assert (off <= tol).all(), float((off - tol).max())


@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(cuda, gpt2b, case):
    NKV, ratio, hs, bs, lens, rows = CASES[case]
    st = _attention_state(NKV, ratio, hs, bs, lens, rows, case)
    out = _attend(st, max(rows))
    _check_attention(st, out)
    assert gpt2b.device_error() == 0
    # max_q is a hint: a wrong one gives the same values within rounding; the same call the same bits
    for hint in (1, 3, 64):
        _check_attention(st, _attend(st, hint))
    assert torch.equal(out, _attend(st, max(rows)))


@pytest.mark.parametrize("spread,q_scale", [(6, 1.0), (0, 300.0), (0, 1e-30), (3, 0.0), (0, 3e4)])
@pytest.mark.parametrize("hs", [64, 128])
def test_attention_of_uneven_magnitudes(cuda, spread, q_scale, hs):
    """Steps that differ by 2^12 between positions, scores that saturate the softmax, queries of zero."""
    st = _attention_state(2, 2, hs, 16, [333, 40, 1], [3, 2, 1], 5, spread=spread, q_scale=q_scale)
    _check_attention(st, _attend(st, 3))


@pytest.mark.parametrize("factor", [2.0 ** -90, 2.0 ** 60])
def test_attention_of_extreme_values(cuda, factor):
    NH, qkv, codes, scales, table, lens, start = _attention_state(2, 1, 64, 16, [200, 33], [2, 1], 6)
    scales[:, 1] = (scales[:, 1].float() * factor).to(BF)
    st = (NH, qkv, codes, scales, table, lens, start)
    _check_attention(st, _attend(st, 2))


def test_attention_growing_values(cuda):
    """Each later position's values are larger: what was accumulated is rescaled again and again."""
    NH, qkv, codes, scales, table, lens, start = _attention_state(1, 1, 64, 16, [600], [2], 8)
    for j in range(38):
        for o in range(16):
            scales[int(table[0, j]), 1, :, o] = (scales[int(table[0, j]), 1, :, o].float() * 2.0 ** ((16 * j + o) // 8 - 40)).to(BF)
    st = (NH, qkv, codes, scales, table, lens, start)
    _check_attention(st, _attend(st, 2))


def test_attention_scale_strides_and_stream(cuda):
    from cuda_gpt2_inference_b200 import ops
    st = _attention_state(3, 2, 64, 16, [90, 17], [2, 1], 9)
    _check_attention(st, _attend(st, 2, scale=0.3), scale=0.3)
    # rows of a wider buffer, on another stream than the current one
    NH, qkv, codes, scales, table, lens, start = st
    wide = torch.zeros(qkv.shape[0], qkv.shape[1] + 24, dtype=BF, device="cuda")
    view = wide[:, 8:8 + qkv.shape[1]]
    view.copy_(qkv)
    side = torch.cuda.Stream()
    out = torch.full((qkv.shape[0], NH * 64), 123.0, dtype=BF, device="cuda")
    ws = torch.empty(ops.attention_paged_w4_workspace(NH, 3, 64, 2), dtype=torch.uint8, device="cuda")
    d = [t.cuda() for t in st[2:]]
    torch.cuda.synchronize()
    ops.attention_forward_paged_w4(out, view, d[0], d[1], d[2], d[3], d[4], NH, 2, ws, stream=side)
    side.synchronize()
    _check_attention(st, out)


def test_attention_reports_bad_blocks_and_lengths(cuda, gpt2b):
    """A block outside the cache is left out; the other positions and requests are as they were."""
    st = _attention_state(2, 1, 64, 16, [100, 50], [1, 2], 11)
    NH, qkv, codes, scales, table, lens, start = st
    good = _attend(st, 2)
    bad = table.clone()
    bad[0, 2] = codes.shape[0]
    out = _attend((NH, qkv, codes, scales, bad, lens, start), 2)
    torch.cuda.synchronize()
    assert gpt2b.device_error() == gpt2b.DEVERR_BAD_BLOCK
    assert torch.isfinite(out[0]).all() and torch.equal(out[1:], good[1:]) and not torch.equal(out[0], good[0])
    bad[0, :7] = -1  # every block
    out = _attend((NH, qkv, codes, scales, bad, lens, start), 2)
    torch.cuda.synchronize()
    assert gpt2b.device_error() == gpt2b.DEVERR_BAD_BLOCK
    assert not out[0].any() and torch.equal(out[1:], good[1:])
    # a length beyond the table is cut to it and reported
    table[1, 4:] = int(table[1, 0])
    long = lens.clone()
    long[1] = 2 ** 31 - 1
    cut = lens.clone()
    cut[1] = table.shape[1] * 16
    clean = torch.where(torch.isfinite(scales.float()), scales.float(), torch.zeros(())).to(BF)
    table[1, :] = table[1].clamp(0, codes.shape[0] - 1)
    table[0, 7:] = 0
    a = _attend((NH, qkv, codes, clean, table, long, start), 2)
    torch.cuda.synchronize()
    assert gpt2b.device_error() == gpt2b.DEVERR_BAD_POS
    assert torch.equal(a, _attend((NH, qkv, codes, clean, table, cut, start), 2))
    # row offsets outside the rows
    wrong = start.clone()
    wrong[2] = 1000
    out = _attend((NH, qkv, codes, scales, table, lens, wrong), 2)
    torch.cuda.synchronize()
    assert gpt2b.device_error() == gpt2b.DEVERR_BAD_POS
    assert torch.equal(out[0], good[0])


def test_attention_offsets_beyond_32_bits(cuda):
    """Blocks behind 2^32 bytes of codes (and 2^31 code bytes, 2^31 values)."""
    from cuda_gpt2_inference_b200 import ops
    NKV, hs, bs = 8, 128, 64
    per = 2 * NKV * bs * (hs // 2)
    nb = (2 ** 32 + 2 ** 28) // per
    codes = torch.zeros(nb, 2, NKV, bs, hs // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(nb, 2, NKV, bs, 2, 2, dtype=BF, device="cuda")
    g = torch.Generator().manual_seed(1)
    n = 150
    qkv = torch.randn(n, 3 * NKV * hs, generator=g).to(BF)
    blocks = [nb - 1, 2 ** 31 // per, 2 ** 32 // per + 1]
    slots = torch.tensor([blocks[p // bs] * bs + p % bs for p in range(n)])
    ops.kv_cache_write_w4(codes, scales, qkv.cuda(), slots.cuda(), NKV)
    small_c, small_s = codes[blocks].cpu(), scales[blocks].cpu()
    kv = qkv[:, NKV * hs:].view(n, 2, NKV, hs)
    back = torch.empty(n, 2, NKV, hs, dtype=BF, device="cuda")
    ops.kv_cache_read_w4(back, codes, scales, slots.cuda())
    step = small_s.double()[[p // bs for p in range(n)], :, :, [p % bs for p in range(n)]][..., 0].repeat_interleave(64, -1)
    assert ((back.cpu().double() - kv.double()).abs() <= step * 0.57 + plain.BF16 * kv.double().abs() * 2).all()
    out = torch.full((2, NKV * hs), 123.0, dtype=BF, device="cuda")
    ws = torch.empty(ops.attention_paged_w4_workspace(NKV, NKV, hs, 1), dtype=torch.uint8, device="cuda")
    ops.attention_forward_paged_w4(out, qkv[:2].cuda(), codes, scales, i32([blocks]), i32([n]), i32([0, 1]), NKV, 1, ws)
    st = (NKV, qkv[:2], small_c, small_s, torch.tensor([[0, 1, 2]], dtype=I32), torch.tensor([n], dtype=I32),
          torch.tensor([0, 1], dtype=I32))
    _check_attention(st, out)


# ------------------------------------------------------------------ together ----
def test_serving_steps_of_a_batch(cuda, gpt2b):
    """Tables, append and attention of several steps, with a prompt in pieces, a request that waits for
    blocks and one that ends, against a plain cache of the same rows; the last step also captured."""
    from cuda_gpt2_inference_b200 import ops
    NKV, NH, hs, bs, nb, mb, B, cap = 2, 4, 64, 16, 14, 6, 3, 64
    g = torch.Generator().manual_seed(3)
    codes = torch.zeros(nb, 2, NKV, bs, hs // 2, dtype=torch.uint8, device="cuda")
    scales = torch.full((nb, 2, NKV, bs, 1, 2), math.nan, dtype=BF, device="cuda")
    table = torch.full((B, mb), -1, dtype=I32, device="cuda")
    free, count, have = i32(list(range(nb))), i32([nb]), i32([0] * B)
    slot, pos = torch.empty(cap, dtype=I64, device="cuda"), torch.empty(cap, dtype=I32, device="cuda")
    start, lens, blocks, left = i32([0] * (B + 1)), i32([0] * B), i32([0] * B), i32([0])
    ws = torch.empty(ops.attention_paged_w4_workspace(NH, NKV, hs, 32), dtype=torch.uint8, device="cuda")
    past = [torch.zeros(0, 2, NKV, hs, dtype=BF) for _ in range(B)]
    ctx = [0] * B
    for new in ([30, 5, 17], [25, 1, 1], [1, 1, 0], [40, 1, 29], [1, 5, 3]):
        qkv = torch.randn(cap, (NH + 2 * NKV) * hs, generator=g).to(BF)
        dq, dctx, dnew = qkv.cuda(), i32(ctx), i32(new)
        out = torch.full((cap, NH * hs), 123.0, dtype=BF, device="cuda")

        def step():
            ops.kv_block_tables(table, slot, pos, start, lens, blocks, left, dctx, dnew, have, free, count, bs)
            ops.kv_cache_write_w4(codes, scales, dq, slot, NH)
            ops.attention_forward_paged_w4(out, dq, codes, scales, table, lens, start, NH, 32, ws)

        step()
        eager = out.clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
            step()
        out.fill_(123.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert gpt2b.device_error() == 0
        got_lens = lens.tolist()
        r = 0
        pc, psc, ptab, plens = [], [], [], []
        for b in range(B):
            if got_lens[b]:
                assert got_lens[b] == ctx[b] + new[b]
                past[b] = torch.cat([past[b], qkv[r:r + new[b], NH * hs:].view(-1, 2, NKV, hs)])
                ctx[b] += new[b]
            r += new[b]
        # a plain contiguous cache: one block of 16 rows after another
        for b in range(B):
            n = got_lens[b]
            fill = torch.zeros(-(-n // bs) * bs - n, 2, NKV, hs, dtype=BF)
            c, s_ = plain.quantise(torch.cat([past[b][:n], fill]).view(-1, bs, 2, NKV, hs).permute(0, 2, 3, 1, 4))
            ptab.append(list(range(len(torch.cat(pc)) if pc else 0, (len(torch.cat(pc)) if pc else 0) + len(c))))
            pc.append(c)
            psc.append(s_)
        wide = max(map(len, ptab))
        pt = torch.tensor([t + [0] * (wide - len(t)) for t in ptab], dtype=I32)
        _check_attention((NH, qkv, torch.cat(pc), torch.cat(psc), pt, lens.cpu(), start.cpu()), out)
        have.copy_(blocks)
        count.copy_(left)
    # every block is held by one request, or free
    t, h, f = table.tolist(), have.tolist(), free.tolist()[:int(count)]
    assert sorted(sum((t[b][:h[b]] for b in range(B)), []) + f) == list(range(nb))


def test_operators_on_the_tensors_own_device(cuda):
    """Called with another device current (where there is one) they run where the tensors are."""
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    from cuda_gpt2_inference_b200 import ops
    st = _attention_state(2, 1, 64, 16, [40], [1], 2)
    with torch.cuda.device(1):
        ws = torch.empty(ops.attention_paged_w4_workspace(2, 2, 64, 1), dtype=torch.uint8, device="cuda:0")
        out = torch.full((st[1].shape[0], 128), 123.0, dtype=BF, device="cuda:0")
        d = [t.to("cuda:0") for t in st[1:]]
        ops.attention_forward_paged_w4(out, *d[:3], *d[3:], 2, 1, ws)
    _check_attention(st, out)


# ------------------------------------------------------------------- ordering ----
def test_calls_wait_for_whatever_came_before(cuda):
    """The kernels are launched before their predecessor has ended; copies, fills, kernels of other libraries and
    joins of streams in front of them are waited for all the same, eagerly and captured."""
    from cuda_gpt2_inference_b200 import ops
    NKV, NH, hs, bs, nb, n = 4, 8, 128, 16, 600, 4096
    g = torch.Generator().manual_seed(21)
    qkv = torch.randn(n, (NH + 2 * NKV) * hs, generator=g).to(BF).cuda()
    slots = torch.randperm(nb * bs, generator=g)[:n].cuda()
    src = torch.zeros_like(qkv)
    codes = torch.zeros(nb, 2, NKV, bs, hs // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(nb, 2, NKV, bs, hs // 64, 2, dtype=BF, device="cuda")
    out, copy = torch.zeros(n, 2, NKV, hs, dtype=BF, device="cuda"), torch.zeros(n, 2, NKV, hs, dtype=BF, device="cuda")
    big = torch.randn(4096, 4096, device="cuda")
    side = torch.cuda.Stream()

    def run():
        here = torch.cuda.current_stream()
        codes.zero_(), scales.zero_(), out.zero_()      # fills
        src.copy_(qkv)                                   # a copy right in front of the append
        ops.kv_cache_write_w4(codes, scales, src, slots, NH)
        src.zero_()                                      # and a fill of what it reads right behind it
        side.wait_stream(here)
        with torch.cuda.stream(side):
            torch.mm(big, big)                           # some time on another stream
            ops.kv_cache_read_w4(out, codes, scales, slots)
        here.wait_stream(side)
        ops.kv_cache_write_w4(codes, scales, src, slots, NH)   # overwrites behind the join
        copy.copy_(out)
        ops.kv_cache_read_w4(out, codes, scales, slots)

    kv = qkv[:, NH * hs:].view(n, 2, NKV, hs).cpu()
    c, s = plain.quantise(kv)
    want = plain.values(c, s)
    tol = plain.BF16 * want.abs() + s[..., 0].double().repeat_interleave(64, -1) * 1e-2  # (ties: see the append's test)

    def check():
        torch.cuda.synchronize()
        near = (copy.cpu().double() - want).abs() <= tol
        assert near.float().mean() > 0.999
        assert ((copy.cpu().double() - want).abs() <= tol + s[..., 0].double().repeat_interleave(64, -1)).all()
        assert not out.any()

    run()
    check()
    work = torch.cuda.Stream()
    work.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(work), torch.cuda.graph(graph, stream=work):
        run()
    for _ in range(3):
        copy.zero_()
        graph.replay()
        check()


def test_attention_hides_what_a_row_does_not_see(cuda):
    """A draft's own position may hold NaN (a group with an infinity): the rows before it do not see it."""
    for NKV, ratio, hs in ((2, 1, 64), (1, 8, 128), (2, 4, 64)):
        NH, qkv, codes, scales, table, lens, start = _attention_state(NKV, ratio, hs, 16, [70, 45], [5, 3], 31)
        for b, n in ((0, 70), (1, 45)):
            scales[int(table[b, (n - 1) // 16]), :, :, (n - 1) % 16] = math.nan
        out = _attend((NH, qkv, codes, scales, table, lens, start), 5).cpu()
        rows = [0, 1, 2, 3, 5, 6]
        assert out[[4, 7]].isnan().all()
        clean = scales.clone()
        for b, n in ((0, 70), (1, 45)):
            clean[int(table[b, (n - 1) // 16]), :, :, (n - 1) % 16] = 0
        want, err = plain.attention(qkv, codes, clean, table, lens, start, NH)
        off = (out[rows].double() - want[rows]).abs()
        assert (off <= plain.BF16 * want[rows].abs() + (1 + plain.BF16) * err[rows] + 2.0 ** -126).all()


def test_attention_of_two_calls_at_once(cuda):
    """Two streams with a workspace each, and the same call again and again on one."""
    from cuda_gpt2_inference_b200 import ops
    sts = [_attention_state(2, 2, 64, 16, [900, 33, 400], [2, 1, 3], 40 + k) for k in range(2)]
    want = [_attend(st, 3) for st in sts]
    ds = [[t.cuda() for t in st[1:]] for st in sts]
    ws = [torch.empty(ops.attention_paged_w4_workspace(4, 2, 64, 3), dtype=torch.uint8, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[torch.full_like(want[k], 123.0) for _ in range(20)] for k in range(2)]
    torch.cuda.synchronize()
    for i in range(20):
        for k in range(2):
            d = ds[k]
            ops.attention_forward_paged_w4(outs[k][i], d[0], d[1], d[2], d[3], d[4], d[5], 4, 3, ws[k], stream=streams[k])
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(o, want[k]) for o in outs[k])


def test_single_row_of_any_width_and_negative_scale(cuda):
    from cuda_gpt2_inference_b200 import ops
    st = _attention_state(2, 1, 64, 16, [50], [1], 51, pad=0)
    NH, qkv, codes, scales, table, lens, start = st
    _check_attention(st, _attend(st, 1, scale=-0.25), scale=-0.25)
    _check_attention(st, _attend(st, 1, scale=0.0), scale=0.0)
    odd = torch.cat([qkv, torch.zeros(1, 3, dtype=BF)], 1).cuda()  # one row has no pitch that could be odd
    ws = torch.empty(ops.attention_paged_w4_workspace(2, 2, 64, 1), dtype=torch.uint8, device="cuda")
    out = torch.zeros(1, 128, dtype=BF, device="cuda")
    ops.attention_forward_paged_w4(out, odd, codes.cuda(), scales.cuda(), table.cuda(), lens.cuda(), start.cuda(), 2, 1, ws)
    assert torch.equal(out, _attend(st, 1))


def test_drafted_decoding_of_a_batch(cuda, gpt2b):
    """Six steps of drafted decoding as one would write them: lengths, tables and cache are carried on the device,
    refused drafts are overwritten, a request without drafts stands beside others.  A stand-in for the model (token
    and position embeddings to q, k, v; attention to logits) keeps the rows' contents honest."""
    from cuda_gpt2_inference_b200 import ops
    NKV, NH, hs, bs, nb, mb, B, V, width = 2, 4, 64, 16, 40, 12, 3, 300, 5
    cap, T = B * width, 0.8
    g = torch.Generator().manual_seed(77)
    emb = torch.randn(V + 400, (NH + 2 * NKV) * hs, generator=g).to(BF).cuda()
    head = (torch.randn(NH * hs, V, generator=g) * 0.3).to(BF).cuda()
    codes = torch.zeros(nb, 2, NKV, bs, hs // 2, dtype=torch.uint8, device="cuda")
    scales = torch.full((nb, 2, NKV, bs, 1, 2), math.nan, dtype=BF, device="cuda")
    table = torch.full((B, mb), -1, dtype=I32, device="cuda")
    free, count, have, ctx = i32(list(range(nb))), i32([nb]), i32([0] * B), i32([0] * B)
    slot, pos = torch.empty(cap, dtype=I64, device="cuda"), torch.empty(cap, dtype=I32, device="cuda")
    start, lens, blocks, left = i32([0] * (B + 1)), i32([0] * B), i32([0] * B), i32([0])
    atty = torch.zeros(cap, NH * hs, dtype=BF, device="cuda")
    probs = torch.zeros(cap, V, device="cuda")
    out, taken = torch.zeros(B, width, dtype=I32, device="cuda"), torch.zeros(B, dtype=I32, device="cuda")
    ws = torch.empty(ops.attention_paged_w4_workspace(NH, NKV, hs, width), dtype=torch.uint8, device="cuda")
    seqs = [[5], [7], [9]]                      # what each request has said so far, the last token not yet cached
    drafts_of = [4, 0, 2]
    told = 0
    for step in range(6):
        dp = torch.softmax(torch.randn(cap, V, generator=g), -1)
        rows, tokens = [], []
        for b in range(B):
            guess = torch.multinomial(dp[len(tokens):len(tokens) + max(1, drafts_of[b])], 1, generator=g)[:, 0].tolist()
            row = [seqs[b][-1]] + guess[:drafts_of[b]]
            rows.append(len(row))
            tokens += row
        tokens += [0] * (cap - len(tokens))
        dtok, ua, us = i32(tokens), torch.rand(cap, generator=g) * 0.2, torch.rand(B, generator=g)
        ops.kv_block_tables(table, slot, pos, start, lens, blocks, left, ctx, i32(rows), have, free, count, bs)
        qkv = emb[dtok.long()] + emb[V + pos.long()]
        ops.kv_cache_write_w4(codes, scales, qkv, slot, NH)
        ops.attention_forward_paged_w4(atty, qkv, codes, scales, table, lens, start, NH, width, ws)
        logits = (atty @ head).float()
        ops.softmax_probs(probs, logits, T)
        ops.verify_draft_tokens(out, taken, dtok, probs, dp.cuda(), start, ua.cuda(), us.cuda())
        # what it should have been: the request's whole text, quantised position by position
        st = start.tolist()
        n_ctx = [len(s) - 1 for s in seqs]
        assert lens.tolist() == [c + r for c, r in zip(n_ctx, rows)]
        flat_c, flat_s, tabs = [], [], []
        for b in range(B):
            text = seqs[b][:-1] + tokens[st[b]:st[b + 1]]
            x = emb[torch.tensor(text).cuda()] + emb[V + torch.arange(len(text)).cuda()]
            kv = x[:, NH * hs:].cpu().view(-1, 2, NKV, hs)
            kv = torch.cat([kv, torch.zeros(-len(text) % bs, 2, NKV, hs, dtype=BF)])
            c, s = plain.quantise(kv.view(-1, bs, 2, NKV, hs).permute(0, 2, 3, 1, 4))
            tabs.append(list(range(sum(map(len, flat_c)), sum(map(len, flat_c)) + len(c))))
            flat_c.append(c)
            flat_s.append(s)
        wide = max(map(len, tabs))
        pt = torch.tensor([t + [0] * (wide - len(t)) for t in tabs], dtype=I32)
        want, err = plain.attention(qkv.cpu(), torch.cat(flat_c), torch.cat(flat_s), pt, lens.cpu(), start.cpu(), NH)
        R = st[-1]
        assert ((atty[:R].cpu().double() - want[:R]).abs() <= plain.BF16 * want[:R].abs() + 1.01 * err[:R] + 2.0 ** -126).all()
        ref = torch.softmax(logits[:R].cpu().double() / T, -1)
        assert ((probs[:R].cpu().double() - ref).abs() <= 2.0 ** -17 * ref + 2.0 ** -126).all()
        assert (out.tolist(), taken.tolist()) == plain.verify(torch.tensor(tokens), probs.cpu(), dp, st, ua, us, width)
        for b in range(B):
            got = [t for t in out[b].tolist() if t >= 0]
            assert len(got) == int(taken[b]) + 1
            seqs[b] += got
            told += int(taken[b])
        ctx.add_(taken).add_(1)
        have.copy_(blocks)
        count.copy_(left)
    assert told > 0 and gpt2b.device_error() == 0


def test_attention_of_many_and_of_no_requests(cuda, gpt2b):
    """As many requests as a call takes, most of them with nothing cached or nothing asked; and none with rows."""
    lens, rows = [k % 4 for k in range(4096)], [k % 3 for k in range(4096)]
    st = _attention_state(1, 2, 64, 16, lens, rows, 61)
    _check_attention(st, _attend(st, 2))
    st = _attention_state(2, 1, 128, 16, [20, 0, 7], [0, 0, 0], 62)
    out = _attend(st, 1)
    assert (out == 123.0).all()
    assert gpt2b.device_error() == 0


def test_attention_of_one_long_request_over_one_head(cuda):
    """The whole GPU on one segment: more pieces to join than one pass of the join takes."""
    st = _attention_state(1, 2, 128, 64, [70001], [1], 63)
    _check_attention(st, _attend(st, 1))
    st = _attention_state(1, 1, 64, 16, [30011], [17], 64)
    _check_attention(st, _attend(st, 17))
