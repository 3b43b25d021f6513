"""Refusals of the paged 4-bit cache and draft verification entry points (no GPU): they come before any launch."""
from __future__ import annotations

import ctypes

import pytest
import torch

import paged_w4_plain as plain

I32, I64, BF = torch.int32, torch.int64, torch.bfloat16


@pytest.fixture(scope="module")
def mem():
    buf = ctypes.create_string_buffer(4096 + 16)
    mem.keep = buf
    return (ctypes.addressof(buf) + 15) & ~15


def test_tables_refusals(gpt2b, mem):
    f, a = gpt2b.lib().gpt2b_kv_block_tables, mem
    p = [a + (i << 36) for i in range(12)]  # far apart, never read: these calls are refused
    ok = dict(B=2, mb=4, bs=16, rows=8, cap=4)

    def rc(ptrs=p, **kw):
        v = {**ok, **kw}
        return f(*ptrs, v["B"], v["mb"], v["bs"], v["rows"], v["cap"], None)

    for bad in (dict(B=0), dict(B=-1), dict(mb=0), dict(bs=0), dict(rows=-1), dict(cap=-1)):
        assert rc(**bad) == gpt2b.ERR_INVALID_ARG, bad
    for i in range(12):
        assert rc([None if k == i else x for k, x in enumerate(p)]) == gpt2b.ERR_INVALID_ARG, i
    # results over inputs that every CTA reads, as a whole or by a byte
    for dst in range(7):
        for src in range(7, 12):
            assert rc([p[src] if k == dst else x for k, x in enumerate(p)]) == gpt2b.ERR_INVALID_ARG
            assert rc([p[dst] + 3 if k == src else x for k, x in enumerate(p)]) == gpt2b.ERR_INVALID_ARG
    assert rc(B=4097) == gpt2b.ERR_UNSUPPORTED
    assert rc(mb=2 ** 28, bs=16) == gpt2b.ERR_UNSUPPORTED


def test_cache_refusals(gpt2b, mem):
    lib, a = gpt2b.lib(), mem

    def write(codes=a, scales=a, qkv=a, slots=a, rows=1, NH=2, NKV=2, hs=64, ld=384, nb=2, bs=16):
        return lib.gpt2b_kv_cache_write_w4(codes, scales, qkv, slots, rows, NH, NKV, hs, ld, nb, bs, None)

    def read(out=a, codes=a, scales=a, slots=a, rows=1, NKV=2, hs=64, nb=2, bs=16):
        return lib.gpt2b_kv_cache_read_w4(out, codes, scales, slots, rows, NKV, hs, nb, bs, None)

    for fn in (write, read):
        for bad in (dict(codes=None), dict(scales=None), dict(slots=None), dict(rows=-1), dict(NKV=0), dict(nb=0), dict(bs=0)):
            assert fn(**bad) == gpt2b.ERR_INVALID_ARG, bad
        for bad in (dict(hs=32), dict(hs=96), dict(hs=256), dict(bs=8), dict(bs=24)):
            assert fn(**bad) == gpt2b.ERR_UNSUPPORTED, bad
        for bad in (dict(codes=a + 4), dict(scales=a + 8)):
            assert fn(**bad) == gpt2b.ERR_ALIGNMENT, bad
        assert fn(rows=0) == gpt2b.OK  # an empty step
    assert write(qkv=None) == gpt2b.ERR_INVALID_ARG and read(out=None) == gpt2b.ERR_INVALID_ARG
    assert write(ld=383) == gpt2b.ERR_INVALID_ARG and write(NH=0) == gpt2b.ERR_INVALID_ARG
    assert write(NH=2 ** 30, NKV=2 ** 24) == gpt2b.ERR_INVALID_ARG  # no overflow in the width
    assert write(ld=385) == gpt2b.ERR_ALIGNMENT and write(qkv=a + 2) == gpt2b.ERR_ALIGNMENT
    assert read(out=a + 8) == gpt2b.ERR_ALIGNMENT


def test_attention_refusals(gpt2b, mem):
    lib, a = gpt2b.lib(), mem
    n = ctypes.c_size_t()
    size = lib.gpt2b_attention_paged_w4_workspace
    assert size(12, 12, 64, 1, ctypes.byref(n)) == gpt2b.OK and n.value > 0
    assert size(12, 12, 64, 1, None) == gpt2b.ERR_INVALID_ARG
    for NH, NKV, hs, q in ((0, 1, 64, 1), (4, 0, 64, 1), (5, 2, 64, 1), (4, 2, 64, 0), (-4, 2, 64, 1)):
        assert size(NH, NKV, hs, q, ctypes.byref(n)) == gpt2b.ERR_INVALID_ARG
    assert size(4, 2, 80, 1, ctypes.byref(n)) == gpt2b.ERR_UNSUPPORTED

    far = 1 << 44

    def rc(out=a + far, qkv=a, codes=a, scales=a, table=a, lens=a, start=a, B=1, rows=1, NH=2, NKV=2, hs=64, ld=384, nb=2, bs=16,
           mb=2, q=1, ws=a + 2 * far, bytes=1 << 40, scale=0.125):
        return lib.gpt2b_attention_forward_paged_w4(out, qkv, codes, scales, table, lens, start, B, rows, NH, NKV, hs, ld, nb,
                                                    bs, mb, q, scale, ws, bytes, None)

    for bad in (dict(out=None), dict(qkv=None), dict(codes=None), dict(scales=None), dict(table=None), dict(lens=None),
                dict(start=None), dict(ws=None), dict(B=0), dict(rows=-1), dict(NH=3), dict(NKV=0), dict(nb=0), dict(bs=0),
                dict(mb=0), dict(q=0), dict(bytes=0), dict(ld=383), dict(out=a), dict(out=a + 16, rows=3), dict(ws=a + far),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=-2e30)):
        assert rc(**bad) == gpt2b.ERR_INVALID_ARG, bad
    for bad in (dict(hs=32), dict(bs=8), dict(B=4097), dict(mb=2 ** 28)):
        assert rc(**{"ld": 4096, **bad}) == gpt2b.ERR_UNSUPPORTED, bad
    for bad in (dict(out=a + far + 8), dict(qkv=a + 2), dict(codes=a + 1), dict(scales=a + 4), dict(ws=a + 2 * far + 4), dict(ld=388)):
        assert rc(**bad) == gpt2b.ERR_ALIGNMENT, bad
    assert rc(rows=0) == gpt2b.OK


def test_probs_and_verify_refusals(gpt2b, mem):
    lib, a = gpt2b.lib(), mem
    inf, nan = float("inf"), float("nan")

    def probs(out=a, x=a, rows=1, V=8, li=8, lo=8, T=1.0):
        return lib.gpt2b_softmax_probs(out, x, rows, V, li, lo, T, None)

    for bad in (dict(out=None), dict(x=None), dict(rows=-1), dict(V=0), dict(li=7), dict(lo=7), dict(T=-1.0), dict(T=nan), dict(T=1e-31), dict(T=1e31),
                dict(T=inf), dict(li=9), dict(out=a + 4), dict(out=a + 32, rows=2), dict(out=a + 36, rows=2, li=16, lo=16)):
        assert probs(**bad) == gpt2b.ERR_INVALID_ARG, bad
    assert probs(rows=0) == gpt2b.OK

    def verify(out=a, n=a + (1 << 40), tok=a + (2 << 40), p=a, q=a, start=a + (3 << 40), ua=a, us=a, B=1, rows=2, V=8, lp=8, lq=8, width=3):
        return lib.gpt2b_verify_draft_tokens(out, n, tok, p, q, start, ua, us, B, rows, V, lp, lq, width, None)

    for bad in (dict(out=None), dict(n=None), dict(tok=None), dict(p=None), dict(start=None), dict(ua=None), dict(us=None),
                dict(B=0), dict(rows=-1), dict(V=0), dict(lp=7), dict(lq=7), dict(width=0), dict(out=a + (2 << 40)),
                dict(n=a + (2 << 40) + 4), dict(out=a + (3 << 40)), dict(n=a + (3 << 40)), dict(tok=a + 8)):
        assert verify(**bad) == gpt2b.ERR_INVALID_ARG, bad


def _refused(gpt2b, fn, *args, status=None, **kw):
    with pytest.raises(gpt2b.Gpt2bError) as e:
        fn(*args, **kw)
    assert e.value.status == (status or gpt2b.ERR_INVALID_ARG)
    return str(e.value)


def test_python_refusals(gpt2b):
    from cuda_gpt2_inference_b200 import ops
    nb, NKV, NH, bs, hs, R, B = 3, 2, 4, 16, 64, 5, 2
    codes = torch.zeros(nb, 2, NKV, bs, hs // 2, dtype=torch.uint8)
    scales = torch.zeros(nb, 2, NKV, bs, 1, 2, dtype=BF)
    qkv, slots = torch.zeros(R, (NH + 2 * NKV) * hs, dtype=BF), torch.zeros(R, dtype=I64)
    w = [codes, scales, qkv, slots, NH]

    def swap(args, i, v):
        return [v if k == i else x for k, x in enumerate(args)]

    # CPU tensors, right in all else, are refused as such
    assert "CUDA" in _refused(gpt2b, ops.kv_cache_write_w4, *w)
    for i, v in ((0, codes[0]), (0, codes.int()), (0, codes.transpose(2, 3)), (1, scales.half()), (1, scales[:, :, :1]),
                 (2, qkv.float()), (2, qkv[:, :-1]), (2, qkv.t()), (3, slots.int()), (3, slots[:-1]), (4, 5)):
        assert "CUDA" not in _refused(gpt2b, ops.kv_cache_write_w4, *swap(w, i, v)), i
    small = [codes[:, :, :, :8].contiguous(), scales[:, :, :, :8].contiguous(), qkv, slots, NH]
    _refused(gpt2b, ops.kv_cache_write_w4, *small, status=gpt2b.ERR_UNSUPPORTED)
    r = [torch.zeros(R, 2, NKV, hs, dtype=BF), codes, scales, slots]
    assert "CUDA" in _refused(gpt2b, ops.kv_cache_read_w4, *r)
    for i, v in ((0, r[0][:, :1].contiguous()), (0, r[0].float()), (3, slots[1:])):
        assert "CUDA" not in _refused(gpt2b, ops.kv_cache_read_w4, *swap(r, i, v))
    i = lambda n: torch.zeros(n, dtype=I32)  # noqa: E731
    a = [torch.zeros(R, NH * hs, dtype=BF), qkv, codes, scales, torch.zeros(B, 4, dtype=I32), i(B), i(B + 1), NH, 1,
         torch.zeros(64, dtype=torch.uint8)]
    assert "CUDA" in _refused(gpt2b, ops.attention_forward_paged_w4, *a)
    for k, v in ((0, a[0][:-1]), (0, a[0][:, :-64].contiguous()), (4, i(4)), (4, a[4].long()), (5, i(B + 1)), (6, i(B)),
                 (9, torch.zeros(64))):
        assert "CUDA" not in _refused(gpt2b, ops.attention_forward_paged_w4, *swap(a, k, v)), k
    t = [torch.zeros(B, 4, dtype=I32), torch.zeros(R, dtype=I64), i(R), i(B + 1), i(B), i(B), i(1), i(B), i(B), i(B), i(7), i(1), bs]
    assert "CUDA" in _refused(gpt2b, ops.kv_block_tables, *t)
    for k in range(12):
        if k != 10:
            wrong = torch.zeros(B + 9, dtype=t[k].dtype) if t[k].dim() == 1 and k != 1 else t[k].float()
            assert "CUDA" not in _refused(gpt2b, ops.kv_block_tables, *swap(t, k, wrong)), k
    x = torch.zeros(R, 9)
    assert "CUDA" in _refused(gpt2b, ops.softmax_probs, x, x.clone())
    for args in ((x, x.double()), (x[:-1], x), (x[:, :-1], x), (x.t(), x)):
        assert "CUDA" not in _refused(gpt2b, ops.softmax_probs, *args)
    v = [torch.zeros(B, 3, dtype=I32), i(B), i(R), x, x, i(B + 1), torch.zeros(R), torch.zeros(B)]
    assert "CUDA" in _refused(gpt2b, ops.verify_draft_tokens, *v)
    for k, bad in ((0, i(3)), (1, i(B + 1)), (2, i(R - 1)), (2, torch.zeros(R)), (3, x[:-1]), (4, x[:, :-1]), (4, x.half()),
                   (5, i(B)), (6, torch.zeros(R + 1)), (7, torch.zeros(B + 1))):
        assert "CUDA" not in _refused(gpt2b, ops.verify_draft_tokens, *swap(v, k, bad)), k


def test_plain_forms_hold_together():
    """The plain forms the GPU tests compare with: values near what was quantised, and a known small case."""
    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(0)).to(BF)
    c, s = plain.quantise(x)
    step = s[..., 0].double().repeat_interleave(64, -1)
    assert ((plain.values(c, s) - x.double()).abs() <= step * (0.5 + 15 * plain.BF16)).all()
    assert plain.tables([[4, -1], [-1, -1]], [16, 0], [1, 2], [1, 0], [7, 8, 9], 3, 16, 4) == \
        ([[4, 9], [8, -1]], [9 * 16, 8 * 16, 8 * 16 + 1, -1], [16, 0, 1, 0], [0, 1, 3], [17, 2], [2, 1], 1)
    p = torch.tensor([[0.2, 0.3, 0.5], [0.1, 0.9, 0.0]])
    q = torch.tensor([[0.1, 0.8, 0.1], [0, 0, 0]])
    u = torch.tensor([0.9])
    assert plain.verify(torch.tensor([0, 1]), p, q, [0, 2], torch.tensor([0.1, 0.0]), u, 3) == ([[1, 1, -1]], [1])
    assert plain.verify(torch.tensor([0, 1]), p, q, [0, 2], torch.tensor([0.9, 0.0]), u, 3) == ([[2, -1, -1]], [0])
