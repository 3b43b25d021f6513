"""A serving program's steps as the integration notes describe them: prompts in pieces, requests without rows in a step,
requests that wait for blocks, one that ends and gives its blocks back."""
from __future__ import annotations

import math

import pytest
import torch

import paged_w4_plain as plain

pytestmark = pytest.mark.gpu
I32, I64, BF = torch.int32, torch.int64, torch.bfloat16
NKV, NH, hs, bs, V, T = 2, 4, 64, 16, 300, 0.8


def i32(v):
    return torch.tensor(v, dtype=I32, device="cuda")


def _plain_cache(texts, emb):
    """One contiguous cache of each text's tokens: (codes, scales, table, lens)."""
    codes, scales, table = [], [], []
    for text in texts:
        x = emb[torch.tensor(text, dtype=I64, device="cuda")] + emb[V + torch.arange(len(text), device="cuda")]
        kv = torch.cat([x[:, NH * hs:].cpu().view(-1, 2, NKV, hs), torch.zeros(-len(text) % bs, 2, NKV, hs, dtype=BF)])
        c, s = plain.quantise(kv.view(-1, bs, 2, NKV, hs).permute(0, 2, 3, 1, 4))
        table.append(list(range(sum(map(len, codes)), sum(map(len, codes)) + len(c))))
        codes.append(c)
        scales.append(s)
    wide = max(map(len, table))
    return torch.cat(codes), torch.cat(scales), torch.tensor([t + [0] * (wide - len(t)) for t in table], dtype=I32)


def test_next_lengths_of_mixed_requests(cuda, gpt2b):
    """The next step's context is seq_lens behind a piece of a prompt, ctx + 1 + n_accepted behind a decoding request's
    rows, and what it was where a request was not served or had no rows.  Positions never written hold NaN, so a length
    that ran ahead would show in the attention."""
    from cuda_gpt2_inference_b200 import ops
    B, nb, mb, cap, width = 4, 9, 12, 64, 4
    g = torch.Generator().manual_seed(78)
    emb = torch.randn(V + 400, (NH + 2 * NKV) * hs, generator=g).to(BF).cuda()
    head = (torch.randn(NH * hs, V, generator=g) * 0.3).to(BF).cuda()
    codes = torch.zeros(nb, 2, NKV, bs, hs // 2, dtype=torch.uint8, device="cuda")
    scales = torch.full((nb, 2, NKV, bs, 1, 2), math.nan, dtype=BF, device="cuda")
    table = torch.full((B, mb), -1, dtype=I32, device="cuda")
    free, count, have, ctx = i32(list(range(nb))), i32([nb]), i32([0] * B), i32([0] * B)
    slot, pos = torch.empty(cap, dtype=I64, device="cuda"), torch.empty(cap, dtype=I32, device="cuda")
    start, lens, blocks, left = i32([0] * (B + 1)), i32([0] * B), i32([0] * B), i32([0])
    atty, probs = torch.zeros(cap, NH * hs, dtype=BF, device="cuda"), torch.zeros(cap, V, device="cuda")
    out, taken = torch.zeros(B, width, dtype=I32, device="cuda"), torch.zeros(B, dtype=I32, device="cuda")
    ws = torch.empty(ops.attention_paged_w4_workspace(NH, NKV, hs, 25), dtype=torch.uint8, device="cuda")

    # a request's tokens; of a prompt all but the last go in as pieces, the last is its first decoding row
    said = [torch.randint(0, V, (n,), generator=g).tolist() for n in (50, 71, 1, 20)]
    cached = [0] * B
    begins = [0, 1, 3, 0]  # step in which a request arrives
    ended = set()
    waited = told = idle = 0
    for step in range(14):
        dp = torch.softmax(torch.randn(cap, V, generator=g), -1)
        rows, tokens, prompt = [], [], []
        for b in range(B):
            todo = len(said[b]) - 1 - cached[b]
            if step < begins[b] or b in ended or (b == 2 and step % 3 == 1):
                row = []
            elif todo > 0:
                row = said[b][cached[b]:cached[b] + min(25, todo)]
            else:
                row = said[b][-1:] + torch.multinomial(dp[len(tokens):len(tokens) + 3], 1, generator=g)[:b, 0].tolist()
            prompt.append(bool(row) and todo > 0)
            rows.append(len(row))
            tokens += row
        tokens += [0] * (cap - len(tokens))
        dtok, new, ua, us = i32(tokens), i32(rows), torch.rand(cap, generator=g) * 0.2, torch.rand(B, generator=g)
        ops.kv_block_tables(table, slot, pos, start, lens, blocks, left, ctx, new, have, free, count, bs)
        qkv = emb[dtok.long()] + emb[V + pos.long()]
        ops.kv_cache_write_w4(codes, scales, qkv, slot, NH)
        ops.attention_forward_paged_w4(atty, qkv, codes, scales, table, lens, start, NH, 25, ws)
        ops.softmax_probs(probs, (atty @ head).float(), T)
        ops.verify_draft_tokens(out, taken, dtok, probs, dp.cuda(), start, ua.cuda(), us.cuda())

        st, served = start.tolist(), lens.tolist()
        texts = [(said[b][:cached[b]] + tokens[st[b]:st[b + 1]]) if served[b] else [] for b in range(B)]
        assert served == [len(t) for t in texts]
        want, err = plain.attention(qkv.cpu(), *_plain_cache(texts, emb), lens.cpu(), start.cpu(), NH)
        R = st[-1]
        assert ((atty[:R].cpu().double() - want[:R]).abs() <= plain.BF16 * want[:R].abs() + 1.01 * err[:R] + 2.0 ** -126).all()
        drawn = plain.verify(torch.tensor(tokens), probs.cpu(), dp, st, ua, us, width)
        assert (out.tolist(), taken.tolist()) == drawn

        # the next step's state, on the device
        ctx.copy_(torch.where((lens == 0) | (new == 0), ctx, torch.where(torch.tensor(prompt, device="cuda"), lens, ctx + 1 + taken)))
        have.copy_(blocks)
        count.copy_(left)

        # and as the program keeps it: tokens count only of decoding requests that were served and had rows
        for b in range(B):
            waited += rows[b] > 0 and not served[b]
            idle += rows[b] == 0 and served[b] > 0
            if not served[b] or not rows[b]:
                continue
            if prompt[b]:
                cached[b] += rows[b]
            else:
                got = [t for t in out[b].tolist() if t >= 0]
                assert len(got) == int(taken[b]) + 1
                said[b] += got
                cached[b] += len(got)
                told += len(got)
        assert ctx.tolist() == cached
        if step == 8:  # the first request ends: its blocks go back to the list
            n, k = int(count), int(have[0])
            free[n:n + k] = table[0, :k]
            count += k
            have[0] = ctx[0] = 0
            cached[0] = 0
            ended.add(0)
    assert waited > 2 and idle > 0 and told > 10 and gpt2b.device_error() == 0
    held = [table[b, :int(have[b])].tolist() for b in range(B)]
    assert sorted(sum(held, []) + free[:int(count)].tolist()) == list(range(nb))


def test_calls_of_two_threads_at_once(cuda):
    """The binding lets go of the interpreter lock: two threads, a stream each, the same operators at once."""
    import threading

    from cuda_gpt2_inference_b200 import ops
    from test_paged_w4_gpu import _attend, _attention_state
    sts = [_attention_state(2, r, hs_, 16, [700, 33], [2, 1], 90 + r) for r, hs_ in ((1, 64), (8, 128))]
    want = [_attend(st, 2) for st in sts]
    x = torch.randn(5, 5000, device="cuda")
    probs = torch.empty_like(x)
    ops.softmax_probs(probs, x, 0.7)
    ds = [[t.cuda() for t in st[1:]] for st in sts]
    ws = [torch.empty(ops.attention_paged_w4_workspace(st[0], 2, st[2].shape[4] * 2, 2), dtype=torch.uint8, device="cuda") for st in sts]
    outs = [[torch.full_like(want[k], 123.0) for _ in range(50)] for k in range(2)]
    ps = [[torch.empty_like(x) for _ in range(50)] for _ in range(2)]
    torch.cuda.synchronize()
    failed = []

    def work(k):
        try:
            s = torch.cuda.Stream()
            for i in range(50):
                ops.attention_forward_paged_w4(outs[k][i], *ds[k][:3], ds[k][3], ds[k][4], ds[k][5], sts[k][0], 2, ws[k], stream=s)
                ops.softmax_probs(ps[k][i], x, 0.7, stream=s)
            s.synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed
    for k in range(2):
        assert all(torch.equal(o, want[k]) for o in outs[k]) and all(torch.equal(p, probs) for p in ps[k])
