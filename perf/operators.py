"""The operators of a serving step over a paged 4-bit KV cache with drafted tokens, as measured cases.

Operators (``case["op"]``):

* ``tables``    -- block tables, slot map and row offsets of a step from the requests' lengths;
* ``cache``     -- new rows appended to the 4-bit cache, and the same rows read back as values;
* ``attention`` -- attention of 1..n query rows per sequence over the paged 4-bit cache;
* ``probs``     -- logits to probabilities;
* ``verify``    -- drafted tokens accepted or refused, and the next token drawn.

With ``own`` false, ``run`` computes each in elementary torch operations; with ``own`` true it calls
``cuda_gpt2_inference_b200.ops``.
"""
import math

import torch

own = False

GROUP = 64  # channels that share a step and a low end


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # eight requests decoding one token each: the table update in front of every step
        {"name": "tables_decode", "op": "tables", "B": 8, "bs": 16, "max_blocks": 64, "new_lo": 1, "new_hi": 1},
        # a large mixed batch: prompts in pieces beside decoding requests, some without blocks left
        {"name": "tables_mixed", "op": "tables", "B": 256, "bs": 16, "max_blocks": 512, "new_lo": 0, "new_hi": 511},
        # one request's token and four drafts appended (12 heads of 64, as GPT-2 124M)
        {"name": "cache_draft_step", "op": "cache", "rows": 5, "NH": 12, "NKV": 12, "hs": 64, "bs": 16},
        # a batch of prompts appended at once (32 query heads over 8 shared heads of 128)
        {"name": "cache_prompts", "op": "cache", "rows": 16384, "NH": 32, "NKV": 8, "hs": 128, "bs": 16},
        # one request, one token, 124M's heads at the end of its context: latency
        {"name": "attention_one", "op": "attention", "B": 1, "NH": 12, "NKV": 12, "hs": 64, "bs": 16, "lo": 1001, "hi": 1001,
         "q": 1},
        # a batch of GPT-2-XL requests of uneven lengths, each with up to four drafts
        {"name": "attention_drafts", "op": "attention", "B": 16, "NH": 25, "NKV": 25, "hs": 64, "bs": 16, "lo": 37,
         "hi": 1024, "q": 5},
        # few long requests with shared heads, one token each
        {"name": "attention_long", "op": "attention", "B": 4, "NH": 32, "NKV": 8, "hs": 128, "bs": 32, "lo": 9001,
         "hi": 32000, "q": 1},
        # the largest: a batch of long requests with shared heads and drafts
        {"name": "attention_batch_long", "op": "attention", "B": 32, "NH": 32, "NKV": 8, "hs": 128, "bs": 64, "lo": 4001,
         "hi": 16384, "q": 4},
        # one request's logits with four drafts, GPT-2's vocabulary
        {"name": "probs_draft_step", "op": "probs", "rows": 5, "V": 50257, "T": 1.0},
        # a batch's logits with drafts
        {"name": "probs_batch", "op": "probs", "rows": 320, "V": 50257, "T": 0.7},
        # one request with four drafts
        {"name": "verify_one", "op": "verify", "B": 1, "drafts": 4, "V": 50257, "q_given": True},
        # a batch with up to seven drafts each
        {"name": "verify_batch", "op": "verify", "B": 64, "drafts": 7, "V": 50257, "q_given": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tables", "cache", "attention", "attention", "probs", "verify"])
    if op == "tables":
        bs = rng.choice([16, 32, 64])
        hi = _log(rng, 1, 511)
        return {"op": op, "B": _log(rng, 1, 256), "bs": bs, "max_blocks": _log(rng, 8, 8192 // bs), "new_lo": rng.choice([0, 1]),
                "new_hi": hi}
    if op == "cache":
        hs, NKV = rng.choice([64, 128]), rng.choice([1, 2, 8, 12, 25])
        return {"op": op, "rows": _log(rng, 1, 16384 * 8 * 128 // (NKV * hs * 2)), "NH": NKV * rng.choice([1, 4]), "NKV": NKV,
                "hs": hs, "bs": rng.choice([16, 32, 64])}
    if op == "attention":
        hs, NKV, ratio = rng.choice([64, 128]), rng.choice([1, 2, 5, 8, 12, 25]), rng.choice([1, 1, 3, 4, 8])
        hi, B = _log(rng, 1, 32000), _log(rng, 1, 64)
        most = 32 * 16384 * 8 * 128
        while B * hi * NKV * hs * max(1, ratio // 4) > most // 2:
            B, hi = (B + 1) // 2, max(1, hi * 3 // 4)
        return {"op": op, "B": B, "NH": NKV * ratio, "NKV": NKV, "hs": hs, "bs": rng.choice([16, 32, 64]),
                "lo": max(1, int(hi * rng.uniform(0.05, 1.0))), "hi": hi, "q": rng.randint(1, 8)}
    if op == "probs":
        V = rng.choice([50257, 50304, _log(rng, 100, 131072)])
        return {"op": op, "rows": _log(rng, 1, max(1, 320 * 50257 // V)), "V": V, "T": rng.choice([1.0, 0.7, 1.3])}
    V = rng.choice([50257, 50304, _log(rng, 100, 131072)])
    drafts = rng.randint(1, 8)
    return {"op": "verify", "B": _log(rng, 1, max(1, 512 * 50257 // (V * (drafts + 1)))), "drafts": drafts, "V": V,
            "q_given": rng.choice([True, True, False])}


def _spread(n, lo, hi, step=0.6180339887498949, start=0.37):
    """n whole numbers of [lo, hi], evenly spread but in no order; the same for every seed."""
    return [lo + int(((start + step * i) % 1.0) * (hi - lo + 1)) for i in range(n)]


def _attention_shape(case):
    """Lengths and query rows per sequence; the first sequence has the longest length and the most rows."""
    lens = _spread(case["B"], case["lo"], case["hi"])
    lens[0] = case["hi"]
    rows = _spread(case["B"], 1, case["q"], step=0.7548776662466927)
    rows[0] = case["q"]
    return lens, rows


def _draft_rows(case):
    rows = [1 + n for n in _spread(case["B"], 0, case["drafts"], step=0.7548776662466927)]
    rows[0] = 1 + case["drafts"]
    return rows


def _table_lengths(case):
    new = _spread(case["B"], case["new_lo"], case["new_hi"], step=0.7548776662466927)
    ctx = _spread(case["B"], 0, case["max_blocks"] * case["bs"] - 1)
    return ctx, new


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _starts(counts, dev):
    return torch.tensor([0] + list(counts), dtype=torch.int64, device=dev).cumsum(0).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    h = torch.Generator().manual_seed(int(seed))
    dev, i32 = "cuda", torch.int32
    s = {"case": case}
    if case["op"] == "tables":
        B, bs, mb = case["B"], case["bs"], case["max_blocks"]
        ctx, new = _table_lengths(case)
        # the blocks each request holds: those of its context, and for some one more (left by refused drafts)
        have = [min(mb, -(-c // bs) + int(x)) for c, x in zip(ctx, torch.randint(0, 2, (B,), generator=h).tolist())]
        need = sum(max(0, -(-(c + n) // bs) - k) for c, n, k in zip(ctx, new, have))
        total = sum(have) + need
        order = torch.randperm(total, generator=h).to(i32)
        table = torch.full((B, mb), -1, dtype=i32)
        at = 0
        for b, k in enumerate(have):
            table[b, :k] = order[at:at + k]
            at += k
        free = order[at:]
        left = len(free) - int(torch.randint(0, 1 + len(free) // 8, (1,), generator=h))  # not always enough
        s.update(table=table.to(dev), ctx=torch.tensor(ctx, dtype=i32, device=dev), new=torch.tensor(new, dtype=i32, device=dev),
                 have=torch.tensor(have, dtype=i32, device=dev), free=torch.cat([free, free.new_zeros(1)]).to(dev),
                 free_count=torch.tensor([left], dtype=i32, device=dev))
        rows = sum(new) + 3  # a few padding rows behind the last request
        s.update(slot=torch.empty(rows, dtype=torch.int64, device=dev), pos=torch.empty(rows, dtype=i32, device=dev),
                 start=torch.empty(B + 1, dtype=i32, device=dev), lens=torch.empty(B, dtype=i32, device=dev),
                 have_out=torch.empty(B, dtype=i32, device=dev), left=torch.empty(1, dtype=i32, device=dev))
    elif case["op"] == "cache":
        rows, NH, NKV, hs, bs = (case[k] for k in ("rows", "NH", "NKV", "hs", "bs"))
        blocks = -(-rows // bs) + 3
        qkv = torch.randn(rows, (NH + 2 * NKV) * hs, generator=g, device=dev)
        # some channels of the keys are much larger than the rest, as in trained models
        qkv[:, NH * hs:(NH + NKV) * hs] *= 1 + 6 * (torch.rand(NKV * hs, generator=g, device=dev) > 0.95)
        slots = torch.randperm((blocks - 1) * bs, generator=g, device=dev)[:rows]
        slots[rows // 2] = -1 if rows > 1 else slots[0]  # a padding row
        s.update(qkv=qkv.bfloat16(), slots=slots, codes=torch.zeros(blocks, 2, NKV, bs, hs // 2, dtype=torch.uint8, device=dev),
                 scales=torch.zeros(blocks, 2, NKV, bs, hs // GROUP, 2, dtype=torch.bfloat16, device=dev),
                 out=torch.empty(rows, 2, NKV, hs, dtype=torch.bfloat16, device=dev))
    elif case["op"] == "attention":
        NH, NKV, hs, bs = (case[k] for k in ("NH", "NKV", "hs", "bs"))
        lens, rows = _attention_shape(case)
        held = [-(-n // bs) for n in lens]
        blocks = sum(held) + 1
        order = torch.randperm(blocks, generator=h).to(i32)
        table = torch.full((case["B"], max(held)), -1, dtype=i32)
        at = 0
        for b, k in enumerate(held):
            table[b, :k] = order[at:at + k]
            at += k
        codes = torch.empty(blocks, 2, NKV, bs, hs // 2, dtype=torch.uint8, device=dev)
        scales = torch.empty(blocks, 2, NKV, bs, hs // GROUP, 2, dtype=torch.bfloat16, device=dev)
        per = max(1, (1 << 26) // (2 * NKV * bs * hs))
        for at in range(0, blocks, per):  # bounded memory: a piece of the cache at a time
            x = torch.randn(min(per, blocks - at), 2, NKV, bs, hs, generator=g, device=dev)
            codes[at:at + per], scales[at:at + per] = _quantise(x.bfloat16())
        R = sum(rows)
        qkv = torch.randn(R + 2, (NH + 2 * NKV) * hs, generator=g, device=dev).bfloat16()  # two padding rows
        s.update(qkv=qkv, codes=codes, scales=scales, table=table.to(dev), lens=torch.tensor(lens, dtype=i32, device=dev),
                 start=_starts(rows, dev), out=torch.zeros(R + 2, NH * hs, dtype=torch.bfloat16, device=dev))
    elif case["op"] == "probs":
        logits = torch.randn(case["rows"], case["V"], generator=g, device=dev) * 3
        s.update(logits=logits, out=torch.empty_like(logits))
    else:
        B, V, rows = case["B"], case["V"], _draft_rows(case)
        R = sum(rows)
        logits = torch.randn(R, V, generator=g, device=dev) * 3
        p = _softmax(logits)
        q = _softmax(logits + 0.5 * torch.randn(R, V, generator=g, device=dev))
        tokens = torch.multinomial(q, 1, generator=g)[:, 0].roll(1).to(i32)  # row r holds the draft made from row r - 1
        s.update(p=p, q=q if case["q_given"] else None, tokens=tokens.contiguous(), start=_starts(rows, dev),
                 ua=torch.rand(R, generator=g, device=dev), us=torch.rand(B, generator=g, device=dev),
                 out=torch.empty(B, 1 + case["drafts"], dtype=i32, device=dev), taken=torch.empty(B, dtype=i32, device=dev))
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _quantise(x):
    """BF16 [..., hs] -> packed codes [..., hs/2] and (step, low end) [..., hs/64, 2]."""
    x = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    c = torch.tensor(1 / 15, dtype=torch.float32, device=x.device)
    t = hi * c - lo * c
    step = torch.where(t < 2.0 ** -120, 0, t).bfloat16().float()
    code = torch.where(step > 0, ((x * 0.5 - lo * 0.5) / (step * 0.5)).round().clamp(0, 15), 0)
    code = torch.where(bad, 0, code).to(torch.uint8).flatten(-2)
    scales = torch.where(bad, math.nan, torch.cat([step, lo], -1)).bfloat16()
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def _values(codes, scales):
    """Packed codes [..., hs/2] and (step, low end) [..., hs/64, 2] -> FP32 [..., hs]."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, GROUP)).float()
    return (code * scales[..., 0:1].float() + scales[..., 1:2].float()).flatten(-2)


def _softmax(x):
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_tables(s):
    bs, (B, mb), R = s["case"]["bs"], s["table"].shape, s["slot"].shape[0]
    n, ctx = s["new"].long().clamp(min=0), s["ctx"].long().clamp(min=0)
    have = s["have"].long().clamp(0, mb)
    F = s["free_count"].long().clamp(0, s["free"].shape[0])
    end, rows = ctx + n, n.cumsum(0)
    fits = (end <= mb * bs) & (rows <= R)
    need = torch.where(fits, ((end + bs - 1) // bs - have).clamp(min=0), 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= F))
    lens = torch.where(served, end, 0)
    left = F - torch.where(served & (need > 0), upto, 0).amax()
    j = torch.arange(mb, device=n.device)
    k = j[None] - have[:, None]
    new = served[:, None] & (k >= 0) & (k < need[:, None])
    at = (F - 1 - (upto - need)[:, None] - k).clamp(0, s["free"].shape[0] - 1)
    table = torch.where(new, s["free"][at], s["table"])
    start = torch.cat([rows.new_zeros(1), rows.clamp(max=R)])
    r = torch.arange(R, device=n.device)
    b = torch.searchsorted(rows, r, right=True)
    inside, b = b < B, b.clamp(max=B - 1)
    pos = ctx[b] + r - (rows - n)[b]
    block = table[b, (pos // bs).clamp(0, mb - 1)].long()
    slot = torch.where(inside & served[b] & (block >= 0), block * bs + pos % bs, -1)
    i32 = torch.int32
    return {"table": table, "slot": slot, "positions": torch.where(inside & served[b], pos, 0).to(i32),
            "row_start": start.to(i32), "lens": lens.to(i32), "blocks": torch.where(served, have + need, have).to(i32),
            "left": left.to(i32).reshape(1)}


def _plain_cache(s):
    c = s["case"]
    NH, NKV, hs, bs = (c[k] for k in ("NH", "NKV", "hs", "bs"))
    kv = s["qkv"][:, NH * hs:].unflatten(-1, (2, NKV, hs))
    codes, scales = _quantise(kv)
    # a padding row goes to the last block, which no request holds
    keep = s["slots"] >= 0
    slot = torch.where(keep, s["slots"], (s["codes"].shape[0] - 1) * bs)
    block, off = slot // bs, slot % bs
    s["codes"][block, :, :, off] = codes
    s["scales"][block, :, :, off] = scales
    values = _values(s["codes"][block, :, :, off], s["scales"][block, :, :, off])
    return torch.where(keep[:, None, None, None], values, 0).bfloat16()


def _plain_attention(s):
    c = s["case"]
    NH, NKV, hs, B, q = (c[k] for k in ("NH", "NKV", "hs", "B", "q"))
    start, lens, table = s["start"].long(), s["lens"].long(), s["table"].long().clamp(min=0)
    rows = start[1:] - start[:-1]
    # queries padded to [B, NKV, q * ratio, hs]
    i = torch.arange(q, device=start.device)
    x = s["qkv"][(start[:-1, None] + i).clamp(max=s["qkv"].shape[0] - 1), :NH * hs].float()
    x = x.view(B, q, NKV, NH // NKV, hs).transpose(1, 2).reshape(B, NKV, -1, hs)
    codes, scales = s["codes"][table], s["scales"][table]  # [B, blocks, 2, NKV, bs, ...]
    k = _values(codes[:, :, 0], scales[:, :, 0]).transpose(1, 2).flatten(2, 3)
    score = x @ k.transpose(-1, -2) / math.sqrt(hs)
    del k
    limit = (lens - rows)[:, None] + i  # last position that row i of a sequence sees
    seen = torch.arange(score.shape[-1], device=start.device) <= limit[..., None]
    seen = seen[:, None, :, None].expand(B, 1, q, NH // NKV, -1).flatten(2, 3)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(score - top), 0)
    total = e.sum(-1, keepdim=True)
    w = torch.where(total > 0, e / total, 0)
    v = _values(codes[:, :, 1], scales[:, :, 1]).transpose(1, 2).flatten(2, 3)
    o = (w @ v).view(B, NKV, q, -1, hs).transpose(1, 2).reshape(B, q, NH * hs)
    # back to packed rows; rows behind the last sequence stay as they were
    r = torch.arange(s["out"].shape[0], device=start.device)
    b = torch.searchsorted(start[1:].contiguous(), r, right=True)
    inside, b = b < B, b.clamp(max=B - 1)
    got = o[b, (r - start[b]).clamp(0, q - 1)]
    return torch.where(inside[:, None], got.bfloat16(), s["out"])


def _plain_verify(s):
    p, qs, start = s["p"], s["q"], s["start"].long()
    B, width, V = s["us"].shape[0], s["out"].shape[1], p.shape[1]
    n = (start[1:] - start[:-1] - 1).clamp(max=width - 1)
    i = torch.arange(width, device=p.device)
    row = (start[:-1, None] + i).clamp(max=p.shape[0] - 1)
    draft = s["tokens"][(row + 1).clamp(max=p.shape[0] - 1)].long()
    made = (i < n[:, None]) & (draft >= 0) & (draft < V)
    x = draft.clamp(0, V - 1)
    px = p[row, x].double()
    qx = qs[row, x].double() if qs is not None else torch.ones_like(px)
    ok = made & (s["ua"][row].double() * qx < px)
    taken = ok.long().cumprod(1).sum(1)
    b = torch.arange(B, device=p.device)
    at = row[b, taken]
    refused = made[b, taken]
    w = p[at].double()
    if qs is not None:
        rest = (w - qs[at].double()).clamp(min=0)
    else:
        rest = torch.where(torch.arange(V, device=p.device) == x[b, taken][:, None], 0, w)
    w = torch.where(refused[:, None] & (rest.sum(-1, keepdim=True) > 0), rest, w)
    run_ = w.cumsum(-1)
    over = run_ > s["us"].double()[:, None] * run_[:, -1:]
    k = torch.arange(V, device=p.device)
    last = torch.where(w > 0, k, -1).amax(-1)
    token = torch.where(over.any(-1), over.long().argmax(-1), last)
    out = torch.where(i < taken[:, None], draft, -1)
    out = torch.where(i == taken[:, None], token[:, None], out)
    return out.to(torch.int32), taken.to(torch.int32)


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        from cuda_gpt2_inference_b200 import ops
        if op == "tables":
            ops.kv_block_tables(s["table"], s["slot"], s["pos"], s["start"], s["lens"], s["have_out"], s["left"], s["ctx"], s["new"],
                                s["have"], s["free"], s["free_count"], s["case"]["bs"])
            return {"table": s["table"], "slot": s["slot"], "positions": s["pos"], "row_start": s["start"], "lens": s["lens"],
                    "blocks": s["have_out"], "left": s["left"]}
        if op == "cache":
            ops.kv_cache_write_w4(s["codes"], s["scales"], s["qkv"], s["slots"], s["case"]["NH"])
            ops.kv_cache_read_w4(s["out"], s["codes"], s["scales"], s["slots"])
            return s["out"]
        if op == "attention":
            if "workspace" not in s:  # made by the first pass and kept, as a program does
                s["workspace"] = torch.empty(ops.attention_paged_w4_workspace(s["case"]["NH"], s["case"]["NKV"], s["case"]["hs"],
                                                                              s["case"]["q"]), dtype=torch.uint8, device="cuda")
            ops.attention_forward_paged_w4(s["out"], s["qkv"], s["codes"], s["scales"], s["table"], s["lens"], s["start"],
                                           s["case"]["NH"], s["case"]["q"], s["workspace"])
            return s["out"]
        if op == "probs":
            ops.softmax_probs(s["out"], s["logits"], s["case"]["T"])
            return s["out"]
        ops.verify_draft_tokens(s["out"], s["taken"], s["tokens"], s["p"], s["q"], s["start"], s["ua"], s["us"])
        return s["out"], s["taken"]
    if op == "tables":
        return _plain_tables(s)
    if op == "cache":
        return _plain_cache(s)
    if op == "attention":
        return _plain_attention(s)
    if op == "probs":
        return _softmax(s["logits"] / s["case"]["T"])
    return _plain_verify(s)


# ---------------------------------------------------------------------------
# work, and the definition in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "tables":
        ctx, new = _table_lengths(case)
        R, B, bs = sum(new) + 3, case["B"], case["bs"]
        grown = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(ctx, new))
        return {"bytes": 12 * R + 4 * (6 * B + 3) + 8 * grown, "flops": 0}
    if case["op"] == "cache":
        rows, n = case["rows"], 2 * case["NKV"] * case["hs"]
        return {"bytes": rows * (n * 2 + 2 * (n // 2 + n // GROUP * 4) + n * 2 + 16), "flops": 0}
    if case["op"] == "attention":
        lens, rows = _attention_shape(case)
        NH, NKV, hs = case["NH"], case["NKV"], case["hs"]
        row = 2 * NKV * (hs // 2 + hs // GROUP * 4)
        return {"bytes": sum(lens) * row + sum(rows) * NH * hs * 4 + 4 * sum(-(-n // case["bs"]) for n in lens),
                "flops": 4 * sum(a * b for a, b in zip(lens, rows)) * NH * hs}
    if case["op"] == "probs":
        return {"bytes": 8 * case["rows"] * case["V"], "flops": 0}
    rows = _draft_rows(case)
    return {"bytes": 4 * case["B"] * case["V"] + 16 * sum(rows), "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "probs":
        x = s["logits"].double() / case["T"]
        return (x - torch.logsumexp(x, -1, keepdim=True)).exp()
    if op == "cache":
        NH, NKV, hs = case["NH"], case["NKV"], case["hs"]
        x = s["qkv"].view(case["rows"], -1, hs)[:, NH:].view(case["rows"], 2, NKV, hs // GROUP, GROUP)
        low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
        # the step is held in BF16, rounded from 32 bits by definition
        step = (high.float() * (1 / 15) - low.float() * (1 / 15)).to(torch.bfloat16).double()
        low = low.double()
        code = torch.where(step > 0, torch.round((x.double() - low) / step), torch.zeros_like(step)).clamp_(0, 15)
        value = (low + code * step).view(case["rows"], 2, NKV, hs)
        value[s["slots"] < 0] = 0
        return value
    if op == "attention":
        NH, NKV, hs, bs = (case[k] for k in ("NH", "NKV", "hs", "bs"))
        lens, rows = _attention_shape(case)
        if sum(lens) * NKV * hs > 1 << 30:
            return None
        out, at = s["out"].double(), 0
        for b, (n, m) in enumerate(zip(lens, rows)):
            blocks = s["table"][b, :-(-n // bs)].long()
            nibbles = s["codes"][blocks]
            v = torch.empty(*nibbles.shape[:-1], hs, dtype=torch.float64, device=nibbles.device)
            v[..., 0::2], v[..., 1::2] = (nibbles % 16).double(), (nibbles // 16).double()
            sc = s["scales"][blocks].double()
            v = v * sc[..., 0].repeat_interleave(GROUP, -1) + sc[..., 1].repeat_interleave(GROUP, -1)
            v = v.permute(1, 2, 0, 3, 4).reshape(2, NKV, -1, hs)[:, :, :n]
            for i in range(m):
                last = n - m + i + 1
                if last > 0:
                    x = s["qkv"][at + i, :NH * hs].double().view(NKV, NH // NKV, hs)
                    w = torch.softmax(torch.einsum("hrd,hpd->hrp", x, v[0, :, :last]) / math.sqrt(hs), -1)
                    out[at + i] = torch.einsum("hrp,hpd->hrd", w, v[1, :, :last]).reshape(-1)
                else:
                    out[at + i] = 0
            at += m
        return out
    if op == "tables":
        bs, mb, R = case["bs"], case["max_blocks"], s["slot"].shape[0]
        ctx, new, have = s["ctx"].tolist(), s["new"].tolist(), s["have"].tolist()
        table, free, F = s["table"].tolist(), s["free"].tolist(), int(s["free_count"])
        slot, pos, start, lens, held = [], [], [0], [], []
        asked, left = 0, F
        for b in range(case["B"]):
            end = ctx[b] + new[b]
            fits = end <= mb * bs
            need = max(0, -(-end // bs) - have[b]) if fits else 0
            good = fits and (need == 0 or asked + need <= F)
            if good and need:
                for j in range(need):
                    table[b][have[b] + j] = free[F - 1 - asked - j]
                left = F - asked - need
            asked += need
            for t in range(ctx[b], end):
                slot.append(table[b][t // bs] * bs + t % bs if good else -1)
                pos.append(t if good else 0)
            start.append(start[-1] + new[b])
            lens.append(end if good else 0)
            held.append(have[b] + need if good else have[b])
        slot += [-1] * (R - len(slot))
        pos += [0] * (R - len(pos))
        t32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
        return {"table": t32(table), "slot": torch.tensor(slot), "positions": t32(pos), "row_start": t32(start), "lens": t32(lens),
                "blocks": t32(held), "left": t32([left])}
    start = s["start"].tolist()
    tokens = s["tokens"].tolist()
    out, taken = [], []
    for b in range(case["B"]):
        got, r, end = [], start[b], start[b + 1]
        w = None
        while r + 1 < end:
            x = tokens[r + 1]
            q = s["q"][r].double() if s["q"] is not None else None
            if float(s["ua"][r]) * (float(q[x]) if q is not None else 1.0) < float(s["p"][r, x]):
                got.append(x)
                r += 1
                continue
            w = s["p"][r].double()
            if q is not None:
                w = torch.relu(w - q)
            else:
                w[x] = 0
            break
        if w is None or float(w.sum()) == 0:
            w = s["p"][r].double()
        c = torch.cumsum(w, 0)
        k = int(torch.searchsorted(c, (s["us"][b].double() * c[-1]).reshape(1), right=True))
        taken.append(len(got))
        got.append(min(k, int(w.nonzero()[-1])))
        out.append(got + [-1] * (1 + case["drafts"] - len(got)))
    return torch.tensor(out, dtype=torch.int32), torch.tensor(taken, dtype=torch.int32)
