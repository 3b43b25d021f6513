"""Plain CPU forms of the paged 4-bit cache operators and of draft verification, in 64 bits."""
from __future__ import annotations

import math

import torch

GROUP = 64
BF16, FP16 = 2.0 ** -8, 2.0 ** -11  # half a step relative to the value


def quantise(x):
    """BF16 [..., hs] -> codes u8 [..., hs/2], (step, low end) BF16 [..., hs/64, 2], as the header defines them."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    fin = torch.isfinite(g).all(-1, keepdim=True)
    c = torch.tensor(1.0, dtype=torch.float32) / 15  # FP32 products and difference, each rounded
    t = hi * c - lo * c
    t = torch.where(t < 2.0 ** -120, torch.zeros_like(t), t)
    step = t.bfloat16().double()
    code = torch.where(step > 0, torch.round((g.double() - lo.double()) / step), torch.zeros_like(step)).clamp(0, 15)
    code = torch.where(fin, code, torch.zeros_like(code)).to(torch.uint8).flatten(-2)
    meta = torch.where(fin, torch.cat([step, lo.double()], -1), torch.full((1,), math.nan, dtype=torch.float64)).bfloat16()
    return code[..., 0::2] | (code[..., 1::2] << 4), meta


def values(codes, scales, magnitude=False):
    """Values [..., hs] in 64 bits; ``magnitude``: code * step + |low end|, what bounds their rounding errors."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, GROUP)).double()
    lo = scales[..., 1:2].double()
    return (c * scales[..., 0:1].double() + (lo.abs() if magnitude else lo)).flatten(-2)


def attention(qkv, codes, scales, table, lens, start, NH, scale=None):
    """out [rows, NH*hs] in 64 bits (NaN rows: behind the last request) and the bound of its errors
    before the output's own rounding."""
    _, _, NKV, bs, half = codes.shape
    hs, R = 2 * half, qkv.shape[0]
    scale = 1 / math.sqrt(hs) if scale is None else scale
    out = torch.full((R, NH, hs), math.nan, dtype=torch.float64)
    err = torch.zeros_like(out)
    for b in range(len(lens)):
        n, r0 = int(lens[b]), int(start[b])
        m = int(start[b + 1]) - r0
        held = table[b, :-(-n // bs)].long()
        k, v, va, ka = (values(codes[held, i], scales[held, i], mag).transpose(0, 1).flatten(1, 2)[:, :n]
                        for i, mag in ((0, False), (1, False), (1, True), (0, True)))
        for i in range(m):
            seen = max(0, n - m + i + 1)
            if seen == 0:
                out[r0 + i] = 0
                continue
            x = qkv[r0 + i, :NH * hs].double().view(NKV, NH // NKV, hs)
            s = scale * torch.einsum("hrd,hpd->hrp", x, k[:, :seen])
            w = torch.softmax(s, -1)
            out[r0 + i] = torch.einsum("hrp,hpd->hrd", w, v[:, :seen]).flatten(0, 1)
            # a score is a 32-bit sum of hs products of exact factors (hs + 8 roundings, of magnitude
            # |q||k|), twice (numerator and sum); a weight is held in 16 bits; e^x and the sums add
            # a few 32-bit roundings
            sa = abs(scale) * torch.einsum("hrd,hpd->hrp", x.abs(), ka[:, :seen]).amax(-1, keepdim=True)
            rel = 2 * (hs + 8) * 2.0 ** -24 * sa + FP16 + 2.0 ** -16
            mag = torch.einsum("hrp,hpd->hrd", w, va[:, :seen])
            # weights below 2^-18 of the largest step are held with an absolute error
            floor = seen * 2.0 ** -29 * va[:, :seen].amax((1, 2))[:, None, None]
            err[r0 + i] = (rel * mag + floor).flatten(0, 1)
    return out.flatten(1), err.flatten(1)


def tables(table, ctx, new, have, free, count, bs, max_rows):
    """kv_block_tables on lists; returns (table, slots, positions, start, lens, blocks, left)."""
    table = [list(r) for r in table]
    mb = len(table[0])
    F = min(max(count, 0), len(free))
    slots, pos, start, lens, blocks = [-1] * max_rows, [0] * max_rows, [0], [], []
    rows, asked, left = 0, 0, F
    for b in range(len(table)):
        c, n, h = max(ctx[b], 0), max(new[b], 0), min(max(have[b], 0), mb)
        end = c + n
        fits = end <= mb * bs and rows + n <= max_rows
        need = max(0, -(-end // bs) - h) if fits else 0
        served = fits and (need == 0 or asked + need <= F)
        if served:
            for j in range(need):
                table[b][h + j] = free[F - 1 - asked - j]
            if need:
                left = F - asked - need
            for i in range(n):
                blk = table[b][(c + i) // bs]
                slots[rows + i] = blk * bs + (c + i) % bs if blk >= 0 else -1
                pos[rows + i] = c + i
        asked += need
        rows += n
        start.append(min(rows, max_rows))
        lens.append(end if served else 0)
        blocks.append(h + need if served else h)
    return table, slots, pos, start, lens, blocks, left


def verify(tokens, p, q, start, ua, us, max_out):
    """verify_draft_tokens on CPU tensors: (out_tokens, n_accepted) as lists."""
    out, taken = [], []
    V = p.shape[1]
    for b in range(len(start) - 1):
        r, end = start[b], start[b + 1]
        got, w = [], None
        if r == end:
            out.append([-1] * max_out)
            taken.append(0)
            continue
        while r + 1 < end and len(got) < max_out - 1:
            x = int(tokens[r + 1])
            if not 0 <= x < V:
                break
            qx = float(q[r, x]) if q is not None else 1.0
            if float(ua[r]) * qx < float(p[r, x]):
                got.append(x)
                r += 1
                continue
            w = p[r].double() - q[r].double() if q is not None else p[r].double().clone()
            if q is None:
                w[x] = 0
            break
        if w is not None:
            w = torch.where(w > 0, w, torch.zeros_like(w))  # NaN counts as nothing
        if w is None or not float(w.sum()) > 0:
            w = p[r].double()
            w = torch.where(w > 0, w, torch.zeros_like(w))
        c = torch.cumsum(w, 0)
        over = (c > float(us[b]) * float(c[-1])).nonzero()
        some = (w > 0).nonzero()
        pick = int(over[0]) if len(over) else int(some[-1]) if len(some) else -1
        taken.append(len(got))
        got.append(pick)
        out.append(got + [-1] * (max_out - len(got)))
    return out, taken
