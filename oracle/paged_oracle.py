"""CPU restatement of the operators over a paged K/V cache in 64 bits: one sequence, token and head after the other."""
from __future__ import annotations

import math

import torch


def quantise_row(x: torch.Tensor):
    """(codes as the numbers they stand for, scale) of one row: the least power of two from 2^-126 on with max|x| <= 448 s."""
    x = x.double()
    if not torch.isfinite(x).all():
        return torch.zeros_like(x), math.nan
    top = x.abs().max().item()
    scale = 1.0
    if top > 0:
        e = -126
        while top > 448 * 2.0 ** e:
            e += 1
        scale = 2.0 ** e
    y = x / scale
    step = torch.tensor([2.0 ** (max(math.frexp(v)[1] - 1, -6) - 3) for v in y.tolist()], dtype=torch.float64)
    return torch.round(y / step) * step, scale           # (torch.round goes to the even one of two)


def tokens_of(b: int, x: torch.Tensor, starts):
    """Sequence b's new tokens and where in x they lie."""
    if starts is None:
        return x[b]
    return x[starts[b]:starts[b + 1]]


def paged_write(k, v, cache, table, lengths, scales=None, starts=None):
    """In place, on CPU tensors; cache in float64 (codes as numbers) where there are scales."""
    pages, page = cache.shape[1:3]
    for b, length in enumerate(lengths):
        for half, x in ((0, tokens_of(b, k, starts)), (1, tokens_of(b, v, starts))):
            for i in range(x.shape[0]):
                j = length - x.shape[0] + i
                if j < 0 or not 0 <= table[b][j // page] < pages:
                    continue
                for h in range(x.shape[1]):
                    if scales is None:
                        cache[half, table[b][j // page], j % page, h] = x[i, h]
                    else:
                        cache[half, table[b][j // page], j % page, h], scales[half, table[b][j // page], j % page, h] = quantise_row(x[i, h])


def rows_of(cache, scales, table, length, b):
    """(2, length, Hkv, D) in 64 bits and which of the rows are here."""
    pages, page = cache.shape[1:3]
    here = torch.tensor([0 <= table[b][j // page] < pages for j in range(length)], dtype=torch.bool)
    x = torch.zeros(2, length, *cache.shape[3:], dtype=torch.float64)
    for j in range(length):
        if here[j]:
            row = cache[:, table[b][j // page], j % page].double()
            x[:, j] = row if scales is None else row * scales[:, table[b][j // page], j % page].double()[..., None]
    return x, here


def paged_read(cache, table, lengths, rows, begin=0, scales=None):
    out = torch.zeros(2, len(lengths), rows, *cache.shape[3:], dtype=torch.float64)
    for b, length in enumerate(lengths):
        x, _ = rows_of(cache, scales, table, length, b)
        x = x[:, begin:begin + rows]
        out[:, b, :x.shape[1]] = x
    return out


def paged_attention(q, cache, table, lengths, scale, causal=True, scales=None, starts=None):
    """Per sequence (out (n, Hq, D), lse (Hq, n), how far a kernel may be off in out, and in lse).

    The bound: a kernel that multiplies bf16 by bf16 exactly and sums in fp32 has scores off by delta = scale * sum|q k| * (D + 4)
    2^-24, weights by that and half a step of bf16 (2^-8) relatively, sums of S terms by (S + 64) 2^-23, and rounds the
    result by half a step of bf16."""
    got = []
    for b, length in enumerate(lengths):
        x, here = rows_of(cache, scales, table, length, b)
        qs = tokens_of(b, q, starts).double()
        n, Hq, D = qs.shape
        G = Hq // cache.shape[3]
        out, lse = torch.zeros(n, Hq, D, dtype=torch.float64), torch.full((Hq, n), -math.inf, dtype=torch.float64)
        out_off, lse_off = torch.zeros_like(out), torch.zeros_like(lse)
        for i in range(n):
            seen = here.clone()
            if causal:
                seen[max(length - n + i + 1, 0):] = False
            if not seen.any():
                continue
            k, v = x[0][seen], x[1][seen]
            for h in range(Hq):
                score = k[:, h // G] @ qs[i, h] * scale
                delta = ((k[:, h // G].abs() @ qs[i, h].abs()).max() * scale * (D + 4) * 2.0 ** -24).item()
                sums = (k.shape[0] + 64) * 2.0 ** -23
                weight = torch.softmax(score, 0)
                out[i, h] = weight @ v[:, h // G]
                lse[h, i] = torch.logsumexp(score, 0)
                out_off[i, h] = (weight @ v[:, h // G].abs()) * (2.0 ** -8 + 2 * delta + sums) * (1 + 2.0 ** -8) + 2.0 ** -8 * out[i, h].abs()
                lse_off[h, i] = delta + sums + abs(lse[h, i].item()) * 2.0 ** -22
        got.append((out, lse, out_off, lse_off))
    return got


# The columns of a row in e2m1, 32 at a time: code c stands for E2M1[c % 8], negative from 8 on, times 2^(byte - 127).
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantise_block(x: torch.Tensor):
    """(codes, byte of the scale) of 32 columns: the least power of two from 2^-126 to 2^125 with max|x| <= 6 s."""
    x = x.double()
    if not torch.isfinite(x).all():
        return [0] * x.numel(), 255
    top, e = x.abs().max().item(), 0
    if top > 0:
        e = -126
        while top > 6 * 2.0 ** e and e < 125:
            e += 1
    codes = []
    for v in x.tolist():
        y = abs(v) / 2.0 ** e
        # the nearest, of two equally near the even code, and nothing beyond 6
        best = min(range(8), key=lambda c: (abs(E2M1[c] - y), c % 2))
        codes.append(best + (8 if math.copysign(1.0, v) < 0 else 0))
    return codes, e + 127


def quantise_e2m1(x: torch.Tensor):
    """A row of D columns as D / 2 bytes of two codes and D / 32 bytes of scales."""
    codes, scales = [], []
    for block in x.view(-1, 32):
        c, s = quantise_block(block)
        codes += c
        scales.append(s)
    return torch.tensor([lo + 16 * hi for lo, hi in zip(codes[::2], codes[1::2])], dtype=torch.uint8), torch.tensor(scales, dtype=torch.uint8)


def e2m1_values(codes: torch.Tensor, scales: torch.Tensor):
    """What bytes (..., D / 2) and scales (..., 4) stand for, (..., D) in 64 bits."""
    table = torch.tensor([*E2M1, *(-v for v in E2M1)], dtype=torch.float64)
    x = torch.stack([table[(codes % 16).long()], table[(codes // 16).long()]], -1).flatten(-2)
    power = torch.where(scales == 255, math.nan, torch.exp2(scales.double() - 127))
    return x * power.repeat_interleave(32, -1)[..., :x.shape[-1]]


def paged_write_e2m1(k, v, codes, scales, table, lengths, starts=None):
    """In place, on CPU tensors of bytes (2, pages, page, Hkv, D / 2) and (2, pages, page, Hkv, 4)."""
    pages, page = codes.shape[1:3]
    for b, length in enumerate(lengths):
        for half, x in ((0, tokens_of(b, k, starts)), (1, tokens_of(b, v, starts))):
            for i in range(x.shape[0]):
                j = length - x.shape[0] + i
                if j < 0 or not 0 <= table[b][j // page] < pages:
                    continue
                for h in range(x.shape[1]):
                    row, scale = quantise_e2m1(x[i, h])
                    codes[half, table[b][j // page], j % page, h] = row
                    scales[half, table[b][j // page], j % page, h, :scale.numel()] = scale


def paged_weights(q, cache, table, lengths, scale, lse, weights, causal=True, starts=None, decay=1.0):
    """What attention each key has had, (pages, page, Hkv) in 64 bits, and how far a kernel may be off.

    The bound: with scores off by delta as in paged_attention, a weight exp(s - lse) that is formed in fp32 as 2^(s c - lse c) is
    off by delta + 2^-22 (|s| + |lse|) + 2^-21 relatively, a sum of N weights by N 2^-23 more, and decay times the old one by 2^-23."""
    out, off = weights.double().clone(), torch.zeros(weights.shape, dtype=torch.float64)
    pages, page = cache.shape[1:3]
    for b, length in enumerate(lengths):
        x, here = rows_of(cache, None, table, length, b)
        qs = tokens_of(b, q, starts).double()
        n, Hq, D = qs.shape
        if n == 0:
            continue
        G = Hq // cache.shape[3]
        for h in range(cache.shape[3]):
            total, wrong = torch.zeros(length, dtype=torch.float64), torch.zeros(length, dtype=torch.float64)
            for i in range(n):
                sees = max(length - n + i + 1, 0) if causal else length
                for g in range(G):
                    row = h * G + g
                    l = (lse[b, row, i] if starts is None else lse[row, starts[b] + i]).double().item()
                    if l == -math.inf:
                        continue
                    score = x[0, :sees, h] @ qs[i, row] * scale
                    weight = torch.exp(score - l)
                    delta = x[0, :sees, h].abs() @ qs[i, row].abs() * scale * (D + 4) * 2.0 ** -24
                    total[:sees] += weight
                    wrong[:sees] += weight * (delta + 2.0 ** -22 * (score.abs() + abs(l)) + 2.0 ** -21)
            wrong += total * n * G * 2.0 ** -23
            for j in range(length):
                if here[j]:
                    at = table[b][j // page], j % page, h
                    old = decay * weights[at].double().item() if j < length - n and decay else 0.0
                    out[at], off[at] = old + total[j], wrong[j] + 2.0 ** -23 * abs(old + total[j].item())
    return out, off


def evicted(weights, table, lengths, pages, keep, recent=0, limit=None):
    """kept[b][h], the positions that stay (None where a page is not here), and left[b]."""
    limit = keep if limit is None else limit
    page, Hkv = weights.shape[1:]
    kept, left = [], []
    for b, length in enumerate(lengths):
        if any(not 0 <= table[b][j] < pages for j in range(-(-length // page))):
            kept.append(None)
            left.append(length)
            continue
        left.append(keep if length > limit else length)
        kept.append([])
        for h in range(Hkv):
            stay = list(range(length))
            if length > limit:
                others = list(range(length - recent))
                value = [weights[table[b][j // page], j % page, h].item() for j in others]
                rank = sorted(others, key=lambda j: (0 if math.isnan(value[j]) else 1, 0.0 if math.isnan(value[j]) else -value[j], j))
                stay = sorted(rank[:keep - recent]) + list(range(length - recent, length))
            kept[b].append(stay)
    return kept, left
