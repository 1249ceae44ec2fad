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
