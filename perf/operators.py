"""What is measured of the operators over a paged K/V cache: writing new tokens into it, reading rows of it back as a
dense chunk, and attention of new tokens over it.

A cache is ``(2, pages, page_size, Hkv, D)``, keys and values, in bfloat16 or in e4m3 with one fp32 scale for each row
(``(2, pages, page_size, Hkv)``, a power of two).  ``page_table`` (B, pages of a sequence) says where each sequence's
tokens lie, ``lengths`` (B) how many there are, the new ones among them.  New tokens come as (B, n, H, D), or packed as
(T, H, D) with ``starts`` (B + 1).

Parameters of a case: ``op``; ``B`` sequences of ``low`` to ``high`` tokens; ``new`` of them new in each sequence, or from
``new_low`` to ``new`` where they come ``packed``; ``Hq`` / ``Hkv`` heads of ``D`` columns; ``page`` rows of a page;
``e4m3`` or bfloat16; for reading, ``rows`` of every sequence from ``begin`` on.
"""
from __future__ import annotations

import math

import torch

own = False
DEVICE = "cuda:0"


def _case(op, B, low, high, Hkv, D, page, e4m3, **more):
    return dict(op=op, B=B, low=low, high=high, Hkv=Hkv, D=D, page=page, e4m3=e4m3, **more)


def listed():
    return [
        # One sequence of a unit-scale model (4 heads of 64), one new token: launches and host work are what counts.
        _case("attn", 1, 1024, 1024, 4, 64, 16, False, Hq=4, new=1, new_low=1, packed=False, name="decode_one"),
        # A batch in steady generation: 32 sequences at all stages of up to 16384 tokens, grouped heads.
        _case("attn", 32, 300, 16384, 8, 128, 16, False, Hq=32, new=1, new_low=1, packed=False, name="decode_ragged_gqa"),
        # Few sequences of the long-context configuration's 131072 tokens, the cache in e4m3: all of the time is reading it.
        _case("attn", 4, 131000, 131072, 8, 128, 64, True, Hq=32, new=1, new_low=1, packed=False, name="decode_e4m3_128k"),
        # Five tokens of each sequence checked at once (a draft of four and the one before), head dimension 80.
        _case("attn", 16, 211, 4099, 8, 80, 32, False, Hq=16, new=5, new_low=5, packed=False, name="verify_d80"),
        # A chunk of 2048 tokens at the end of a 32768-token prompt: the products are what counts.  The largest.
        _case("attn", 1, 32768, 32768, 8, 128, 16, False, Hq=32, new=2048, new_low=2048, packed=False, name="chunk_32k"),
        # A serving step: sequences that generate beside sequences whose prompts go in by chunks of up to 512, packed.
        _case("attn", 16, 600, 8192, 4, 128, 32, True, Hq=32, new=512, new_low=1, packed=True, name="mixed_e4m3"),
        # What a step of generation writes: one token of each of 64 sequences, quantised.
        _case("write", 64, 17, 1024, 8, 128, 16, True, new=1, new_low=1, packed=False, name="write_step_e4m3"),
        # What a step with prompts in it writes: 8 sequences' chunks of uneven length, about 16000 tokens, quantised.
        _case("write", 8, 2500, 4096, 8, 128, 16, True, new=2500, new_low=1500, packed=True, name="write_chunks_e4m3"),
        # Two uneven prompts of 1237 tokens into a bfloat16 cache, head dimension 80.
        _case("write", 2, 1237, 1900, 8, 80, 32, False, new=1237, new_low=1237, packed=False, name="write_d80"),
        # A cached 32768-token prefix becomes a K/V chunk of the ring (B1, 32 heads), which takes bfloat16.
        _case("read", 1, 32768, 32768, 32, 128, 64, True, begin=0, rows=32768, name="read_prefix_32k"),
        # Rows 300 to 1800 of eight sequences, some of which end before that; 12 heads of 64.
        _case("read", 8, 200, 2500, 12, 64, 16, False, begin=300, rows=1500, name="read_rows_d64"),
        # The last 256 tokens of a unit-scale model's sequence.
        _case("read", 1, 1024, 1024, 4, 64, 16, True, begin=768, rows=256, name="read_small"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


# what a drawn case may cost: that of the largest listed one
_MOST_FLOPS, _MOST_BYTES, _MOST_SCORES = 1.0e12, 1.0e9, 2.2e9


def draw(rng):
    while True:
        op = rng.choice(["attn", "attn", "attn", "write", "read"])
        e4m3 = rng.random() < 0.5
        D = rng.choice([64, 128, 128, 128, 16 * rng.randint(1, 8)] + ([] if e4m3 else [8 * rng.randint(1, 16)]))
        page = rng.choice([16, 16, 32, 48, 64, 128, 256])
        Hkv = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
        B = _log(rng, 1, 128)
        high = _log(rng, 16, 131072)
        low = rng.choice([high, max(1, high // 2), max(1, high // 50)])
        if op == "read":
            begin = rng.choice([0, 0, rng.randint(0, high - 1)])
            c = _case(op, B, low, high, Hkv, D, page, e4m3, begin=begin, rows=rng.randint(1, high - begin))
        else:
            kind = rng.choice(["one", "few", "chunk", "packed", "packed"])
            new = 1 if kind == "one" else rng.randint(2, 16) if kind == "few" else _log(rng, 2, 8192)
            if new > high:
                continue
            c = _case(op, B, low, high, Hkv, D, page, e4m3, new=new, packed=kind == "packed",
                      new_low=rng.choice([1, max(1, new // 3)]) if kind == "packed" else new)
            if op == "attn":
                c["Hq"] = Hkv * rng.choice([1, 1, 2, 4, 7, 8, 16])
                if c["Hq"] > 128 or B * c["Hq"] * new * high > _MOST_SCORES:
                    continue
        w = work(c)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES and B * high * Hkv * D < 5.5e8:
            return c


def _spread(low, high, B, step):
    """B whole numbers from low to high, the first of them high, in no order."""
    return [high - int((high - low) * ((b * step) % 1.0) + 0.5) for b in range(B)]


def _sizes(c):
    """(lengths, new tokens) of the sequences of a case; no sequence has fewer tokens than new ones."""
    lengths = _spread(c["low"], c["high"], c["B"], 0.618034)
    if c["op"] == "read":
        return lengths, [0] * c["B"]
    new = _spread(c["new_low"], c["new"], c["B"], 0.414214)
    if c["packed"]:                  # half of the sequences that generate have one new token
        new = [1 if c["new_low"] == 1 and b % 2 else n for b, n in enumerate(new)]
    return [max(t, n) for t, n in zip(lengths, new)], new


def work(c):
    lengths, new = _sizes(c)
    element, scale = (1, 4) if c["e4m3"] else (2, 0)
    row = c["D"] * element + scale
    table = 4 * sum(-(-t // c["page"]) for t in lengths)
    if c["op"] == "read":
        held = sum(min(max(t - c["begin"], 0), c["rows"]) for t in lengths)
        return {"bytes": 2 * c["Hkv"] * (held * row + c["B"] * c["rows"] * c["D"] * 2) + 4 * c["B"] * -(-c["rows"] // c["page"]),
                "flops": 2 * c["Hkv"] * held * c["D"]}
    T = sum(new)
    if c["op"] == "write":
        return {"bytes": 2 * c["Hkv"] * T * (c["D"] * 2 + row) + 4 * T, "flops": 2 * c["Hkv"] * T * c["D"]}
    pairs = sum(n * t - n * (n - 1) // 2 for t, n in zip(lengths, new))
    return {"bytes": 2 * c["Hkv"] * row * sum(lengths) + T * c["Hq"] * (4 * c["D"] + 4) + table, "flops": 4 * c["Hq"] * c["D"] * pairs}


def _e4m3(x):
    """Codes and scales of rows: the scale is the least power of two that keeps the row's largest value within 448, so
    that dividing by it is exact, and a code's step is the same share of its value as with any other scale."""
    x = x.float()
    top = x.abs().amax(-1)
    part, power = torch.frexp(top)                       # top = part * 2^power, 0.5 <= part < 1, and 448 = 0.875 * 2^9
    power = torch.where(top > 0, (power - 9 + (part > 0.875).int()).clamp(min=-126), torch.zeros_like(power))
    scale = ((power + 127) << 23).view(torch.float32)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def prepare(c, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, gain=1.0):
        return (torch.randn(*shape, generator=g, device=DEVICE) * gain).bfloat16()

    lengths, new = _sizes(c)
    counts = [-(-t // c["page"]) for t in lengths]
    pages = sum(counts) + 3                              # some are free
    order = torch.randperm(pages, generator=g, device=DEVICE).int()
    table = torch.full((c["B"], max(counts)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, count in enumerate(counts):
        table[b, :count] = order[at:at + count]
        at += count
    # in memory the rows of one head of a page lie together
    rows = torch.empty(2, pages, c["Hkv"], c["page"], c["D"], dtype=torch.bfloat16, device=DEVICE)
    for half in rows:
        half.copy_(normal(*half.shape))
    s = {"c": c, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEVICE), "scales": None, "starts": None}
    if c["e4m3"]:
        codes, scales = torch.empty(rows.shape, dtype=torch.float8_e4m3fn, device=DEVICE), torch.empty(rows.shape[:-1], device=DEVICE)
        for half, code, scale in zip(rows, codes, scales):
            code_, scale_ = _e4m3(half)
            code.copy_(code_)
            scale.copy_(scale_)
        rows, s["scales"] = codes, scales.transpose(2, 3)
    s["cache"] = rows.transpose(2, 3)
    if c["op"] != "read":
        shape = (sum(new),) if c["packed"] else (c["B"], c["new"])
        if c["packed"]:
            s["starts"] = torch.tensor([0, *new], dtype=torch.int32, device=DEVICE).cumsum(0, dtype=torch.int32)
        if c["op"] == "write":
            # one token's keys and values are large now and then, as in earnest
            gain = torch.exp(torch.randn(*shape, 1, 1, generator=g, device=DEVICE))
            s["k"], s["v"] = normal(*shape, c["Hkv"], c["D"], gain=gain), normal(*shape, c["Hkv"], c["D"], gain=gain)
        else:
            s["q"] = normal(*shape, c["Hq"], c["D"])
    return s


def run(s):
    c = s["c"]
    if c["op"] == "write":
        return _write(s)
    return _read(s) if c["op"] == "read" else _attn(s)


def _bytes(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _rows_of(s, half, first, rows):
    """Rows first .. first + rows of every sequence, (B, rows, Hkv, D) in fp32, zeros where there are none, and which there are."""
    cache, scales, page = s["cache"], s["scales"], s["c"]["page"]
    position = first + torch.arange(rows, device=DEVICE)
    there = position < s["lengths"][:, None]
    column = (position // page).clamp(max=s["table"].shape[1] - 1)
    at = s["table"][:, column].clamp(min=0).long()
    x = _bytes(cache[half])[at, position % page].view(cache.dtype).float()
    if scales is not None:
        x = x * scales[half][at, position % page][..., None]
    return torch.where(there[..., None, None], x, 0.0), there


def _places(s, T):
    """Sequence, number among its new tokens and position of every token of a packed batch."""
    token = torch.arange(T, device=DEVICE)
    starts = s["starts"].long()
    b = torch.searchsorted(starts, token, right=True) - 1
    i = token - starts[b]
    return b, i, s["lengths"][b] - (starts[b + 1] - starts[b]) + i


def _write(s):
    k, v, c = s["k"], s["v"], s["c"]
    if own:
        import mercury_artifact_amd as M
        M.paged_cache_write(k, v, s["cache"], s["table"], s["lengths"], scales=s["scales"], starts=s["starts"])
    else:
        if c["packed"]:
            b, _, position = _places(s, k.shape[0])
        else:
            b = torch.arange(c["B"], device=DEVICE)[:, None].expand(k.shape[:2])
            position = s["lengths"][:, None] - c["new"] + torch.arange(c["new"], device=DEVICE)
        at, slot = s["table"][b, position // c["page"]].long(), position % c["page"]
        kv = torch.stack([k, v])
        if c["e4m3"]:
            kv, scale = _e4m3(kv)
            s["scales"][:, at, slot] = scale
        _bytes(s["cache"])[:, at, slot] = _bytes(kv)
    return (s["cache"],) if s["scales"] is None else (s["cache"], s["scales"])


def _read(s):
    c = s["c"]
    if own:
        import mercury_artifact_amd as M
        return M.paged_cache_read(s["cache"], s["table"], s["lengths"], c["rows"], begin=c["begin"], scales=s["scales"])
    return torch.stack([_rows_of(s, half, c["begin"], c["rows"])[0] for half in (0, 1)]).bfloat16()


def _attn(s):
    c, q = s["c"], s["q"]
    scale = c["D"] ** -0.5
    if own:
        import mercury_artifact_amd as M
        return M.paged_attn_fwd(q, s["cache"], s["table"], s["lengths"], scale, causal=True, scales=s["scales"], starts=s["starts"],
                                most_new=c["new"])
    B, Hq, Hkv, D, n = c["B"], c["Hq"], c["Hkv"], c["D"], c["new"]
    if c["packed"]:
        b, i, _ = _places(s, q.shape[0])
        count = s["starts"][1:] - s["starts"][:-1]
        padded = torch.zeros(B, n, Hq, D, device=DEVICE)
        padded[b, i] = q.float()
    else:
        count = torch.full_like(s["lengths"], n)
        padded = q.float()
    S = c["high"]
    k, there = _rows_of(s, 0, 0, S)
    v, _ = _rows_of(s, 1, 0, S)
    # the heads that share a K/V head are rows of one product
    rows = (padded * scale).view(B, n, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    score = rows @ k.permute(0, 2, 3, 1).contiguous()
    position = (s["lengths"] - count)[:, None] + torch.arange(n, device=DEVICE)
    seen = there[:, None, :] & (torch.arange(S, device=DEVICE) <= position[..., None])
    score = score.view(B, Hkv, Hq // Hkv, n, S).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = (weight.view(B, Hkv, -1, S) @ v.permute(0, 2, 1, 3).contiguous()).view(B, Hkv, Hq // Hkv, n, D) / total
    lse = (top + total.log()).view(B, Hq, n)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)
    if c["packed"]:
        return out[b, i].bfloat16(), lse[b, :, i].t().contiguous()
    return out.bfloat16(), lse


def exact(c, seed):
    """The same from the definitions, one sequence after the other, in 64 bits."""
    s = prepare(c, seed)
    lengths, new = _sizes(c)
    table = s["table"].cpu()
    cache = s["cache"]

    def held(half, b):                                   # (tokens, Hkv, D)
        got = []
        for at in table[b, :-(-lengths[b] // c["page"])].tolist():
            x = cache[half, at].double()
            got.append(x if s["scales"] is None else x * s["scales"][half, at].double()[..., None])
        return torch.cat(got)[:lengths[b]]

    if c["op"] == "read":
        out = torch.zeros(2, c["B"], c["rows"], c["Hkv"], c["D"], dtype=torch.float64, device=DEVICE)
        for b in range(c["B"]):
            for half in (0, 1):
                x = held(half, b)[c["begin"]:c["begin"] + c["rows"]]
                out[half, b, :x.shape[0]] = x
        return out
    first = [sum(new[:b]) for b in range(c["B"])]
    if c["op"] == "write":
        pages, scales = cache.double(), None if s["scales"] is None else s["scales"].double()
        for b in range(c["B"]):
            for half, x in enumerate((s["k"], s["v"])):
                x = (x[first[b]:first[b] + new[b]] if c["packed"] else x[b]).double()
                position = torch.arange(lengths[b] - new[b], lengths[b])
                at, slot = table[b][position // c["page"]].long().to(DEVICE), (position % c["page"]).to(DEVICE)
                if scales is not None:
                    powers = torch.tensor([2.0 ** e for e in range(-126, 121)], dtype=torch.float64, device=DEVICE)
                    top = x.abs().amax(-1)               # the least power with top <= 448 * power; rows of zeros have 1
                    scale = torch.where(top > 0, powers[torch.searchsorted(448 * powers, top)], 1.0)
                    y = x / scale[..., None]
                    power = powers[torch.searchsorted(powers, y.abs().clamp(min=2.0 ** -6), right=True) - 1]
                    step = power / 8                     # four bits of what lies between two powers, or of the least normal one
                    x = torch.round(y / step) * step     # to the even one of two
                    scales[half][at, slot] = scale
                pages[half][at, slot] = x
        return (pages,) if scales is None else (pages, scales)
    if sum(n * t for n, t in zip(new, lengths)) * c["Hq"] * c["D"] * 4 > 4e12:
        return None
    G = c["Hq"] // c["Hkv"]
    outs, lses = [], []
    for b in range(c["B"]):
        k, v = held(0, b), held(1, b)
        q = (s["q"][first[b]:first[b] + new[b]] if c["packed"] else s["q"][b]).double()
        hidden = torch.arange(lengths[b], device=DEVICE) > (lengths[b] - new[b] + torch.arange(new[b], device=DEVICE))[:, None]
        out, lse = torch.empty_like(q), torch.empty(c["Hq"], new[b], dtype=torch.float64, device=DEVICE)
        for h in range(c["Hq"]):
            score = (q[:, h] @ k[:, h // G].t().contiguous()) * c["D"] ** -0.5
            score[hidden] = -math.inf
            lse[h] = torch.logsumexp(score, -1)
            out[:, h] = torch.softmax(score, -1) @ v[:, h // G].contiguous()
        outs.append(out)
        lses.append(lse)
    return (torch.cat(outs), torch.cat(lses, 1)) if c["packed"] else (torch.stack(outs), torch.stack(lses))
