"""The operators over a paged cache where every wavefront and workgroup has many units, steps and items one after the other: rings that
are filled again and again, shares that begin and end inside a sequence, a head or an item.  Against the definitions in 64 bits, here on
the GPU, with bounds derived as in oracle/paged_oracle.py; what no key holds is NaN."""
import math

import pytest
import torch

import mercury_artifact_amd as M

pytestmark = pytest.mark.gpu

BF16, E4M3, E2M1 = torch.bfloat16, torch.float8_e4m3fn, torch.float4_e2m1fn_x2
TILE = 32            # keys that a wavefront of few-row attention takes at once


def _ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32).cuda()


def _starts(new):
    at = [0]
    for n in new:
        at.append(at[-1] + n)
    return at


def _spread(low, high, B, step=0.618034):
    return [high - int((high - low) * ((b * step) % 1.0)) for b in range(B)]


class Setting:
    """Sequences that the framework itself has written; `rows(b)` are those of sequence b as the cache holds them, in 64 bits.  Every value column is
    nothing but in one tile of 32 keys out of 64, and positive there: each tile is a twentieth of some column's result or more."""

    def __init__(self, kind, lengths, Hkv, D, page, seed, gone=0):
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.kind, self.lengths, self.page, self.Hkv, self.D = kind, lengths, page, Hkv, D
        counts = [-(-n // page) for n in lengths]
        pages = sum(counts) + 3
        order, at = torch.randperm(pages, generator=g, device="cuda").int(), 0
        table = torch.full((len(lengths), max(counts)), -1, dtype=torch.int32, device="cuda")
        for b, c in enumerate(counts):
            table[b, :c] = order[at:at + c]
            at += c
        self.cache, self.scales = M.paged_cache(pages, page, Hkv, D, kind)
        if kind == BF16:
            self.cache.fill_(math.nan)
        else:
            self.cache.view(torch.uint8).fill_(0x7f)
            self.scales.fill_(math.nan) if kind == E4M3 else self.scales.view(torch.uint8).fill_(255)
        self.dev_lengths = _ints(lengths)
        T = sum(lengths)
        position = torch.cat([torch.arange(n, device="cuda") for n in lengths])
        k = torch.randn(T, Hkv, D, generator=g, device="cuda").bfloat16()
        v = torch.rand(T, Hkv, D, generator=g, device="cuda") + 0.5
        v = torch.where((position // TILE % 64)[:, None, None] == torch.arange(D, device="cuda") % 64, v, 0.0).bfloat16()
        M.paged_cache_write(k, v, self.cache, table, self.dev_lengths, scales=self.scales, starts=_ints(_starts(lengths)))
        self.dense = M.paged_cache_read(self.cache, table, self.dev_lengths, max(lengths), scales=self.scales)
        if gone:                                         # pages that are not here, all over the sequences
            table = torch.where((torch.arange(table.shape[1], device="cuda") + torch.arange(len(lengths), device="cuda")[:, None]) % gone == 1,
                                torch.tensor(pages, dtype=torch.int32, device="cuda"), table)
        self.table, self.pages = table, pages
        self.weights = M.paged_weights(pages, page, Hkv)
        self.weights.copy_(torch.rand(self.weights.shape, generator=g, device="cuda") * 4)

    def rows(self, b):
        """Keys, values (Hkv, S, D), and which of the S rows are here."""
        n = self.lengths[b]
        x = self.dense[:, b, :n].transpose(1, 2).contiguous().double()
        pages = self.table[b, torch.arange(n, device="cuda") // self.page]
        return x[0], x[1], (pages >= 0) & (pages < self.pages)

    def places(self, b):
        position = torch.arange(self.lengths[b], device="cuda")
        return self.table[b, position // self.page].long(), position % self.page

    def queries(self, T, Hq):
        return torch.randn(T, Hq, self.D, generator=self.g, device="cuda").bfloat16()


def _scores(s, b, q, new, causal, scale, h):
    """Of sequence b's rows (new tokens times heads of K/V head h) and keys: the score (-inf where a key is not seen), and how far one summed in fp32 is off."""
    k, _, here = s.rows(b)
    n, Hq, D = q.shape
    G, S = Hq // s.Hkv, k.shape[1]
    x = q[:, h * G:(h + 1) * G].reshape(n * G, D).double()
    kt = k[h].t().contiguous()
    score = (x @ kt) * scale
    size = (x.abs() @ kt.abs()) * scale * ((D + 4) * 2.0 ** -24)
    seen = here[None, :].expand(n, S)
    if causal:
        seen = seen & (torch.arange(S, device="cuda") <= (S - n + torch.arange(n, device="cuda"))[:, None])
    return score.masked_fill_(~seen.repeat_interleave(G, 0), -math.inf), size


def _heads(s, Hq):
    return range(s.Hkv), Hq // s.Hkv


def _lse(s, q, new, causal, scale):
    """(Hq, T) in float32, of packed tokens."""
    at, (heads, G) = _starts(new), _heads(s, q.shape[1])
    lse = torch.empty(q.shape[1], at[-1], device="cuda")
    for b, n in enumerate(new):
        for h in heads if n else ():
            score, _ = _scores(s, b, q[at[b]:at[b + 1]], new, causal, scale, h)
            lse[h * G:(h + 1) * G, at[b]:at[b + 1]] = torch.logsumexp(score, 1).view(n, G).t()
    return lse


def _check_weights(s, q, lse, new, got, before, causal, scale, decay, chain):
    """`chain`: how many terms a kernel adds up one after the other, of the up to new * G of a key."""
    at, (heads, G) = _starts(new), _heads(s, q.shape[1])
    untouched = torch.ones(before.shape, dtype=torch.bool, device="cuda")
    for b, n in enumerate(new):
        page, slot = s.places(b)
        here = (page >= 0) & (page < s.pages)
        old = torch.where(here[:, None], before[page * here, slot], 0.0).double()
        for h in heads:
            want, off = old[:, h].clone(), torch.zeros_like(old[:, h])
            if n:
                score, size = _scores(s, b, q[at[b]:at[b + 1]], new, causal, scale, h)
                l = lse[h * G:(h + 1) * G, at[b]:at[b + 1]].t().reshape(-1, 1).double()
                weight = torch.exp(score - l)
                total = weight.sum(0)
                off = (weight * (size + 2.0 ** -22 * (score.masked_fill(weight == 0, 0.0).abs() + l.abs()) + 2.0 ** -21)).sum(0) + total * chain * 2.0 ** -23
                want = total + torch.where(torch.arange(len(total), device="cuda") < len(total) - n, decay * want, 0.0)
            off += 2.0 ** -23 * want.abs()
            mine = got[page * here, slot, h].double()
            wrong = here & ~((mine - want).abs() <= off)
            assert not wrong.any(), (b, h, wrong.nonzero().flatten()[:8].tolist(), ((mine - want).abs() - off)[here].max().item())
        untouched[page[here], slot[here]] = False
    assert (got[untouched] == 7).all()


def _weigh(s, q, lse, new, packed, causal, scale, decay=1.0):
    out = torch.full_like(s.weights, 7.0)
    starts = _ints(_starts(new)) if packed else None
    if not packed:
        q, lse = q.view(len(new), new[0], *q.shape[1:]), lse.view(lse.shape[0], len(new), new[0]).transpose(0, 1).contiguous()
    M.paged_attn_weights(q, s.cache, s.table, s.dev_lengths, scale, lse, s.weights, causal=causal, scales=s.scales, starts=starts,
                         most_new=max(new), decay=decay, out=out)
    return out


# A register of paged_weights_many takes 64 tiles' weights of a key, its 32 lanes are added as a tree, and each 64 steps of an item and each
# workgroup that shares it (few here) once more: 128 terms in a row at most.
@pytest.mark.parametrize("kind,D,Hq,Hkv,gone", [
    (BF16, 128, 32, 8, 0), (E4M3, 128, 32, 8, 0), (E2M1, 128, 32, 8, 0), (BF16, 64, 32, 8, 7), (E4M3, 96, 16, 8, 0), (E2M1, 64, 32, 4, 5), (E2M1, 96, 8, 8, 0),
])
def test_weights_of_a_prompt_with_hundreds_of_steps_to_a_workgroup(kind, D, Hq, Hkv, gone):
    print(f"case {kind} D{D} H{Hq}/{Hkv} gone {gone}", flush=True)
    s = Setting(kind, [8150], Hkv, D, 16, seed=D, gone=gone)
    q = s.queries(8150, Hq)
    lse = _lse(s, q, [8150], True, D ** -0.5)
    got = _weigh(s, q, lse, [8150], True, True, D ** -0.5)
    _check_weights(s, q, lse, [8150], got, s.weights, True, D ** -0.5, 1.0, 128)


@pytest.mark.parametrize("kind,lengths,new,Hq,Hkv,D,causal,decay", [
    (BF16, _spread(300, 900, 64), _spread(150, 290, 64, 0.414214), 16, 8, 128, True, 0.5),      # several whole items each, of 10 to 18 steps
    (E4M3, _spread(300, 900, 64), _spread(150, 290, 64, 0.414214), 16, 8, 64, False, 1.0),
    (E2M1, _spread(900, 1500, 100), _spread(12, 30, 100, 0.414214), 32, 4, 96, True, 1.0),      # tiles of several heads, of 3 to 5 steps
    (E2M1, _spread(2000, 5000, 24), [900 if b % 3 else 1 for b in range(24)], 12, 4, 128, True, 0.0),
    (BF16, [6000, 6000, 6000], [700, 700, 700], 14, 2, 64, False, 1.0),
    (E4M3, _spread(2000, 5000, 24), [900 if b % 3 else 1 for b in range(24)], 12, 4, 128, True, 0.5),            # divided among both kernels
    (E4M3, _spread(300, 9000, 150), [200 if b % 4 == 0 else b % 6 for b in range(150)], 32, 4, 96, True, 1.0),
    (E4M3, _spread(300, 9000, 100), [70 if b % 9 == 0 else b % 3 for b in range(100)], 48, 2, 64, False, 0.0),
])
def test_weights_of_many_items_to_a_workgroup(kind, lengths, new, Hq, Hkv, D, causal, decay):
    print(f"case {kind} H{Hq}/{Hkv} D{D} causal {causal}", flush=True)
    s = Setting(kind, lengths, Hkv, D, 32, seed=Hq, gone=9 if causal else 0)
    q = s.queries(sum(new), Hq)
    lse = _lse(s, q, new, causal, D ** -0.5)
    got = _weigh(s, q, lse, new, len(set(new)) > 1, causal, D ** -0.5, decay)
    _check_weights(s, q, lse, new, got, s.weights, causal, D ** -0.5, decay, 128)


LONG = [
    ([40000, 39871, 40000, 38111], 1, 32, 8, 128, 64, 0),
    (_spread(300, 16384, 32), 1, 32, 8, 128, 16, 7),
    (_spread(300, 16384, 32), 5, 32, 8, 128, 16, 0),             # 20 rows
    (_spread(300, 9000, 32), 12, 16, 4, 128, 48, 11),            # 48 rows
    (_spread(300, 16384, 32), 3, 32, 8, 64, 16, 5),
    (_spread(300, 16384, 32), 8, 24, 8, 64, 32, 0),              # 24 rows
    (_spread(300, 9000, 32), 15, 16, 4, 64, 16, 7),              # 60 rows
]


@pytest.mark.parametrize("kind", [BF16, E4M3, E2M1], ids=["bf16", "e4m3", "e2m1"])
@pytest.mark.parametrize("lengths,n,Hq,Hkv,D,page,gone", LONG)
def test_weights_of_few_rows_with_many_units_to_a_wavefront(lengths, n, Hq, Hkv, D, page, gone, kind):
    print(f"case {kind} {len(lengths)} sequences, {n} tokens H{Hq}/{Hkv} D{D} gone {gone}", flush=True)
    s = Setting(kind, lengths, Hkv, D, page, seed=n, gone=gone)
    new = [n] * len(lengths)
    q = s.queries(sum(new), Hq)
    lse = _lse(s, q, new, True, D ** -0.5)
    got = _weigh(s, q, lse, new, False, True, D ** -0.5)
    _check_weights(s, q, lse, new, got, s.weights, True, D ** -0.5, 1.0, n * Hq // Hkv)


@pytest.mark.parametrize("kind", [BF16, E4M3, E2M1], ids=["bf16", "e4m3", "e2m1"])
@pytest.mark.parametrize("lengths,n,Hq,Hkv,D,page,gone", LONG)
def test_attention_of_few_rows_with_many_tiles_to_a_wavefront(lengths, n, Hq, Hkv, D, page, gone, kind):
    """A lane adds up eight weights of each tile of its wavefront, which has every second tile of its share at most: S / 8 terms in a row."""
    print(f"case {kind} {len(lengths)} sequences, {n} tokens H{Hq}/{Hkv} D{D} gone {gone}", flush=True)
    s = Setting(kind, lengths, Hkv, D, page, seed=n, gone=gone)
    B, G = len(lengths), Hq // Hkv
    q = s.queries(B * n, Hq).view(B, n, Hq, D)
    out, lse = M.paged_attn_fwd(q, s.cache, s.table, s.dev_lengths, D ** -0.5, scales=s.scales)
    for b in range(B):
        _, v, _ = s.rows(b)
        for h in range(Hkv):
            score, size = _scores(s, b, q[b], None, True, D ** -0.5, h)
            want_lse = torch.logsumexp(score, 1)
            weight = torch.exp(score - want_lse[:, None])
            want = weight @ v[h]                         # (no value is negative)
            delta, sums = size.max(1).values, (lengths[b] / 8 + 64) * 2.0 ** -23
            got = out[b, :, h * G:(h + 1) * G].reshape(n * G, D).double()
            got_lse = lse[b, h * G:(h + 1) * G].t().reshape(-1).double()
            assert ((got_lse - want_lse).abs() <= delta + sums + want_lse.abs() * 2.0 ** -22).all(), (b, h)
            off = want * ((2.0 ** -8 + 2 * delta + sums)[:, None] * (1 + 2.0 ** -8) + 2.0 ** -8)
            assert ((got - want).abs() <= off).all(), (b, h, ((got - want).abs() - off).max().item())
