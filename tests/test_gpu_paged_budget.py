"""A paged cache within a budget: what attention its keys have had, and the eviction of those that had least, against the 64-bit
restatement (oracle/paged_oracle.py, whose docstrings derive how far sums may be off).  What no key holds is NaN here."""
import math

import pytest
import torch

import mercury_artifact_amd as M
from mercury_artifact_amd import _native as N
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

E4M3, E2M1, E8M0 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
KINDS = [torch.bfloat16, E4M3, E2M1]
NAMES = ["bf16", "e4m3", "e2m1"]


def _ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32).cuda()


def _raw(t):
    """Bytes of a tensor, whatever it holds."""
    return (t.view(torch.uint8).flatten() if t.element_size() == 1 else t.flatten().clone().view(torch.uint8)).cpu()


class Setting:
    """Sequences in a cache of any kind, written by the framework itself; `values` is what the cache stands for, in 64 bits."""

    def __init__(self, kind, lengths, Hkv, D, page=16, seed=0, spare=2, width=None, token_major=False):
        g = self.g = torch.Generator().manual_seed(seed)
        self.kind, self.lengths, self.page = kind, list(lengths), page
        counts = [-(-n // page) for n in lengths]
        pages = sum(counts) + spare
        order, at = torch.randperm(pages, generator=g).tolist(), 0
        width = max([*counts, 1]) if width is None else width
        self.table = []
        for c in counts:
            self.table.append(order[at:at + c] + [-1] * (width - c))
            at += c
        self.free = order[at:]
        self.dev, self.scales = M.paged_cache(pages, page, Hkv, D, kind)
        self.weights = M.paged_weights(pages, page, Hkv)
        if token_major:
            self.dev, self.weights = self.dev.contiguous(), self.weights.contiguous()
            self.scales = None if self.scales is None else self.scales.contiguous()
        if kind == torch.bfloat16:
            self.dev.fill_(math.nan)
        else:
            self.dev.view(torch.uint8).fill_(0x7f)
            if kind == E4M3:
                self.scales.fill_(math.nan)
            else:
                self.scales.view(torch.uint8).fill_(255)
        self.weights.copy_((torch.rand(pages, page, Hkv, generator=g) * 4).cuda())
        most = max([*lengths, 1])
        kv = torch.randn(2, sum(lengths), Hkv, D, generator=g).bfloat16().cuda()
        starts = [sum(lengths[:b]) for b in range(len(lengths) + 1)]
        M.paged_cache_write(kv[0], kv[1], self.dev, *self.tables(), scales=self.scales, starts=_ints(starts))
        dense = M.paged_cache_read(self.dev, *self.tables(), most, scales=self.scales).cpu().double()
        self.values = torch.zeros(2, pages, page, Hkv, D, dtype=torch.float64)
        for b, n in enumerate(lengths):
            for j in range(n):
                self.values[:, self.table[b][j // page], j % page] = dense[:, b, j]

    def tables(self):
        return _ints(self.table).view(len(self.lengths), -1), _ints(self.lengths)


def _weigh(s, q, lse, scale, causal=True, starts=None, **kw):
    got = M.paged_attn_weights(q.cuda(), s.dev, *s.tables(), scale, lse.cuda(), s.weights, causal=causal, scales=s.scales, starts=_ints(starts), **kw)
    torch.cuda.synchronize()
    return got.cpu()


def _lse(s, q, scale, causal=True, starts=None):
    """In float32, from the restatement."""
    got = [l for _, l, _, _ in P.paged_attention(q, s.values, s.table, s.lengths, scale, causal, None, starts)]
    return (torch.stack(got) if starts is None else torch.cat(got, 1)).float()


def _check(got, s, q, lse, scale, before, causal=True, starts=None, decay=1.0):
    want, off = P.paged_weights(q, s.values, s.table, s.lengths, scale, lse, before, causal, starts, decay)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    assert ((got.double() - want).abs() <= off)[torch.isfinite(want)].all(), ((got.double() - want).abs() - off).max()


@pytest.mark.parametrize("kind", KINDS, ids=NAMES)
@pytest.mark.parametrize("lengths,new,Hq,Hkv,D,page,causal", [
    ([1], 1, 1, 1, 128, 16, True),
    ([0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65], 1, 4, 2, 128, 16, True),
    ([127, 128, 129, 300, 1, 0], 1, 8, 2, 64, 16, True),
    ([500, 3], 1, 5, 5, 96, 32, True),
    ([257, 64, 1], 1, 32, 2, 128, 48, False),
    ([200], 1, 7, 1, 32, 64, True),
    ([40, 5, 129], 5, 4, 2, 128, 16, True),
    ([40, 5, 129], 5, 4, 2, 64, 16, False),
    ([90, 33], 4, 16, 2, 64, 16, True),              # 32 rows
    ([90, 33], 4, 17, 1, 32, 16, True),              # 68 rows
    ([2, 3, 50], 6, 2, 2, 128, 16, True),            # more new tokens than keys
    ([150, 130], 130, 2, 2, 128, 16, True),
    ([320], 77, 6, 2, 32, 256, True),
    ([100, 180], 90, 4, 1, 96, 32, False),
    ([700], 300, 2, 1, 64, 16, True),
])
def test_weights(lengths, new, Hq, Hkv, D, page, causal, kind):
    print(f"case {lengths} new {new} H{Hq}/{Hkv} D{D} page {page} causal {causal} {kind}", flush=True)
    s = Setting(kind, lengths, Hkv, D, page, seed=len(lengths) + new)
    q = torch.randn(len(lengths), new, Hq, D, generator=s.g).bfloat16()
    lse, before = _lse(s, q, D ** -0.5, causal), s.weights.cpu()
    _check(_weigh(s, q, lse, D ** -0.5, causal), s, q, lse, D ** -0.5, before, causal)


@pytest.mark.parametrize("D", [8, 24, 40, 72, 88, 104, 120])
def test_weights_of_other_head_dimensions(D):
    s = Setting(torch.bfloat16, [70, 200], 2, D, seed=D)
    for new in (3, 70):
        q = torch.randn(2, new, 4, D, generator=s.g).bfloat16()
        lse, before = _lse(s, q, D ** -0.5), s.weights.cpu()
        _check(_weigh(s, q, lse, D ** -0.5), s, q, lse, D ** -0.5, before)


@pytest.mark.parametrize("kind", KINDS, ids=NAMES)
@pytest.mark.parametrize("most", [None, 1, 40, 1000])
def test_weights_packed(kind, most):
    """Sequences of any number of new tokens, none among them, which keep what they had; rows outside of all take no part; decay."""
    lengths, new = [40, 150, 17, 9, 0, 64], [1, 0, 3, 9, 0, 40]
    s = Setting(kind, lengths, 2, 64, seed=5, width=40)
    starts = [2 + sum(new[:b]) for b in range(7)]
    q = torch.randn(starts[-1] + 3, 4, 64, generator=s.g).bfloat16()
    lse = torch.full((4, starts[-1] + 3), math.nan)
    lse[:, 2:starts[-1]] = _lse(s, q, 0.125, starts=starts)
    q[:2], q[starts[-1]:] = math.nan, math.nan
    for decay in (1.0, 0.25, 0.0):
        before = s.weights.cpu()
        out = torch.full_like(s.weights, 7.0)
        got = _weigh(s, q, lse, 0.125, starts=starts, most_new=most, decay=decay, out=out)
        assert torch.equal(s.weights.cpu(), before)
        held = torch.zeros(before.shape, dtype=torch.bool)
        for b, n in enumerate(lengths):
            for j in range(n):
                held[s.table[b][j // 16], j % 16] = True
        assert (got[~held] == 7).all()
        _check(torch.where(held, got, before), s, q, lse, 0.125, before, starts=starts, decay=decay)
        again = _weigh(s, q, lse, 0.125, starts=starts, most_new=most, decay=decay)                 # in place
        assert again.data_ptr() != got.data_ptr() and torch.equal(again[held], got[held]) and torch.equal(again[~held], before[~held])


@pytest.mark.parametrize("new", [1, 100])
def test_weights_that_nothing_holds_are_not_read(new):
    """NaN in the weights of new tokens and, with decay 0, of all keys; pages that are not here; rows that see no key."""
    s = Setting(torch.bfloat16, [210, 5, 130], 2, 64, seed=11)
    q = torch.randn(3, new, 4, 64, generator=s.g).bfloat16()
    whole = s.table
    for decay in (1.0, 0.0):
        for nobody in (-1, s.values.shape[1], 2 ** 31 - 1, -2 ** 31):
            s.table = [[nobody if i % 3 == 1 else e for i, e in enumerate(row)] for row in whole]
            lse = _lse(s, q, 0.125)
            s.weights.copy_(torch.rand(s.weights.shape, generator=s.g))
            for b, n in enumerate(s.lengths):
                for j in range(0 if decay == 0 else max(n - new, 0), n):
                    s.weights[whole[b][j // 16], j % 16] = math.nan
            before = s.weights.cpu()
            got = _weigh(s, q, lse, 0.125, decay=decay)
            _check(got, s, q, lse, 0.125, before, decay=decay)


@pytest.mark.parametrize("new", [1, 20, 100])
def test_a_key_that_is_no_number_has_its_own_weight_alone(new):
    """And an infinite key whose score is -inf in every row has none."""
    s = Setting(torch.bfloat16, [230], 1, 64, seed=3)
    q = torch.randn(1, new, 2, 64, generator=s.g).abs().bfloat16()
    lse = _lse(s, q, 0.1)
    for at, what in ((5, math.nan), (77, -math.inf), (229, math.nan)):
        s.dev[0, s.table[0][at // 16], at % 16, 0, 9] = what
    before = s.weights.cpu()
    got = _weigh(s, q, lse, 0.1, decay=0.0)
    want, off = P.paged_weights(q, s.values, s.table, s.lengths, 0.1, lse, before, True, None, 0.0)
    flat = torch.stack([got[s.table[0][j // 16], j % 16, 0] for j in range(230)])
    assert torch.isnan(flat[[5, 229]]).all() and flat[77] == 0
    for j in range(230):
        if j not in (5, 77, 229):
            at = s.table[0][j // 16], j % 16, 0
            assert abs(got[at].double() - want[at]) <= off[at]


@pytest.mark.parametrize("kind", KINDS, ids=NAMES)
def test_weights_strides_and_many_sequences(kind):
    lengths = [(37 * b) % 61 for b in range(150)]
    lengths[77] = 900
    s = Setting(kind, lengths, 2, 64, seed=9, token_major=True)
    q = torch.randn(150, 1, 4, 64, generator=s.g).bfloat16()
    lse, before = _lse(s, q, 0.125), s.weights.cpu()
    big = torch.full((150, 1, 8, 128), math.nan, dtype=torch.bfloat16).cuda()
    big[:, :, 2:6, 64:] = q.cuda()
    wide = torch.full((before.shape[0], 17, 5), 3.0).cuda()
    out = wide[:, 1:, 1:3]
    M.paged_attn_weights(big[:, :, 2:6, 64:], s.dev, *s.tables(), 0.125, lse.cuda(), s.weights, scales=s.scales, out=out)
    got = out.cpu()
    held = got != 3
    _check(torch.where(held, got, before), s, q, lse, 0.125, before)
    out.fill_(3.0)
    assert (wide == 3).all()


def test_weights_of_many_query_heads_and_thousands_of_sequences():
    for Hq in (65, 128):
        s = Setting(E4M3, [200, 1, 77], 1, 64, seed=Hq)
        q = torch.randn(3, 1, Hq, 64, generator=s.g).bfloat16()
        lse, before = _lse(s, q, 0.125), s.weights.cpu()
        _check(_weigh(s, q, lse, 0.125), s, q, lse, 0.125, before)
    s = Setting(torch.bfloat16, [(7 * b) % 25 for b in range(2500)], 1, 16, seed=1)
    q = torch.randn(2500, 1, 1, 16, generator=s.g).bfloat16()
    lse, before = _lse(s, q, 0.25), s.weights.cpu()
    _check(_weigh(s, q, lse, 0.25), s, q, lse, 0.25, before)


def test_weights_of_lengths_and_starts_outside_the_tensors():
    s = Setting(torch.bfloat16, [64, 64, 64], 1, 64, seed=2)
    table, _ = s.tables()
    q = torch.randn(9, 2, 64, generator=s.g).bfloat16()
    s.lengths, starts = [64, 0, 64], [0, 3, 3, 9]
    lse = _lse(s, q, 0.1, causal=False, starts=starts)
    odd, odd_starts = _ints([2 ** 31 - 1, -5, 65]), _ints([-7, 3, 3, 2 ** 31 - 1])
    before = s.weights.cpu()
    got = M.paged_attn_weights(q.cuda(), s.dev, table, odd, 0.1, lse.cuda(), s.weights, causal=False, starts=odd_starts, decay=0.5).cpu()
    _check(got, s, q, lse, 0.1, before, causal=False, starts=starts, decay=0.5)
    before = s.weights.cpu()
    M.paged_attn_weights(q.cuda(), s.dev, table, odd, 0.1, lse.cuda(), s.weights, starts=_ints([8, 2, 2, 0]))
    assert torch.equal(s.weights.cpu(), before)


def test_weights_are_the_same_in_every_call():
    for new in (1, 120):
        s = Setting(torch.bfloat16, [900, 131, 450], 2, 128, seed=13)
        q = torch.randn(3, new, 8, 128, generator=s.g).bfloat16().cuda()
        out, lse = M.paged_attn_fwd(q, s.dev, *s.tables(), 0.1)
        calls = [M.paged_attn_weights(q, s.dev, *s.tables(), 0.1, lse, s.weights, out=torch.zeros_like(s.weights)).cpu() for _ in range(4)]
        assert all(torch.equal(x, calls[0]) for x in calls)
        # every row's weights add up to one (the sums of 8 heads' rows, each off by the roundings of its lse and of 900 weights)
        total = M.paged_attn_weights(q, s.dev, *s.tables(), 0.1, lse, s.weights, decay=0.0, out=torch.zeros_like(s.weights)).double().sum().item()
        assert abs(total - 3 * new * 8) <= 3 * new * 8 * 1e-4


@pytest.mark.parametrize("new", [1, 20, 100])
def test_a_row_whose_lse_is_no_number_counts_for_the_keys_that_it_sees(new):
    """Queries that are no numbers, and weights past the largest: the keys behind the row's token have nothing of them."""
    s = Setting(torch.bfloat16, [230, 90], 2, 64, seed=4)
    q = torch.randn(2, new, 4, 64, generator=s.g).bfloat16()
    lse = _lse(s, q, 0.1)
    for b, h, i, what in ((0, 1, 0, math.nan), (1, 2, new // 2, -2.0 ** 127), (1, 0, max(new - 11, 0), math.nan)):
        lse[b, h, i] = what
        if math.isnan(what):
            q[b, i, h] = what
    before = s.weights.cpu()
    got = _weigh(s, q, lse, 0.1)
    _check(got, s, q, lse, 0.1, before)
    assert new == 1 or torch.isfinite(got[s.table[0][-1]]).all()


@pytest.mark.parametrize("kind", KINDS, ids=NAMES)
@pytest.mark.parametrize("lengths,new,G,D,causal", [
    ([300, 41], 41, 3, 64, True),
    ([300, 41], 41, 6, 128, True),
    ([290, 530], 12, 6, 96, False),
    ([290, 9], 9, 16, 64, True),
    ([260, 517], 2, 64, 128, True),
    ([70, 31], 31, 64, 64, False),
    ([5, 257], 33, 32, 32, True),                    # more new tokens than keys
    ([513], 129, 2, 64, True),
])
@pytest.mark.parametrize("by_heads", [False, True], ids=["by_tokens", "by_heads"])
def test_weights_of_chunks_of_grouped_heads(lengths, new, G, D, causal, by_heads, kind):
    """A tile of rows is of several tokens and heads, whichever of them lies farther apart."""
    print(f"case {lengths} new {new} G{G} D{D} causal {causal} {kind} by heads {by_heads}", flush=True)
    s = Setting(kind, lengths, 2, D, seed=G + new)
    q = torch.randn(len(lengths), new, 2 * G, D, generator=s.g).bfloat16()
    lse, before = _lse(s, q, D ** -0.5, causal), s.weights.cpu()
    laid = q.cuda().transpose(1, 2).contiguous().transpose(1, 2) if by_heads else q.cuda()
    _check(_weigh(s, laid, lse, D ** -0.5, causal), s, q, lse, D ** -0.5, before, causal)


@pytest.mark.parametrize("new,Hq", [(70, 2), (5, 32)])
@pytest.mark.parametrize("far", [(1 << 23) + 8, (1 << 20) + 8])
def test_weights_of_queries_that_lie_far_apart(new, Hq, far):
    """Tokens, then heads, whose distances pass what a descriptor spans."""
    s = Setting(torch.bfloat16, [200], 1, 64, seed=new)
    q = torch.randn(1, new, Hq, 64, generator=s.g).bfloat16()
    lse, before = _lse(s, q, 0.125), s.weights.cpu()
    for steps in ((far, 64), (64, far)):
        laid = torch.empty((new if steps[0] == far else Hq) * far, dtype=torch.bfloat16, device="cuda")
        laid = laid.as_strided((1, new, Hq, 64), (far, *steps, 1)).copy_(q)
        out = torch.zeros_like(s.weights)
        M.paged_attn_weights(laid, s.dev, *s.tables(), 0.125, lse.cuda(), s.weights, out=out)
        held = torch.zeros(before.shape, dtype=torch.bool)
        for j in range(200):
            held[s.table[0][j // 16], j % 16] = True
        _check(torch.where(held, out.cpu(), before), s, q, lse, 0.125, before)


@pytest.mark.parametrize("new", [3, 90])
def test_weights_of_e4m3_keys_whose_scales_are_any_numbers(new):
    """Long chunks take scale times code rounded to bf16, off by up to 2^-8 of each product, and a weight by as much of their sum."""
    s = Setting(E4M3, [190], 2, 64, seed=new)
    times = torch.rand(s.scales.shape, generator=s.g) * 0.9 + 0.55
    s.scales.mul_(times.cuda())
    dense = M.paged_cache_read(s.dev.view(torch.uint8).clone().view(E4M3), *s.tables(), 190, scales=torch.ones_like(s.scales)).cpu().double()
    scales = s.scales.cpu().double()
    for j in range(190):
        at = s.table[0][j // 16], j % 16
        s.values[:, at[0], at[1]] = dense[:, 0, j] * scales[:, at[0], at[1]].view(2, 2, 1)
    q = torch.randn(1, new, 4, 64, generator=s.g).bfloat16()
    lse, before = _lse(s, q, 0.125), s.weights.cpu()
    got = _weigh(s, q, lse, 0.125, decay=0.0)
    want, off = P.paged_weights(q, s.values, s.table, s.lengths, 0.125, lse, before, True, None, 0.0)
    x = torch.stack([s.values[0, s.table[0][j // 16], j % 16] for j in range(190)])                  # (190, 2, 64)
    for h in range(4):
        for i in range(new):
            sees = 190 - new + i + 1
            score, size = x[:sees, h // 2] @ q[0, i, h].double() * 0.125, x[:sees, h // 2].abs() @ q[0, i, h].double().abs() * 0.125
            more = torch.exp(score - lse[0, h, i].double()) * (torch.exp(size * 2.0 ** -8) - 1)
            for j in range(sees):
                off[s.table[0][j // 16], j % 16, h // 2] += more[j]
    assert ((got.double() - want).abs() <= off).all()


@pytest.mark.parametrize("lengths,new,Hq,Hkv", [([1500], [1500], 2, 1), ([1300, 290, 40], [900, 33, 40], 4, 2), ([2050], [130], 8, 1)])
def test_weights_of_prompts_that_many_workgroups_share(lengths, new, Hq, Hkv):
    s = Setting(torch.bfloat16, lengths, Hkv, 64, seed=Hq)
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    q = torch.randn(starts[-1], Hq, 64, generator=s.g).bfloat16()
    lse, before = _lse(s, q, 0.125, starts=starts), s.weights.cpu()
    _check(_weigh(s, q, lse, 0.125, starts=starts), s, q, lse, 0.125, before, starts=starts)


# ---- eviction ------------------------------------------------------------------------------------------------------------------

def _rows(s, table, kept):
    """Bytes of rows, scales and weights at positions kept (of one K/V head h) in the pages of a table row."""
    at = lambda j: (table[j // s.page], j % s.page)                               # noqa: E731
    return [at(j) for j in kept]


def _check_evicted(s, keep, recent=0, limit=None, out=False, spare_width=None):
    limit_ = keep if limit is None else limit
    before, before_scales, before_weights = (None if t is None else t.clone() for t in (s.dev, s.scales, s.weights))
    want, left = P.evicted(s.weights.cpu(), s.table, s.lengths, s.dev.shape[1], keep, recent, limit_)
    out_table = None
    if out:
        width = -(-limit_ // s.page) if spare_width is None else spare_width
        out_table = [s.free[b * width:(b + 1) * width] for b in range(len(s.lengths))]
        assert all(len(row) == width for row in out_table)
    table, lengths = s.tables()
    kept, got_left = M.paged_cache_evict(s.dev, table, lengths, s.weights, keep, recent=recent, limit=limit, scales=s.scales,
                                         out_table=None if out_table is None else _ints(out_table).view(len(s.lengths), -1))
    torch.cuda.synchronize()
    assert kept.shape == (len(s.lengths), s.dev.shape[3], limit_) and kept.dtype == torch.int32
    assert got_left.tolist() == left and torch.equal(lengths.cpu(), torch.tensor(s.lengths, dtype=torch.int32).cpu())
    expect = [None if x is None else x.clone() for x in (before, before_scales, before_weights)]
    for b, per_head in enumerate(want):
        for h in range(s.dev.shape[3]):
            stay = [] if per_head is None or (not out and per_head is not None and len(per_head[h]) > limit_) else per_head[h]
            assert kept[b, h].tolist() == stay + [-1] * (limit_ - len(stay)), (b, h)
            if not stay:
                continue
            old = torch.tensor(stay)
            new = torch.arange(len(stay))
            from_, to = torch.tensor(s.table[b])[old // s.page].cuda(), torch.tensor((out_table or s.table)[b])[new // s.page].cuda()
            from_slot, to_slot = (old % s.page).cuda(), (new % s.page).cuda()
            for t, x in zip(expect, (before, before_scales, before_weights)):
                if t is None:
                    continue
                if t.dim() == 3:
                    t[to, to_slot, h] = x[from_, from_slot, h]
                elif t.dtype in (E2M1, E8M0, E4M3):
                    t.view(torch.uint8)[:, to, to_slot, h] = x.view(torch.uint8)[:, from_, from_slot, h]
                else:
                    t[:, to, to_slot, h] = x[:, from_, from_slot, h]
    for t, x in zip((s.dev, s.scales, s.weights), expect):
        assert t is None or torch.equal(_raw(t), _raw(x))
    return kept, got_left


@pytest.mark.parametrize("kind", KINDS, ids=NAMES)
@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("lengths,Hkv,D,page,keep,recent,limit", [
    ([1], 1, 128, 16, 0, 0, 0),
    ([5], 2, 64, 16, 1, 0, 1),
    ([40, 5, 33, 0, 32, 31], 2, 128, 16, 32, 8, 32),
    ([40, 5, 33, 0, 47, 31], 2, 64, 16, 16, 16, 32),         # the last ones alone
    ([300, 257, 1100], 3, 96, 48, 256, 0, 256),
    ([2100, 700], 1, 128, 64, 513, 100, 600),
    ([1500, 1501, 90], 2, 32, 16, 1499, 7, 1499),           # nearly all stay: every row moves a little
    ([90], 5, 128, 256, 3, 1, 70),
])
def test_evict(lengths, Hkv, D, page, keep, recent, limit, out, kind):
    print(f"case {lengths} Hkv {Hkv} D{D} page {page} keep {keep} recent {recent} limit {limit} out {out} {kind}", flush=True)
    spare = 2 + (-(-limit // page) * len(lengths) if out else 0)
    s = Setting(kind, lengths, Hkv, D, page, seed=len(lengths) + keep, spare=spare)
    _check_evicted(s, keep, recent, limit, out)


@pytest.mark.parametrize("pattern", ["equal", "zeros", "nan", "negative", "infinite", "rising", "falling", "least"])
def test_which_weights_count_as_largest(pattern):
    """Ties go to the first; NaN of either sign above all, then infinity; -0 is 0; differences in the last bit count."""
    n = 2300
    s = Setting(torch.bfloat16, [n, 100], 2, 64, seed=7)
    w = s.weights
    g = torch.Generator().manual_seed(1)
    if pattern == "equal":
        w.fill_(0.5)
    elif pattern == "zeros":
        w.copy_(torch.where(torch.rand(w.shape, generator=g) < 0.5, -0.0, 0.0))
    elif pattern == "nan":
        w[torch.rand(w.shape, generator=g).cuda() < 0.1] = math.nan
        w[torch.rand(w.shape, generator=g).cuda() < 0.1] = -math.nan
    elif pattern == "negative":
        w.sub_(2.0)
    elif pattern == "infinite":
        w[torch.rand(w.shape, generator=g).cuda() < 0.1] = math.inf
        w[torch.rand(w.shape, generator=g).cuda() < 0.3] = -math.inf
    elif pattern == "least":
        w.copy_(1.0 + torch.randint(0, 3, w.shape, generator=g) * 2.0 ** -23)
    else:
        for j in range(n):
            w[s.table[0][j // 16], j % 16] = float(j if pattern == "rising" else n - j)
    for keep, recent in ((1000, 0), (1500, 300)):
        t = Setting(torch.bfloat16, [n, 100], 2, 64, seed=7)
        t.weights.copy_(w)
        _check_evicted(t, keep, recent)


@pytest.mark.parametrize("out", [False, True])
def test_a_sequence_with_a_page_that_is_not_here_stays_as_it_is(out):
    s = Setting(E4M3, [100, 100, 100, 30], 2, 64, seed=4, spare=20)
    s.table[0][3], s.table[1][0], s.table[3][1] = -1, s.dev.shape[1], 2 ** 31 - 1
    s.table = [row + [-1, -7] for row in s.table]           # (past the end: nobody looks)
    kept, left = _check_evicted(s, 40, 4, 50, out)
    assert left.tolist() == [100, 100, 40, 30] and (kept[[0, 1, 3]] == -1).all()


def test_rows_of_out_pages_that_are_not_here_are_dropped():
    s = Setting(torch.bfloat16, [70], 1, 64, seed=4, spare=6)
    out_table = [[s.free[0], -1, s.free[1]]]
    before, weights = s.dev.clone(), s.weights.clone()
    kept, left = M.paged_cache_evict(s.dev, *s.tables(), s.weights, 40, out_table=_ints(out_table))
    assert left.item() == 40
    for i, j in enumerate(kept[0, 0].tolist()):
        if out_table[0][i // 16] >= 0:
            assert torch.equal(s.dev[:, out_table[0][i // 16], i % 16], before[:, s.table[0][j // 16], j % 16])
            before[:, out_table[0][i // 16], i % 16] = s.dev[:, out_table[0][i // 16], i % 16]
            weights[out_table[0][i // 16], i % 16] = s.weights[out_table[0][i // 16], i % 16]
    assert torch.equal(_raw(s.dev), _raw(before)) and torch.equal(s.weights, weights)


def test_evict_strides_and_many_sequences():
    s = Setting(E2M1, [(53 * b) % 170 for b in range(70)], 2, 64, seed=2, token_major=True)
    _check_evicted(s, 60, 20, 80)
    wide = torch.full((s.weights.shape[0], 17, 5), 3.0).cuda()
    wide[:, 1:, 1:3] = s.weights
    before = wide.clone()
    s.lengths = [min(n, 60) for n in s.lengths]
    s.weights = wide[:, 1:, 1:3]
    _check_evicted(s, 10, 3)
    before[:, 1:, 1:3] = s.weights
    assert torch.equal(wide, before)


def test_long_sequences_and_pages_past_four_gigabytes():
    kind, page, Hkv, D = E2M1, 64, 8, 128
    pages = (2 << 32) // (page * Hkv * D // 2) + 50
    cache, scales = M.paged_cache(pages, page, Hkv, D, kind)
    weights = M.paged_weights(pages, page, Hkv)
    length = 40000
    count = -(-length // page)
    g = torch.Generator().manual_seed(0)
    order = torch.cat([torch.arange(pages - count // 2, pages), torch.arange(count - count // 2)])[torch.randperm(count, generator=g)]
    table = order.int().view(1, -1).cuda()
    cache.view(torch.uint8)[:, order.cuda()] = torch.randint(0, 256, (2, count, page, Hkv, D // 2), generator=g, dtype=torch.uint8).cuda()
    scales.view(torch.uint8)[:, order.cuda()] = torch.randint(1, 250, (2, count, page, Hkv, 4), generator=g, dtype=torch.uint8).cuda()
    weights[order.cuda()] = torch.rand(count, page, Hkv, generator=g).cuda()
    position = torch.arange(length)
    at, slot = order[position // page].cuda(), (position % page).cuda()
    rows, row_scales, had = cache.view(torch.uint8)[:, at, slot], scales.view(torch.uint8)[:, at, slot], weights[at, slot]
    kept, left = M.paged_cache_evict(cache, table, _ints([length]), weights, 30000, recent=1000, scales=scales)
    assert left.item() == 30000
    for h in range(Hkv):
        value = had[:length - 1000, h].cpu()
        stay = torch.sort(torch.sort(value, descending=True, stable=True).indices[:29000]).values
        want = torch.cat([stay, torch.arange(length - 1000, length)])
        assert torch.equal(kept[0, h].cpu(), want.int())
        want = want.cuda()
        assert torch.equal(cache.view(torch.uint8)[:, at[:30000], slot[:30000], h], rows[:, want, h])
        assert torch.equal(scales.view(torch.uint8)[:, at[:30000], slot[:30000], h], row_scales[:, want, h])
        assert torch.equal(weights[at[:30000], slot[:30000], h], had[want, h])


@pytest.mark.parametrize("pattern", ["spread", "equal", "few", "close", "two"])
@pytest.mark.parametrize("length", [2048, 2049, 8193, 32768, 32800, 70000])
def test_which_positions_of_long_sequences_stay(length, pattern):
    """Every way a sequence's weights are held, with weights that share all, most or few of their bits."""
    page, Hkv, D = 64, 2, 8
    count = -(-length // page)
    g = torch.Generator().manual_seed(length)
    cache, _ = M.paged_cache(2 * count, page, Hkv, D)
    table = torch.randperm(2 * count, generator=g)[:count].int().view(1, -1)
    w = {"spread": torch.exp(4 * torch.randn(length, Hkv, generator=g)), "equal": torch.full((length, Hkv), 0.25),
         "few": torch.randint(0, 3, (length, Hkv), generator=g).float(), "close": 1 + torch.rand(length, Hkv, generator=g) / 4,
         "two": torch.where(torch.rand(length, Hkv, generator=g) < 0.5, -1.5, 1.5)}[pattern]
    weights = M.paged_weights(2 * count, page, Hkv)
    position = torch.arange(length)
    at, slot = table[0][position // page].long().cuda(), (position % page).cuda()
    weights[at, slot] = w.cuda()
    out_table = torch.tensor([sorted(set(range(2 * count)) - set(table[0].tolist()))[:count]], dtype=torch.int32).cuda()
    for keep, recent in ((length - 1, 0), (length // 3, 100), (101, 100), (200, 200)):
        kept, left = M.paged_cache_evict(cache, table.cuda(), _ints([length]), weights, keep, recent=recent, out_table=out_table)
        assert left.item() == keep
        for h in range(Hkv):
            order = torch.sort(w[:length - recent, h], descending=True, stable=True).indices[:keep - recent]
            want = torch.cat([torch.sort(order).values, torch.arange(length - recent, length)])
            assert torch.equal(kept[0, h].cpu(), want.int()), (keep, recent, h)


@pytest.mark.parametrize("kind", KINDS, ids=NAMES)
def test_a_serving_run_within_a_budget(kind):
    """Prompts by packed chunks, then token by token; every step writes, attends, adds up weights and evicts, captured once and
    replayed: attention is over the keys that stayed, those are the ones with the largest sums, and lengths stay within the limit."""
    H, Hkv, D, page, keep, recent, limit = 4, 2, 64, 16, 40, 12, 48
    g = torch.Generator().manual_seed(31)
    pages = 16
    cache, scales = M.paged_cache(pages, page, Hkv, D, kind)
    weights = M.paged_weights(pages, page, Hkv)
    table = torch.randperm(pages, generator=g)[:10].view(2, 5).tolist()
    dev_table, lengths, starts = _ints(table), _ints([0, 0]), _ints([0, 0, 0])
    T = 60
    q, k, v = (torch.zeros(T, h, D, dtype=torch.bfloat16).cuda() for h in (H, Hkv, Hkv))
    out, lse = torch.zeros(T, H, D, dtype=torch.bfloat16).cuda(), torch.zeros(H, T).cuda()
    result = {}

    def step():
        M.paged_cache_write(k, v, cache, dev_table, lengths, scales=scales, starts=starts)
        M.paged_attn_fwd(q, cache, dev_table, lengths, D ** -0.5, scales=scales, starts=starts, most_new=T, out=out, lse=lse)
        M.paged_attn_weights(q, cache, dev_table, lengths, D ** -0.5, lse, weights, scales=scales, starts=starts, most_new=T)
        result["kept"], result["left"] = M.paged_cache_evict(cache, dev_table, lengths, weights, keep, recent=recent, limit=limit, scales=scales)

    graphed = M.GraphedStep(step)
    for t in (cache, scales):
        if t is not None:
            (t if t.dtype == torch.float32 else t.view(torch.uint8)).zero_()
    weights.zero_()
    values = torch.zeros(2, pages, page, Hkv, D, dtype=torch.float64)          # what the cache stands for
    want_weights = torch.zeros(pages, page, Hkv, dtype=torch.float64)
    now = [0, 0]
    for new in ([30, 21], [20, 1], [1, 1], *([1, 1] for _ in range(12)), [0, 25], [1, 1], [9, 1]):
        at = [0, new[0], sum(new)]
        now = [a + b for a, b in zip(now, new)]
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        starts.copy_(torch.tensor(at, dtype=torch.int32))
        read_before = M.paged_cache_read(cache, dev_table, lengths, 5 * page, scales=scales)                # (other work between the replays)
        graphed.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(read_before[:, 0, :max(now[0] - new[0], 0)]).all()
        # the new rows, as the cache holds them
        for b in (0, 1):
            x = torch.stack([k, v])[:, at[b]:at[b + 1]].cpu()
            for half in (0, 1):
                for i in range(new[b]):
                    j = now[b] - new[b] + i
                    for h in range(Hkv):
                        row = x[half, i, h]
                        if kind == E4M3:
                            codes, scale = P.quantise_row(row)
                            row = codes * scale
                        elif kind == E2M1:
                            codes, scale = P.quantise_e2m1(row)
                            row = P.e2m1_values(codes, torch.cat([scale, scale]))
                        values[half, table[b][j // page], j % page, h] = row.double()
        rows = q.cpu()[:at[2]]
        for b, (o, l, o_off, l_off) in enumerate(P.paged_attention(rows, values, table, now, D ** -0.5, True, None, at)):
            mine = slice(at[b], at[b + 1])
            assert ((out[mine].cpu().double() - o).abs() <= o_off).all() and ((lse[:, mine].cpu().double() - l).abs() <= l_off).all()
        # (the kernel's own lse, which is what the weights are taken with)
        before = want_weights.clone()
        want_weights, off = P.paged_weights(rows, values, table, now, D ** -0.5, lse.cpu()[:, :at[2]], before, True, at)
        kept, left = result["kept"].cpu(), result["left"].tolist()
        assert left == [keep if n > limit else n for n in now]
        moved = values.clone(), want_weights.clone()
        for b in (0, 1):
            for h in range(Hkv):
                stay = [j for j in kept[b, h].tolist() if j >= 0]
                assert len(stay) == left[b] and stay == sorted(stay)
                if now[b] > limit:
                    assert stay[-recent:] == list(range(now[b] - recent, now[b]))
                    had = [want_weights[table[b][j // page], j % page, h].item() for j in range(now[b] - recent)]
                    gone = [w for j, w in enumerate(had) if j not in stay]
                    # sums in 32 bits over at most 100 steps differ from those in 64 by less than this
                    assert max(gone) <= min(w for j, w in enumerate(had) if j in stay) * (1 + 1e-3) + 1e-6
                for i, j in enumerate(stay):
                    to, from_ = (table[b][i // page], i % page), (table[b][j // page], j % page)
                    values[:, to[0], to[1], h] = moved[0][:, from_[0], from_[1], h]
                    want_weights[to[0], to[1], h] = moved[1][from_[0], from_[1], h]
        now = left
        # the restatement goes on from the kernel's sums, so that ties stay ties
        got = weights.cpu().double()
        for b in (0, 1):
            for j in range(now[b]):
                at_ = table[b][j // page], j % page
                assert ((got[at_] - want_weights[at_]).abs() <= 1e-4 + 1e-3 * want_weights[at_].abs()).all()
                want_weights[at_] = got[at_]


def test_on_other_streams_and_two_at_once():
    settings = [Setting(E4M3, [900, 131, 450], 2, 128, seed=i) for i in (1, 2)]
    want = []
    for s in settings:
        w = P.evicted(s.weights.cpu(), s.table, s.lengths, s.dev.shape[1], 100, 10)
        want.append(w)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s, st in zip(settings, streams):
        table, lengths = s.tables()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            got.append(M.paged_cache_evict(s.dev, table, lengths, s.weights, 100, recent=10, scales=s.scales))
    torch.cuda.synchronize()
    for (kept, left), (stay, n) in zip(got, want):
        assert left.tolist() == n and kept.tolist() == stay


def test_weights_of_two_prompts_at_once_on_two_streams():
    """Each call has partial sums of its own."""
    calls = []
    for i, (lengths, new) in enumerate((([2100, 300], 300), ([900, 1700, 64], 64))):
        s = Setting(torch.bfloat16, lengths, 2, 128, seed=50 + i)
        q = torch.randn(len(lengths), new, 8, 128, generator=s.g).bfloat16().cuda()
        _, lse = M.paged_attn_fwd(q, s.dev, *s.tables(), 0.1)
        calls.append((s, q, lse, s.tables(), torch.zeros_like(s.weights)))
    alone = [M.paged_attn_weights(q, s.dev, *tables, 0.1, lse, s.weights, out=torch.zeros_like(out)) for s, q, lse, tables, out in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for (s, q, lse, tables, out), stream in zip(calls, streams):
            with torch.cuda.stream(stream):
                M.paged_attn_weights(q, s.dev, *tables, 0.1, lse, s.weights, out=out)
    torch.cuda.synchronize()
    for (*_, out), want in zip(calls, alone):
        assert torch.equal(out, want)


@pytest.mark.parametrize("lengths,page", [([1999, 63, 5000], 48), ([8300, 17000, 300], 64), ([33100, 40007], 112)])
def test_which_positions_stay_whatever_the_strides(lengths, page):
    """Weights that lie by tokens, inside a wider tensor, and pages that end inside a wavefront's run of positions."""
    g = torch.Generator().manual_seed(page)
    counts = [-(-n // page) for n in lengths]
    pages, keep, recent = sum(counts), 200, 37
    order = torch.randperm(pages, generator=g).tolist()
    table = [order[sum(counts[:b]):sum(counts[:b + 1])] for b in range(len(lengths))]
    wide = torch.randn(pages, page + 1, 5, generator=g).cuda()
    weights = wide[:, 1:, 1:4:2]
    assert weights.stride() == ((page + 1) * 5, 5, 2)
    cache, _ = M.paged_cache(pages, page, 2, 8)
    cache.zero_()
    want, left = P.evicted(weights.cpu(), table, lengths, pages, keep, recent)
    rows = _ints([row + [-1] * (max(counts) - len(row)) for row in table])
    kept, now = M.paged_cache_evict(cache, rows, _ints(lengths), weights, keep, recent=recent)
    assert now.tolist() == left
    for b, n in enumerate(left):
        for h in range(2):
            assert kept[b, h, :n].tolist() == want[b][h] and (kept[b, h, n:] == -1).all()


def test_the_interpreters_path_gives_the_same(monkeypatch):
    def run():
        s = Setting(E2M1, [140, 95], 2, 64, seed=3, spare=20)
        q = torch.randn(2, 3, 4, 64, generator=s.g).bfloat16().cuda()
        _, lse = M.paged_attn_fwd(q, s.dev, *s.tables(), 0.1, scales=s.scales)
        w = M.paged_attn_weights(q, s.dev, *s.tables(), 0.1, lse, s.weights, scales=s.scales, decay=0.5)
        assert w is s.weights
        kept, left = M.paged_cache_evict(s.dev, *s.tables(), s.weights, 60, 7, 100, scales=s.scales)
        first = [_raw(t) for t in (w, kept, left, s.dev, s.scales)]
        kept, left = M.paged_cache_evict(s.dev, *s.tables(), s.weights, 60, 7, scales=s.scales,
                                         out_table=_ints([s.free[:4], s.free[4:8]]))
        return first + [_raw(t) for t in (kept, left, s.dev, s.scales, s.weights)]

    want = run()

    class Declines:
        def __init__(self, host):
            self.written = host.written

        def __getattr__(self, name):
            return lambda *args: None

    versions = []
    monkeypatch.setattr(N, "host", Declines(N.host))
    got = run()
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and versions == []


def test_what_is_written_counts_as_written():
    s = Setting(E4M3, [60], 2, 64)
    table, lengths = s.tables()
    q = torch.randn(1, 1, 4, 64).bfloat16().cuda()
    _, lse = M.paged_attn_fwd(q, s.dev, table, lengths, 0.1, scales=s.scales)
    other = torch.zeros_like(s.weights)
    for call, changed in [
        (lambda: M.paged_attn_weights(q, s.dev, table, lengths, 0.1, lse, s.weights, scales=s.scales), (s.weights,)),
        (lambda: M.paged_attn_weights(q, s.dev, table, lengths, 0.1, lse, s.weights, scales=s.scales, out=other), (other,)),
        (lambda: M.paged_cache_evict(s.dev, table, lengths, s.weights, 50, scales=s.scales), (s.dev, s.scales, s.weights)),
    ]:
        tensors = (q, lse, table, lengths, s.dev, s.scales, s.weights, other)
        before = [t._version for t in tensors]
        call()
        assert [t._version > n for t, n in zip(tensors, before)] == [any(t is c for c in changed) for t in tensors]


def test_nothing_to_do():
    cache, scales = M.paged_cache(4, 16, 2, 64, E4M3)
    weights = M.paged_weights(4, 16, 2)
    empty = torch.zeros(0, 4, dtype=torch.int32).cuda(), torch.zeros(0, dtype=torch.int32).cuda()
    q = torch.zeros(0, 1, 4, 64, dtype=torch.bfloat16).cuda()
    assert M.paged_attn_weights(q, cache, *empty, 0.1, torch.zeros(0, 4, 1).cuda(), weights, scales=scales) is weights
    kept, left = M.paged_cache_evict(cache, *empty, weights, 5, scales=scales)
    assert kept.shape == (0, 2, 5) and left.shape == (0,)
    none, _ = M.paged_cache(0, 16, 2, 64)
    no_weights = M.paged_weights(0, 16, 2)
    table, lengths = torch.zeros(2, 0, dtype=torch.int32).cuda(), torch.full((2,), 7, dtype=torch.int32).cuda()
    q = torch.ones(2, 3, 4, 64, dtype=torch.bfloat16).cuda()
    M.paged_attn_weights(q, none, table, lengths, 0.1, torch.zeros(2, 4, 3).cuda(), no_weights)
    kept, left = M.paged_cache_evict(none, table, lengths, no_weights, 5)
    assert (kept == -1).all() and (left == 0).all()                                # (a table without columns holds no token)
    s = Setting(torch.bfloat16, [40, 9], 2, 64)
    before = s.weights.clone()
    M.paged_attn_weights(torch.zeros(2, 0, 4, 64, dtype=torch.bfloat16).cuda(), s.dev, *s.tables(), 0.1, torch.zeros(2, 4, 0).cuda(), s.weights, decay=0.5)
    assert torch.equal(s.weights, before)


def test_refusals_say_why():
    s = Setting(E4M3, [40], 2, 64, spare=8)
    table, lengths = s.tables()
    q, lse = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16).cuda(), torch.zeros(1, 4, 1).cuda()
    weigh = lambda q=q, lse=lse, weights=s.weights, scale=0.1, **kw: M.paged_attn_weights(                 # noqa: E731
        q, s.dev, table, lengths, scale, lse, weights, scales=s.scales, **kw)
    evict = lambda keep=10, weights=s.weights, **kw: M.paged_cache_evict(s.dev, table, lengths, weights, keep, scales=s.scales, **kw)      # noqa: E731
    weigh()
    out_table = _ints([s.free[:3]])
    for message, call in [
        ("lse must", lambda: weigh(lse=lse[:, :2])),
        ("lse must", lambda: weigh(lse=lse.double())),
        ("weights must", lambda: weigh(weights=s.weights[1:])),
        ("weights must", lambda: weigh(weights=s.weights.double())),
        ("out must", lambda: weigh(out=s.weights[1:])),
        ("GPU only", lambda: weigh(weights=s.weights.cpu())),
        ("GPU only", lambda: weigh(lse=lse.cpu())),
        ("multiple", lambda: weigh(q=q[:, :, :3])),
        ("q must be", lambda: weigh(q=q.float())),
        ("scale", lambda: weigh(scale=0.0)),
        ("invalid", lambda: weigh(decay=-0.5)),
        ("invalid", lambda: weigh(decay=math.nan)),
        ("no gradients", lambda: weigh(weights=s.weights.clone().requires_grad_())),
        ("no gradients", lambda: weigh(lse=lse.clone().requires_grad_())),
        ("scales", lambda: M.paged_attn_weights(q, s.dev, table, lengths, 0.1, lse, s.weights)),
        ("weights must", lambda: evict(weights=s.weights[1:])),
        ("no gradients", lambda: evict(weights=s.weights.clone().requires_grad_())),
        ("keep", lambda: evict(keep=-1)),
        ("whole number", lambda: evict(keep=1.5)),
        ("whole number", lambda: evict(keep=2 ** 31)),
        ("recent", lambda: evict(recent=11)),
        ("limit", lambda: evict(limit=9)),
        ("out_table must be", lambda: evict(out_table=out_table.long())),
        ("out_table must be", lambda: evict(out_table=out_table[0])),
        ("pages for 49 rows", lambda: evict(limit=49, out_table=out_table)),
        ("GPU only", lambda: evict(out_table=out_table.cpu())),
        ("scales", lambda: M.paged_cache_evict(s.dev, table, lengths, s.weights, 10)),
    ]:
        with pytest.raises(RuntimeError, match=message):
            call()
