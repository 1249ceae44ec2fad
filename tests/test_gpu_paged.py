"""The operators over a paged K/V cache against their 64-bit restatement (oracle/paged_oracle.py), whose docstring derives how
far attention may be off.  Whatever a cache holds where no key of a sequence lies is NaN here."""
import math

import pytest
import torch

import mercury_artifact_amd as M
from mercury_artifact_amd import _native as N
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


class Setting:
    """A cache whose sequences' rows are N(0, 1) and whose other rows are NaN, with its table, on the CPU and on the GPU."""

    def __init__(self, lengths, Hkv, D, page, e4m3, seed=0, spare=2, width=None, token_major=False, gain=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.page, self.e4m3, self.D, self.Hkv = list(lengths), page, e4m3, D, Hkv
        counts = [-(-n // page) for n in lengths]
        pages = sum(counts) + spare
        order, at = torch.randperm(pages, generator=g).tolist(), 0
        width = max([*counts, 1]) if width is None else width
        self.table = []
        for c in counts:
            self.table.append(order[at:at + c] + [-1] * (width - c))
            at += c
        real = torch.zeros(pages, page, dtype=torch.bool)
        for b, n in enumerate(lengths):
            for j in range(n):
                real[self.table[b][j // page], j % page] = True
        x = torch.randn(2, pages, page, Hkv, D, generator=g) * gain
        self.scales = None
        if e4m3:
            codes = torch.full(x.shape, math.nan, dtype=torch.float64)
            scales = torch.full(x.shape[:-1], math.nan)
            for p_, s in real.nonzero().tolist():
                for half in (0, 1):
                    for h in range(Hkv):
                        codes[half, p_, s, h], scales[half, p_, s, h] = P.quantise_row(x[half, p_, s, h].bfloat16())
            self.scales, self.cache = scales, codes
            dev = codes.float().to(E4M3)
        else:
            self.cache = torch.where(real[None, :, :, None, None], x, math.nan).bfloat16()
            dev = self.cache
        if not token_major:
            order5 = lambda t: t.transpose(2, 3).contiguous().cuda().transpose(2, 3)           # noqa: E731
        else:
            order5 = lambda t: t.cuda()                                                        # noqa: E731
        self.dev = order5(dev)
        self.dev_scales = None if self.scales is None else order5(self.scales)
        self.g = g

    def tables(self):
        return torch.tensor(self.table, dtype=torch.int32).view(len(self.lengths), -1).cuda(), torch.tensor(self.lengths, dtype=torch.int32).cuda()


def _starts(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return s


def _attend(s, q, scale, causal=True, starts=None, **kw):
    table, lengths = s.tables()
    out, lse = M.paged_attn_fwd(q.cuda(), s.dev, table, lengths, scale, causal=causal, scales=s.dev_scales,
                                starts=None if starts is None else torch.tensor(starts, dtype=torch.int32).cuda(), **kw)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def _check(s, q, out, lse, scale, causal=True, starts=None, table=None):
    want = P.paged_attention(q, s.cache, s.table if table is None else table, s.lengths, scale, causal, s.scales, starts)
    for b, (o, l, o_off, l_off) in enumerate(want):
        got = P.tokens_of(b, out, starts).double()
        got_l = (lse[b] if starts is None else lse[:, starts[b]:starts[b + 1]]).double()
        assert torch.equal(torch.isfinite(got), torch.isfinite(o)), b
        assert torch.equal(got_l == -math.inf, l == -math.inf), b
        assert ((got - o).abs() <= o_off)[torch.isfinite(o)].all(), (b, ((got - o).abs() - o_off).max())
        seen = torch.isfinite(l)
        assert ((got_l - l).abs() <= l_off)[seen].all(), (b, ((got_l - l).abs() - l_off)[seen].max())


CASES = [
    # lengths, new, Hq, Hkv, D, page, causal
    ([1], 1, 1, 1, 128, 16, True),
    ([0, 1, 15, 16, 17, 31, 32, 33], 1, 4, 2, 128, 16, True),
    ([127, 128, 129, 300, 1, 0], 1, 8, 2, 64, 16, True),
    ([500, 3, 1029], 1, 5, 5, 80, 32, True),
    ([257, 64, 1], 1, 32, 2, 128, 48, False),
    ([700], 1, 7, 1, 96, 64, True),
    ([40, 5, 129], 5, 4, 2, 128, 16, True),
    ([40, 5, 129], 5, 4, 2, 128, 16, False),
    ([90, 33], 4, 16, 2, 64, 16, True),             # 32 rows
    ([90, 33], 4, 17, 1, 32, 16, True),             # 68 rows, two tiles of them
    ([260, 131], 9, 6, 1, 112, 16, True),           # 54 rows
    ([2, 3, 50], 6, 2, 2, 128, 16, True),           # more new tokens than keys
    ([150, 130], 130, 2, 2, 128, 16, True),
    ([320], 77, 6, 2, 48, 256, True),
    ([200, 333], 150, 4, 1, 128, 32, False),
    ([1500], 300, 2, 1, 64, 16, True),
    ([16], 1, 2, 1, 16, 16, True),
]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths,new,Hq,Hkv,D,page,causal", CASES)
def test_attention(lengths, new, Hq, Hkv, D, page, causal, e4m3):
    print(f"case {lengths} new {new} H{Hq}/{Hkv} D{D} page {page} causal {causal} e4m3 {e4m3}", flush=True)
    s = Setting(lengths, Hkv, D, page, e4m3, seed=len(lengths) + new)
    q = torch.randn(len(lengths), new, Hq, D, generator=s.g).bfloat16()
    out, lse = _attend(s, q, D ** -0.5, causal)
    _check(s, q, out, lse, D ** -0.5, causal)


@pytest.mark.parametrize("D", [8, 24, 40, 72, 88, 104, 120])
def test_attention_head_dimensions_that_are_no_multiple_of_16(D):
    s = Setting([70, 200], 2, D, 16, False, seed=D)
    q = torch.randn(2, 3, 4, D, generator=s.g).bfloat16()
    out, lse = _attend(s, q, D ** -0.5)
    _check(s, q, out, lse, D ** -0.5)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("most", [None, 1, 3, 40, 1000])
@pytest.mark.parametrize("lengths,new,Hq,Hkv,D", [
    ([40, 300, 17, 9, 0, 64], [1, 0, 3, 9, 0, 40], 4, 2, 128),
    ([500, 130, 260, 5], [1, 130, 1, 5], 4, 1, 64),
    ([33], [0], 2, 2, 64),
])
def test_attention_packed(lengths, new, Hq, Hkv, D, most, e4m3):
    """Sequences of any number of new tokens, none among them; rows before the first and behind the last are left alone,
    whatever form the hint chooses."""
    s = Setting(lengths, Hkv, D, 16, e4m3, seed=5, width=40)
    starts = [2 + x for x in _starts(new)]
    T = starts[-1] + 3
    q = torch.randn(T, Hq, D, generator=s.g).bfloat16()
    q[:2], q[T - 3:] = math.nan, math.nan
    out = torch.full((T, Hq, D), 7.0, dtype=torch.bfloat16).cuda()
    lse = torch.full((Hq, T), 7.0).cuda()
    out, lse = _attend(s, q, D ** -0.5, starts=starts, most_new=most, out=out, lse=lse)
    _check(s, q, out, lse, D ** -0.5, starts=starts)
    assert (out[:2] == 7).all() and (out[T - 3:] == 7).all() and (lse[:, :2] == 7).all() and (lse[:, T - 3:] == 7).all()


@pytest.mark.parametrize("e4m3", [False, True])
def test_many_sequences(e4m3):
    """More sequences than lanes of a wavefront, the longest beside the shortest, shares that end inside an item."""
    lengths = [(37 * b) % 61 for b in range(150)]
    lengths[77] = 2000
    s = Setting(lengths, 1, 64, 16, e4m3, seed=9)
    q = torch.randn(150, 1, 3, 64, generator=s.g).bfloat16()
    out, lse = _attend(s, q, 0.125)
    _check(s, q, out, lse, 0.125)


@pytest.mark.parametrize("new", [1, 3, 100])
@pytest.mark.parametrize("e4m3", [False, True])
def test_pages_that_are_not_here_and_parts_that_merge(e4m3, new):
    """Keys of pages that are not here (whatever number says so) are seen by nobody; two ranks with the even and the odd
    pages merge to the whole."""
    s = Setting([210, 5, 400], 2, 128, 16, e4m3, seed=11)
    q = torch.randn(3, new, 4, 128, generator=s.g).bfloat16()
    scale, parts = 128 ** -0.5, []
    whole, pages = s.table, s.cache.shape[1]
    for rank, nobody in ((0, -1), (1, pages), (1, 2 ** 31 - 1), (0, -2 ** 31)):
        s.table = [[e if i % 2 == rank else nobody for i, e in enumerate(row)] for row in whole]
        out, lse = _attend(s, q, scale)
        _check(s, q, out, lse, scale)
        parts.append((out, lse))
    s.table = whole
    # the merge weighs two results, each off by its bound, and rounds once more
    out, lse = torch.empty(q.shape, dtype=torch.bfloat16).cuda(), torch.empty(3, 4, new).cuda()
    M.merge_many([o.cuda() for o, _ in parts[:2]], [l.cuda() for _, l in parts[:2]], out, lse)
    want = P.paged_attention(q, s.cache, whole, s.lengths, scale, True, s.scales)
    for b, (o, l, o_off, l_off) in enumerate(want):
        assert ((out[b].cpu().double() - o).abs() <= 3 * o_off).all()
        seen = torch.isfinite(l)
        assert ((lse[b].cpu().double() - l).abs() <= 2 * l_off + 1e-5)[seen].all()


@pytest.mark.parametrize("new", [4, 70, 200])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_a_value_that_is_no_number_reaches_the_rows_that_see_it_alone(what, new):
    """In the values (and keys) of a new token, which the tokens before it do not see though their tile holds it."""
    s = Setting([230], 1, 128, 16, False, seed=3)
    q = torch.randn(1, new, 2, 128, generator=s.g).bfloat16()
    at = 230 - new + new // 2
    page, slot = s.table[0][at // 16], at % 16
    s.cache[1, page, slot, 0, 5] = what
    s.dev[1, page, slot, 0, 5] = what
    if math.isnan(what):
        s.cache[0, page, slot, 0, 7] = what
        s.dev[0, page, slot, 0, 7] = what
    out, lse = _attend(s, q, 0.1)
    finite = torch.isfinite(out[0])
    assert finite[:new // 2].all() and torch.isfinite(lse[0, :, :new // 2]).all()
    if math.isnan(what):
        assert torch.isnan(out[0, new // 2:]).all() and torch.isnan(lse[0, :, new // 2:]).all()
    else:
        assert (out[0, new // 2:, :, 5] == what).all()
        finite[new // 2:, :, 5] = True
        assert finite.all()
    want = P.paged_attention(q, s.cache, s.table, s.lengths, 0.1)[0]
    good = torch.isfinite(want[0])
    assert torch.equal(good, torch.isfinite(out[0])) and ((out[0].double() - want[0]).abs() <= want[2])[good].all()


def test_an_e4m3_row_that_is_no_number_reaches_the_rows_that_see_it_alone():
    s = Setting([90], 1, 64, 16, True, seed=4)
    table, lengths = s.tables()
    k = torch.randn(1, 6, 1, 64, generator=s.g).bfloat16()
    v = k.clone()
    v[0, 3, 0, 9] = math.inf
    M.paged_cache_write(k.cuda(), v.cuda(), s.dev, table, lengths, scales=s.dev_scales)
    q = torch.randn(1, 6, 2, 64, generator=s.g).bfloat16()
    out, lse = _attend(s, q, 0.1)
    assert torch.isfinite(out[0, :3]).all() and torch.isnan(out[0, 3:]).all() and torch.isfinite(lse).all()
    got = M.paged_cache_read(s.dev, table, lengths, 90, scales=s.dev_scales)
    assert torch.isnan(got[1, 0, 87]).all() and torch.isfinite(got[0]).all() and torch.isfinite(got[1, 0, :87]).all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [1, 90])
def test_large_scores(e4m3, new):
    """Rising and falling scores far apart: the maximum moves with every tile, weights underflow."""
    s = Setting([600], 1, 64, 16, e4m3, seed=6, gain=6.0)
    q = (torch.randn(1, new, 4, 64, generator=s.g) * 6).bfloat16()
    out, lse = _attend(s, q, 1.0)
    _check(s, q, out, lse, 1.0)


def test_strides_and_orders():
    """A cache in the order of its tokens, q and out as slices of wider tensors, a table as a slice of a wider one."""
    for e4m3 in (False, True):
        s = Setting([100, 37], 2, 64, 16, e4m3, seed=8, token_major=True)
        table, lengths = s.tables()
        wide = torch.full((2, table.shape[1] + 5), 10 ** 6, dtype=torch.int32).cuda()
        wide[:, :table.shape[1]] = table
        q = torch.randn(2, 3, 4, 64, generator=s.g).bfloat16()
        big = torch.full((2, 3, 8, 128), math.nan, dtype=torch.bfloat16).cuda()
        big[:, :, 2:6, 64:] = q.cuda()
        res = torch.full((2, 4, 5, 80), 3.0, dtype=torch.bfloat16).cuda()
        out, lse = M.paged_attn_fwd(big[:, :, 2:6, 64:], s.dev, wide[:, :table.shape[1]], lengths, 0.1, scales=s.dev_scales,
                                    out=res[:, 1:, :4, 8:72])
        _check(s, q, out.cpu(), lse.cpu(), 0.1)
        res[:, 1:, :4, 8:72] = 3.0
        assert (res == 3).all()


@pytest.mark.parametrize("D,e4m3", [(128, False), (128, True), (80, True), (72, False), (16, True), (8, False)])
@pytest.mark.parametrize("packed", [False, True])
def test_written_and_read_back(D, e4m3, packed):
    """Bit for bit; rows beside the new ones are left as they were; rows past an end are zeros."""
    s = Setting([50, 7, 130, 0, 33], 3, D, 16, e4m3, seed=D, width=10)
    table, lengths = s.tables()
    new = [5, 7, 40, 0, 1] if packed else [7] * 5
    starts = [1 + x for x in _starts(new)] if packed else None
    shape = (starts[-1] + 2,) if packed else (5, 7)
    k = (torch.randn(*shape, 3, D, generator=s.g) * torch.exp2(torch.randint(-20, 20, (*shape, 3, 1), generator=s.g))).bfloat16()
    v = torch.randn(*shape, 3, D, generator=s.g).bfloat16()
    first = (2,) if packed else (2, 1)
    k[first], v[first] = 0.0, v[first] * 2.0 ** -124         # a row of zeros, one below the least scale
    if e4m3:
        k[(4,) if packed else (0, 3)][1, 3] = math.nan
    s.table[2][7] = -1                                     # a page that is not here: its rows are dropped
    table, lengths = s.tables()
    want, want_scales = s.cache.clone(), None if s.scales is None else s.scales.clone()
    P.paged_write(k, v, want, s.table, s.lengths, want_scales, starts)
    M.paged_cache_write(k.cuda(), v.cuda(), s.dev, table, lengths, scales=s.dev_scales,
                        starts=None if starts is None else torch.tensor(starts, dtype=torch.int32).cuda())
    got = s.dev.float().cpu().double()
    assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(want.double(), nan=1e9))
    if e4m3:
        assert torch.equal(torch.nan_to_num(s.dev_scales.cpu(), nan=1e9), torch.nan_to_num(want_scales, nan=1e9))
    for begin, rows in ((0, 140), (20, 60), (129, 1), (0, 0), (200, 3)):
        read = M.paged_cache_read(s.dev, table, lengths, rows, begin=begin, scales=s.dev_scales)
        plain = P.paged_read(want, s.table, s.lengths, rows, begin, want_scales).bfloat16()
        assert torch.equal(torch.nan_to_num(read.cpu(), nan=1e9), torch.nan_to_num(plain, nan=1e9))


def test_read_into_a_slice():
    s = Setting([50, 7], 2, 64, 16, True, seed=1)
    table, lengths = s.tables()
    big = torch.full((2, 3, 70, 2, 72), 3.0, dtype=torch.bfloat16).cuda()
    out = M.paged_cache_read(s.dev, table, lengths, 60, scales=s.dev_scales, out=big[:, 1:, 5:65, :, 8:])
    assert torch.equal(out.cpu(), P.paged_read(s.cache, s.table, s.lengths, 60, 0, s.scales).bfloat16())
    big[:, 1:, 5:65, :, 8:] = 3.0
    assert (big == 3).all()


def test_lengths_and_starts_outside_the_tensors_count_as_the_nearest_inside():
    s = Setting([64, 64, 64], 1, 64, 16, False, seed=2)
    table, _ = s.tables()
    q = torch.randn(9, 2, 64, generator=s.g).bfloat16()
    odd = torch.tensor([2 ** 31 - 1, -5, 65], dtype=torch.int32).cuda()
    s.lengths = [64, 0, 64]
    starts = torch.tensor([-7, 3, 3, 2 ** 31 - 1], dtype=torch.int32).cuda()
    out, lse = M.paged_attn_fwd(q.cuda(), s.dev, table, odd, 0.1, starts=starts, causal=False)
    _check(s, q, out.cpu(), lse.cpu(), 0.1, causal=False, starts=[0, 3, 3, 9])
    # starts that fall: nothing out of bounds, rows of no sequence left alone
    keep = torch.full((9, 2, 64), 5.0, dtype=torch.bfloat16).cuda()
    M.paged_attn_fwd(q.cuda(), s.dev, table, odd, 0.1, starts=torch.tensor([8, 2, 2, 0], dtype=torch.int32).cuda(), out=keep)
    assert (keep == 5).all()
    k = torch.randn(9, 1, 64, generator=s.g).bfloat16().cuda()
    before = s.dev.clone()
    M.paged_cache_write(k, k, s.dev, table, odd, starts=torch.tensor([8, 2, 2, 0], dtype=torch.int32).cuda())
    assert torch.equal(s.dev.view(torch.int16), before.view(torch.int16))
    read = M.paged_cache_read(s.dev, table, odd, 80)
    assert torch.equal(read.cpu(), P.paged_read(s.cache, s.table, s.lengths, 80).bfloat16())


@pytest.mark.parametrize("e4m3", [False, True])
def test_rows_past_four_gigabytes(e4m3):
    """Pages whose place passes 32 bits, in elements and in bytes."""
    pages, page, Hkv, D = (2 << 32) // (16 * 8 * 128) + 50, 16, 8, 128
    pages = pages // 2 if not e4m3 else pages
    cache, scales = M.paged_cache(pages, page, Hkv, D, E4M3 if e4m3 else torch.bfloat16)
    assert cache.stride(0) * cache.element_size() > 1 << 32
    table = torch.tensor([[pages - 1, 0, pages // 2 + 1]], dtype=torch.int32).cuda()
    lengths = torch.tensor([41], dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(1, 41, Hkv, D, generator=g).bfloat16(), torch.randn(1, 41, Hkv, D, generator=g).bfloat16()
    M.paged_cache_write(k.cuda(), v.cuda(), cache, table, lengths, scales=scales)
    read = M.paged_cache_read(cache, table, lengths, 41, scales=scales).cpu()
    if not e4m3:
        assert torch.equal(read[0], k) and torch.equal(read[1], v)
    else:
        assert ((read[0].float() - k.float()).abs() <= 2.0 ** -4 * k.float().abs() + 2.0 ** -9).all()
    q = torch.randn(1, 3, 8, D, generator=g).bfloat16()
    out, lse = M.paged_attn_fwd(q.cuda(), cache, table, lengths, 0.1, scales=scales)
    dense = torch.zeros(2, 3, 16, Hkv, D, dtype=torch.bfloat16)
    dense.view(2, 48, Hkv, D)[:, :41] = read[:, 0]
    for b, (o, l, o_off, l_off) in enumerate(P.paged_attention(q, dense, [[0, 1, 2]], [41], 0.1)):
        assert ((out[b].cpu().double() - o).abs() <= o_off).all() and ((lse[b].cpu().double() - l).abs() <= l_off).all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [1, 80])
def test_the_same_call_gives_the_same_bits(e4m3, new):
    s = Setting([900, 31, 450], 2, 128, 16, e4m3, seed=13)
    q = torch.randn(3, new, 8, 128, generator=s.g).bfloat16()
    first = _attend(s, q, 0.1)
    for _ in range(5):
        again = _attend(s, q, 0.1)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("e4m3", [False, True])
def test_a_captured_step_follows_lengths_and_table(e4m3):
    """Write and attend, captured once, replayed while the sequences grow by a token each time and one moves to other pages;
    an eager call and other work between the replays."""
    s = Setting([40, 100], 2, 64, 16, e4m3, seed=21, spare=12, width=12)
    table, lengths = s.tables()
    q, k, v = (torch.zeros(2, 1, h, 64, dtype=torch.bfloat16).cuda() for h in (4, 2, 2))
    out, lse = torch.empty_like(q), torch.empty(2, 4, 1).cuda()

    def step():
        M.paged_cache_write(k, v, s.dev, table, lengths, scales=s.dev_scales)
        M.paged_attn_fwd(q, s.dev, table, lengths, 0.1, scales=s.dev_scales, out=out, lse=lse)

    spare = [p for p in range(s.cache.shape[1]) if p not in sum(s.table, [])]
    graphed = M.GraphedStep(step)
    want, want_scales = s.cache, s.scales
    s.dev.copy_(want.float().to(E4M3).cuda() if e4m3 else want.cuda())         # (the capture's own runs wrote zeros)
    if e4m3:
        s.dev_scales.copy_(want_scales.cuda())
    for i in range(12):
        s.lengths = [n + 1 for n in s.lengths]
        for b, n in enumerate(s.lengths):
            if s.table[b][(n - 1) // 16] == -1:
                s.table[b][(n - 1) // 16] = spare.pop()
        table.copy_(torch.tensor(s.table, dtype=torch.int32))
        lengths.copy_(torch.tensor(s.lengths, dtype=torch.int32))
        new = [torch.randn(2, 1, h, 64, generator=s.g).bfloat16() for h in (4, 2, 2)]
        for t, x in zip((q, k, v), new):
            t.copy_(x)
        graphed.replay()
        torch.cuda.synchronize()
        got = out.cpu(), lse.cpu()
        P.paged_write(new[1], new[2], want, s.table, s.lengths, want_scales)
        _check(s, new[0], *got, 0.1)
        eager = _attend(s, new[0], 0.1)
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])


def test_on_another_stream_and_two_at_once():
    s = Setting([900, 31, 450], 2, 128, 16, False, seed=13)
    q = torch.randn(3, 1, 8, 128, generator=s.g).bfloat16()
    table, lengths = s.tables()
    want = _attend(s, q, 0.1)
    qs = [(q * f).bfloat16().cuda() for f in (1, 2)]
    wants = [want, _attend(s, (q * 2).bfloat16(), 0.1)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(M.paged_attn_fwd(qs[i], s.dev, table, lengths, 0.1))
    torch.cuda.synchronize()
    for i in (0, 1):
        for out, lse in got[i]:
            assert torch.equal(out.cpu(), wants[i][0]) and torch.equal(lse.cpu(), wants[i][1])


@pytest.mark.parametrize("e4m3", [False, True])
def test_a_prompt_by_chunks_and_then_token_by_token(e4m3):
    """As a serving program uses them together: prompts go in by packed chunks of uneven length, tokens follow one by one;
    every step's attention is that over what has been written so far, and at the end the rows read back are a chunk that a
    ring step takes, with the same result."""
    H, Hkv, D, page = 4, 2, 128, 16
    cache, scales = M.paged_cache(40, page, Hkv, D, E4M3 if e4m3 else torch.bfloat16)
    g = torch.Generator().manual_seed(31)
    want = torch.zeros(2, 40, page, Hkv, D, dtype=torch.float64 if e4m3 else torch.bfloat16)
    want_scales = torch.ones(2, 40, page, Hkv) if e4m3 else None
    order, table, lengths = torch.randperm(40, generator=g).tolist(), [[-1] * 16, [-1] * 16], [0, 0]
    for new in ([100, 33], [70, 1], [1, 1], [1, 1], [1, 0], [1, 1]):
        starts = _starts(new)
        lengths = [a + b for a, b in zip(lengths, new)]
        for b in (0, 1):
            for i in range(-(-lengths[b] // page)):
                if table[b][i] < 0:
                    table[b][i] = order.pop()
        q, k, v = (torch.randn(starts[-1], h, D, generator=g).bfloat16() for h in (H, Hkv, Hkv))
        dev = [torch.tensor(x, dtype=torch.int32).cuda() for x in (table, lengths, starts)]
        M.paged_cache_write(k.cuda(), v.cuda(), cache, dev[0], dev[1], scales=scales, starts=dev[2])
        out, lse = M.paged_attn_fwd(q.cuda(), cache, dev[0], dev[1], D ** -0.5, scales=scales, starts=dev[2], most_new=max(new))
        P.paged_write(k, v, want, table, lengths, want_scales, starts)
        for b, (o, l, o_off, l_off) in enumerate(P.paged_attention(q, want, table, lengths, D ** -0.5, True, want_scales, starts)):
            rows = slice(starts[b], starts[b + 1])
            assert ((out[rows].cpu().double() - o).abs() <= o_off).all() and ((lse[:, rows].cpu().double() - l).abs() <= l_off).all()
    chunk = M.paged_cache_read(cache, dev[0][:1], dev[1][:1], lengths[0], scales=scales)
    q1 = q[:1].cuda().view(1, 1, H, D)
    o, l = torch.empty_like(q1), torch.empty(1, H, 1).cuda()
    M.gqa_pack_kv(q1, chunk, o, l, D ** -0.5, ring=M.LocalRing((1,), 0, [chunk]))
    want0 = P.paged_attention(q, want, table, lengths, D ** -0.5, True, want_scales, starts)[0]
    assert ((o[0].cpu().double() - want0[0]).abs() <= 2 * want0[2]).all() and ((l[0].cpu().double() - want0[1]).abs() <= want0[3] + 1e-5).all()


def test_nothing_to_do():
    cache, scales = M.paged_cache(4, 16, 2, 64, E4M3)
    empty = torch.zeros(0, 4, dtype=torch.int32).cuda(), torch.zeros(0, dtype=torch.int32).cuda()
    q = torch.zeros(0, 1, 4, 64, dtype=torch.bfloat16).cuda()
    out, lse = M.paged_attn_fwd(q, cache, *empty, 0.1, scales=scales)
    assert out.shape == q.shape and lse.shape == (0, 4, 1)
    M.paged_cache_write(q[:, :, :2], q[:, :, :2], cache, *empty, scales=scales)
    assert M.paged_cache_read(cache, *empty, 5, scales=scales).shape == (2, 0, 5, 2, 64)
    none, _ = M.paged_cache(0, 16, 2, 64)                   # a cache without pages, a table without columns
    table, lengths = torch.zeros(2, 0, dtype=torch.int32).cuda(), torch.zeros(2, dtype=torch.int32).cuda()
    q = torch.ones(2, 3, 4, 64, dtype=torch.bfloat16).cuda()
    out, lse = M.paged_attn_fwd(q, none, table, lengths, 0.1)
    assert (out == 0).all() and (lse == -math.inf).all()
    M.paged_cache_write(q[:, :, :2], q[:, :, :2], none, table, lengths)
    assert (M.paged_cache_read(none, table, lengths, 5) == 0).all()


def test_refusals_say_why():
    s = Setting([40], 2, 64, 16, True)
    table, lengths = s.tables()
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16).cuda()
    M.paged_attn_fwd(q, s.dev, table, lengths, 0.1, scales=s.dev_scales)
    for message, call in [
        ("scales", lambda: M.paged_attn_fwd(q, s.dev, table, lengths, 0.1)),
        ("int32", lambda: M.paged_attn_fwd(q, s.dev, table.long(), lengths, 0.1, scales=s.dev_scales)),
        ("lengths", lambda: M.paged_attn_fwd(q, s.dev, table, lengths.long(), 0.1, scales=s.dev_scales)),
        ("multiple", lambda: M.paged_attn_fwd(q[:, :, :3], s.dev, table, lengths, 0.1, scales=s.dev_scales)),
        ("q must be", lambda: M.paged_attn_fwd(q.float(), s.dev, table, lengths, 0.1, scales=s.dev_scales)),
        ("q must be", lambda: M.paged_attn_fwd(q[0], s.dev, table, lengths, 0.1, scales=s.dev_scales)),
        ("starts", lambda: M.paged_attn_fwd(q[0], s.dev, table, lengths, 0.1, scales=s.dev_scales, starts=lengths)),
        ("GPU only", lambda: M.paged_attn_fwd(q.cpu(), s.dev, table, lengths, 0.1, scales=s.dev_scales)),
        ("GPU only", lambda: M.paged_attn_fwd(q, s.dev, table.cpu(), lengths, 0.1, scales=s.dev_scales)),
        ("scale", lambda: M.paged_attn_fwd(q, s.dev, table, lengths, 0.0, scales=s.dev_scales)),
        ("lse must", lambda: M.paged_attn_fwd(q, s.dev, table, lengths, 0.1, scales=s.dev_scales, lse=torch.zeros(1, 1, 4).cuda())),
        ("not implemented", lambda: M.paged_attn_fwd(q, s.dev[:, :, :8], table, lengths, 0.1, scales=s.dev_scales[:, :, :8])),
        ("head dimension", lambda: M.paged_attn_fwd(q[..., :24], s.dev[..., :24], table, lengths, 0.1, scales=s.dev_scales)),
        ("aligned", lambda: M.paged_attn_fwd(torch.zeros(1, 1, 4, 72, dtype=torch.bfloat16).cuda()[..., 4:68], s.dev, table, lengths, 0.1, scales=s.dev_scales)),
        ("k must be", lambda: M.paged_cache_write(q, q, s.dev, table, lengths, scales=s.dev_scales)),
        ("out must be", lambda: M.paged_cache_read(s.dev, table, lengths, 5, scales=s.dev_scales, out=q)),
        ("invalid", lambda: M.paged_cache_read(s.dev, table, lengths, 5, begin=-1, scales=s.dev_scales)),
    ]:
        with pytest.raises(RuntimeError, match=message):
            call()


@pytest.mark.parametrize("Hq,new", [(80, 1), (128, 1), (80, 2), (65, 1), (64, 1), (33, 2)])
def test_many_query_heads_on_one_key_head(Hq, new):
    """More rows of one token than the kernel for few rows takes, padded and packed."""
    s = Setting([200, 1, 77], 1, 64, 16, True, seed=Hq)
    q = torch.randn(3, new, Hq, 64, generator=s.g).bfloat16()
    out, lse = _attend(s, q, 0.125)
    _check(s, q, out, lse, 0.125)
    starts = [0, new, 2 * new, 3 * new]
    packed = q.reshape(3 * new, Hq, 64)
    for most in (None, new):
        out, lse = _attend(s, packed, 0.125, starts=starts, most_new=most)
        _check(s, packed, out, lse, 0.125, starts=starts)


@pytest.mark.parametrize("new,Hq", [(1, 2), (40, 2)])
def test_thousands_of_sequences(new, Hq):
    """More sequences than the plan of a launch keeps on chip; some of them against the restatement."""
    B = 2500
    s = Setting([(7 * b) % 45 for b in range(B)], 1, 16, 16, False, seed=B)
    q = torch.randn(B, new, Hq, 16, generator=s.g).bfloat16()
    out, lse = _attend(s, q, 0.25)
    for b in (0, 1, 63, 64, 65, 1000, 2047, 2048, 2049, 2499):
        one = Setting.__new__(Setting)
        one.cache, one.scales, one.lengths, one.table = s.cache, None, [s.lengths[b]], [s.table[b]]
        _check(one, q[b:b + 1], out[b:b + 1], lse[b:b + 1], 0.25)


def test_scales_that_are_no_powers_of_two():
    """Such as max|x| / 448: few rows take them exactly, long chunks count the rows as rounded to bf16."""
    for new in (1, 90):
        s = Setting([300], 1, 64, 16, True, seed=17)
        s.scales = s.scales * 0.77
        s.dev_scales = s.scales.transpose(2, 3).contiguous().cuda().transpose(2, 3)
        q = torch.randn(1, new, 2, 64, generator=s.g).bfloat16()
        out, lse = _attend(s, q, 0.125)
        if new > 1:
            s.cache, s.scales = (s.cache * s.scales.double()[..., None]).bfloat16(), None
        _check(s, q, out, lse, 0.125)


@pytest.mark.parametrize("e4m3", [False, True])
def test_no_new_tokens_and_outputs_over_q(e4m3):
    s = Setting([40, 9], 2, 64, 16, e4m3, seed=1)
    out, lse = _attend(s, torch.zeros(2, 0, 4, 64, dtype=torch.bfloat16), 0.1)
    assert out.shape == (2, 0, 4, 64) and lse.shape == (2, 4, 0)
    out, lse = _attend(s, torch.zeros(0, 4, 64, dtype=torch.bfloat16), 0.1, starts=[0, 0, 0])
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    for new in (1, 100):
        q = torch.randn(2, new, 4, 64, generator=s.g).bfloat16()
        want = _attend(s, q, 0.1)
        dev = q.cuda()
        table, lengths = s.tables()
        got, _ = M.paged_attn_fwd(dev, s.dev, table, lengths, 0.1, scales=s.dev_scales, out=dev)
        assert got.data_ptr() == dev.data_ptr() and torch.equal(got.cpu(), want[0])


@pytest.mark.parametrize("new", [1, 90])
def test_the_interpreters_path_gives_the_same(monkeypatch, new):
    """A call that the compiled host module leaves to Python."""
    s = Setting([140, 95], 2, 64, 16, True, seed=3)
    q = torch.randn(2, new, 4, 64, generator=s.g).bfloat16()
    k = torch.randn(2, 3, 2, 64, generator=s.g).bfloat16().cuda()
    table, lengths = s.tables()
    M.paged_cache_write(k, k, s.dev, table, lengths, scales=s.dev_scales)
    want, want_read = _attend(s, q, 0.1), M.paged_cache_read(s.dev, table, lengths, 150, scales=s.dev_scales)
    codes = s.dev.view(torch.uint8).clone()

    class Declines:
        def __getattr__(self, name):
            return lambda *args: None

    monkeypatch.setattr(N, "host", Declines())
    M.paged_cache_write(k, k, s.dev, table, lengths, scales=s.dev_scales)
    assert torch.equal(s.dev.view(torch.uint8), codes)
    got, got_read = _attend(s, q, 0.1), M.paged_cache_read(s.dev, table, lengths, 150, scales=s.dev_scales)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got_read, want_read)


def test_a_captured_packed_step_follows_its_starts():
    """Long chunks and single tokens in one captured call, replayed with other shares of the same packed rows."""
    s = Setting([150, 260, 90], 1, 64, 16, False, seed=23)
    table, lengths = s.tables()
    T, starts = 140, torch.zeros(4, dtype=torch.int32).cuda()
    q = torch.randn(T, 4, 64, generator=s.g).bfloat16()
    dev, out, lse = q.cuda(), torch.zeros(T, 4, 64, dtype=torch.bfloat16).cuda(), torch.zeros(4, T).cuda()
    graphed = M.GraphedStep(lambda: M.paged_attn_fwd(dev, s.dev, table, lengths, 0.1, starts=starts, out=out, lse=lse))
    for new in ([130, 1, 9], [1, 130, 2], [50, 0, 90], [0, 0, 0], [1, 1, 1], [140, 0, 0]):
        out.fill_(7.0)
        starts.copy_(torch.tensor(_starts(new), dtype=torch.int32))
        graphed.replay()
        torch.cuda.synchronize()
        _check(s, q, out.cpu(), lse.cpu(), 0.1, starts=_starts(new))
        assert (out[sum(new):] == 7).all()


@pytest.mark.parametrize("new,Hq", [(1, 4), (16, 1), (12, 2), (20, 2), (130, 1)])
def test_infinite_values_that_every_row_sees(new, Hq):
    """Weights are all above 2^-60 here: a value of infinity is one in every row's result, whatever sign, and no NaN."""
    s = Setting([200], 1, 64, 16, False, seed=new)
    q = torch.randn(1, new, Hq, 64, generator=s.g).bfloat16()
    for key, column, what in ((3, 5, math.inf), (70, 6, -math.inf), (199, 7, math.inf)):
        page, slot = s.table[0][key // 16], key % 16
        s.cache[1, page, slot, 0, column] = what
        s.dev[1, page, slot, 0, column] = what
    out, lse = _attend(s, q, 0.125, causal=False)
    _check(s, q, out, lse, 0.125, causal=False)
    for column, what in ((5, math.inf), (6, -math.inf), (7, math.inf)):
        assert (out[0, :, :, column] == what).all()


def test_numbers_that_no_c_int_holds():
    s = Setting([40], 1, 64, 16, False)
    table, lengths = s.tables()
    for rows, begin in ((5, 2 ** 32), (2 ** 32 + 5, 0), (5, 1.5), (None, 0)):
        with pytest.raises(RuntimeError, match="invalid"):
            M.paged_cache_read(s.dev, table, lengths, rows, begin)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16).cuda()
    starts = torch.tensor([0, 1], dtype=torch.int32).cuda()
    for most in (2 ** 63, -1, "1"):
        with pytest.raises(RuntimeError, match="invalid"):
            M.paged_attn_fwd(q, s.dev, table, lengths, 0.1, starts=starts, most_new=most)
    assert (M.paged_cache_read(s.dev, table, lengths, 3, 2 ** 31 - 4) == 0).all()
    for most in (2 ** 32 + 1, 1):
        M.paged_attn_fwd(q, s.dev, table, lengths, 0.1, starts=starts, most_new=most)


@pytest.mark.parametrize("new,Hq", [(1, 4), (12, 4), (20, 8), (300, 2)])
def test_out_may_take_the_place_of_q(new, Hq):
    s = Setting([1500, 320, 700], 2, 128, 16, True, seed=new)
    q = torch.randn(3, new, Hq, 128, generator=s.g).bfloat16()
    want = _attend(s, q, 0.1)
    table, lengths = s.tables()
    mine = q.cuda()
    out, lse = M.paged_attn_fwd(mine, s.dev, table, lengths, 0.1, scales=s.dev_scales, out=mine)
    assert out.data_ptr() == mine.data_ptr()
    assert torch.equal(out.cpu(), want[0]) and torch.equal(lse.cpu(), want[1])
    starts = torch.tensor([0, new, 2 * new, 3 * new], dtype=torch.int32).cuda()
    mine = q.reshape(3 * new, Hq, 128).cuda()
    packed, lse = M.paged_attn_fwd(mine.clone(), s.dev, table, lengths, 0.1, scales=s.dev_scales, starts=starts)
    M.paged_attn_fwd(mine, s.dev, table, lengths, 0.1, scales=s.dev_scales, starts=starts, out=mine)
    assert torch.equal(mine, packed)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [1, 3, 130])
def test_a_rank_that_holds_no_page(e4m3, new):
    """Sequences with tokens, all of whose pages are elsewhere: no row sees a key, in a cache of no pages too."""
    for pages in (0, 3):
        cache, scales = M.paged_cache(pages, 16, 2, 64, E4M3 if e4m3 else torch.bfloat16)
        table = torch.full((2, 20), pages, dtype=torch.int32).cuda()
        table[1] = -1
        lengths = torch.tensor([300, 150], dtype=torch.int32).cuda()
        q = torch.ones(2, new, 4, 64, dtype=torch.bfloat16).cuda()
        M.paged_cache_write(q[:, :, :2], q[:, :, :2], cache, table, lengths, scales=scales)
        out, lse = M.paged_attn_fwd(q, cache, table, lengths, 0.1, scales=scales)
        assert (out == 0).all() and (lse == -math.inf).all()
        assert (M.paged_cache_read(cache, table, lengths, 310, scales=scales) == 0).all()
