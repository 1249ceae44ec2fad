"""The paged K/V cache in four bits against its 64-bit restatement (oracle/paged_oracle.py, whose docstring derives how far
attention may be off: a code times its scale is exact in bf16, so the bound is that of a bf16 cache).  Rows that hold no key, and
scales of columns that are not there, are NaN here."""
import math

import pytest
import torch

import mercury_artifact_amd as M
from mercury_artifact_amd import _native as N
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

E2M1, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


class Setting:
    """A cache whose sequences' rows hold any codes, with scales around 2^-2 (`spread` binades apart), on the CPU and on the GPU."""

    def __init__(self, lengths, Hkv, D, page, seed=0, spare=2, width=None, token_major=False, spread=3, gain=0):
        g = self.g = torch.Generator().manual_seed(seed)
        self.lengths, self.page, self.D, self.Hkv = list(lengths), page, D, Hkv
        counts = [-(-n // page) for n in lengths]
        pages = sum(counts) + spare
        order, at = torch.randperm(pages, generator=g).tolist(), 0
        width = max([*counts, 1]) if width is None else width
        self.table = []
        for c in counts:
            self.table.append(order[at:at + c] + [-1] * (width - c))
            at += c
        self.codes = torch.randint(0, 256, (2, pages, page, Hkv, D // 2), generator=g, dtype=torch.uint8)
        self.scales = torch.full((2, pages, page, Hkv, 4), 255, dtype=torch.uint8)
        real = torch.randint(125 + gain - spread // 2, 126 + gain + spread // 2, (2, pages, page, Hkv, D // 32), generator=g, dtype=torch.uint8)
        for b, n in enumerate(lengths):
            for j in range(n):
                p, s = self.table[b][j // page], j % page
                self.scales[:, p, s, :, :D // 32] = real[:, p, s]
        order5 = (lambda t: t.cuda()) if token_major else (lambda t: t.transpose(2, 3).contiguous().cuda().transpose(2, 3))
        self.dev, self.dev_scales = order5(self.codes).view(E2M1), order5(self.scales).view(E8M0)

    def tables(self):
        return torch.tensor(self.table, dtype=torch.int32).view(len(self.lengths), -1).cuda(), torch.tensor(self.lengths, dtype=torch.int32).cuda()

    def bytes(self):
        return self.dev.view(torch.uint8).cpu(), self.dev_scales.view(torch.uint8).cpu()


def _starts(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return s


def _ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32).cuda()


def _attend(s, q, scale, causal=True, starts=None, **kw):
    table, lengths = s.tables()
    out, lse = M.paged_attn_fwd(q.cuda(), s.dev, table, lengths, scale, causal=causal, scales=s.dev_scales, starts=_ints(starts), **kw)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def _check(s, q, out, lse, scale, causal=True, starts=None):
    values = P.e2m1_values(s.codes, s.scales)
    want = P.paged_attention(q, values, s.table, s.lengths, scale, causal, None, starts)
    # Codes are zero one time in eight, so that a result may be made of keys whose weights are nothing in 32 bits: each of the S weights,
    # relative to the largest, is off by 2^-126 at most where it is below the least normal number.
    least = max(s.lengths) * 2.0 ** -126 * values.nan_to_num().abs().max()
    for b, (o, l, o_off, l_off) in enumerate(want):
        got = P.tokens_of(b, out, starts).double()
        got_l = (lse[b] if starts is None else lse[:, starts[b]:starts[b + 1]]).double()
        assert torch.equal(torch.isnan(got), torch.isnan(o)), b
        assert torch.equal(got_l == -math.inf, l == -math.inf), b
        assert torch.equal(torch.isnan(got_l), torch.isnan(l)), b
        assert ((got - o).abs() <= o_off + least)[torch.isfinite(o)].all(), (b, ((got - o).abs() - o_off).max())
        seen = torch.isfinite(l)
        assert ((got_l - l).abs() <= l_off)[seen].all(), (b, ((got_l - l).abs() - l_off)[seen].max())


@pytest.mark.parametrize("lengths,new,Hq,Hkv,D,page,causal", [
    ([1], 1, 1, 1, 128, 16, True),
    ([0, 1, 15, 16, 17, 31, 32, 33], 1, 4, 2, 128, 16, True),
    ([127, 128, 129, 300, 1, 0], 1, 8, 2, 64, 16, True),
    ([500, 3, 1029], 1, 5, 5, 96, 32, True),
    ([257, 64, 1], 1, 32, 2, 128, 48, False),
    ([700], 1, 7, 1, 32, 64, True),
    ([40, 5, 129], 5, 4, 2, 128, 16, True),
    ([40, 5, 129], 5, 4, 2, 64, 16, False),
    ([90, 33], 4, 16, 2, 64, 16, True),             # 32 rows
    ([90, 33], 4, 17, 1, 32, 16, True),             # 68 rows, two tiles of them
    ([260, 131], 9, 6, 1, 96, 16, True),            # 54 rows
    ([2, 3, 50], 6, 2, 2, 128, 16, True),           # more new tokens than keys
    ([150, 130], 130, 2, 2, 128, 16, True),
    ([320], 77, 6, 2, 32, 256, True),
    ([200, 333], 150, 4, 1, 96, 32, False),
    ([1500], 300, 2, 1, 64, 16, True),
])
def test_attention(lengths, new, Hq, Hkv, D, page, causal):
    print(f"case {lengths} new {new} H{Hq}/{Hkv} D{D} page {page} causal {causal}", flush=True)
    s = Setting(lengths, Hkv, D, page, seed=len(lengths) + new)
    q = torch.randn(len(lengths), new, Hq, D, generator=s.g).bfloat16()
    out, lse = _attend(s, q, D ** -0.5, causal)
    _check(s, q, out, lse, D ** -0.5, causal)


@pytest.mark.parametrize("most", [None, 1, 3, 40, 1000])
@pytest.mark.parametrize("lengths,new,Hq,Hkv,D", [
    ([40, 300, 17, 9, 0, 64], [1, 0, 3, 9, 0, 40], 4, 2, 128),
    ([500, 130, 260, 5], [1, 130, 1, 5], 4, 1, 64),
    ([33], [0], 2, 2, 64),
])
def test_attention_packed(lengths, new, Hq, Hkv, D, most):
    s = Setting(lengths, Hkv, D, 16, seed=5, width=40)
    starts = [2 + x for x in _starts(new)]
    T = starts[-1] + 3
    q = torch.randn(T, Hq, D, generator=s.g).bfloat16()
    q[:2], q[T - 3:] = math.nan, math.nan
    out, lse = torch.full((T, Hq, D), 7.0, dtype=torch.bfloat16).cuda(), torch.full((Hq, T), 7.0).cuda()
    out, lse = _attend(s, q, D ** -0.5, starts=starts, most_new=most, out=out, lse=lse)
    _check(s, q, out, lse, D ** -0.5, starts=starts)
    assert (out[:2] == 7).all() and (out[T - 3:] == 7).all() and (lse[:, :2] == 7).all() and (lse[:, T - 3:] == 7).all()


def test_many_sequences():
    lengths = [(37 * b) % 61 for b in range(150)]
    lengths[77] = 2000
    s = Setting(lengths, 1, 64, 16, seed=9)
    q = torch.randn(150, 1, 3, 64, generator=s.g).bfloat16()
    out, lse = _attend(s, q, 0.125)
    _check(s, q, out, lse, 0.125)


@pytest.mark.parametrize("new", [1, 3, 100])
def test_pages_that_are_not_here(new):
    s = Setting([210, 5, 400], 2, 128, 16, seed=11)
    q = torch.randn(3, new, 4, 128, generator=s.g).bfloat16()
    whole, pages = s.table, s.codes.shape[1]
    for rank, nobody in ((0, -1), (1, pages), (1, 2 ** 31 - 1), (0, -2 ** 31)):
        s.table = [[e if i % 2 == rank else nobody for i, e in enumerate(row)] for row in whole]
        out, lse = _attend(s, q, 128 ** -0.5)
        _check(s, q, out, lse, 128 ** -0.5)


@pytest.mark.parametrize("new", [1, 6, 20, 90])
@pytest.mark.parametrize("half", [0, 1])
def test_a_block_that_is_no_number_reaches_the_rows_that_see_it_alone(new, half):
    """A key's block makes all of its rows' results NaN, a value's those 32 columns, with whatever codes, however small its weight."""
    s = Setting([230], 1, 128, 16, seed=3)
    q = torch.randn(1, new, 2, 128, generator=s.g).bfloat16()
    at = 230 - new + new // 2
    page, slot = s.table[0][at // 16], at % 16
    s.scales[half, page, slot, 0, 2] = 255
    s.dev_scales.view(torch.uint8)[half, page, slot, 0, 2] = 255
    if half:                                             # the key's weight is nothing in 32 bits
        s.codes[0, page, slot], s.scales[0, page, slot] = 0x77, 127 + 8
        s.dev.view(torch.uint8)[0, page, slot], s.dev_scales.view(torch.uint8)[0, page, slot] = 0x77, 127 + 8
        q = -q.abs()
    out, lse = _attend(s, q, 0.1)
    _check(s, q, out, lse, 0.1)
    seen = torch.isnan(out[0, new // 2:])
    assert (seen[..., 64:96] if half else seen).all() and not torch.isnan(out[0, :new // 2]).any()
    assert not half or not (seen[..., :64].any() or seen[..., 96:].any())


@pytest.mark.parametrize("new", [1, 90])
def test_large_scores_and_scales_far_apart(new):
    s = Setting([600], 1, 64, 16, seed=6, spread=12, gain=2)
    q = (torch.randn(1, new, 4, 64, generator=s.g) * 3).bfloat16()
    out, lse = _attend(s, q, 1.0)
    _check(s, q, out, lse, 1.0)


@pytest.mark.parametrize("Hq,new", [(80, 1), (128, 1), (65, 1), (64, 1), (33, 2)])
def test_many_query_heads_on_one_key_head(Hq, new):
    s = Setting([200, 1, 77], 1, 64, 16, seed=Hq)
    q = torch.randn(3, new, Hq, 64, generator=s.g).bfloat16()
    out, lse = _attend(s, q, 0.125)
    _check(s, q, out, lse, 0.125)
    starts = [0, new, 2 * new, 3 * new]
    packed = q.reshape(3 * new, Hq, 64)
    out, lse = _attend(s, packed, 0.125, starts=starts, most_new=new)
    _check(s, packed, out, lse, 0.125, starts=starts)


def test_strides_and_orders():
    """A cache and scales in the order of their tokens, as slices of wider tensors."""
    s = Setting([100, 37], 2, 64, 16, seed=8, token_major=True)
    table, lengths = s.tables()
    wide = torch.full((2, s.codes.shape[1], 16, 3, 64), 0x55, dtype=torch.uint8).cuda()
    wide[:, :, :, 1:, 16:48] = s.codes.cuda()
    wide_scales = torch.full((2, s.codes.shape[1], 17, 2, 12), 255, dtype=torch.uint8).cuda()
    wide_scales[:, :, 1:, :, 4:8] = s.scales.cuda()
    s.dev, s.dev_scales = wide.view(E2M1)[:, :, :, 1:, 16:48], wide_scales.view(E8M0)[:, :, 1:, :, 4:8]
    for new in (3, 80):
        q = torch.randn(2, new, 4, 64, generator=s.g).bfloat16()
        out, lse = _attend(s, q, 0.1)
        _check(s, q, out, lse, 0.1)
    read = M.paged_cache_read(s.dev, table, lengths, 100, scales=s.dev_scales)
    assert torch.equal(read.cpu(), P.paged_read(P.e2m1_values(s.codes, s.scales), s.table, s.lengths, 100).bfloat16())
    k = torch.randn(2, 5, 2, 64, generator=s.g).bfloat16()
    before = wide.clone(), wide_scales.clone()
    M.paged_cache_write(k.cuda(), k.cuda(), s.dev, table, lengths, scales=s.dev_scales)
    P.paged_write_e2m1(k, k, s.codes, s.scales, s.table, s.lengths)
    assert torch.equal(wide[:, :, :, 1:, 16:48].cpu(), s.codes) and torch.equal(wide_scales[:, :, 1:, :, 4:8].cpu(), s.scales)
    for now, was in zip((wide, wide_scales), before):
        view = now.clone()
        if now is wide:
            view[:, :, :, 1:, 16:48] = was[:, :, :, 1:, 16:48]
        else:
            view[:, :, 1:, :, 4:8] = was[:, :, 1:, :, 4:8]
        assert torch.equal(view, was)


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("packed", [False, True])
def test_written_and_read_back(D, packed):
    """Byte for byte; rows beside the new ones, and scales of columns that are not there, are left as they were."""
    s = Setting([50, 7, 130, 0, 33], 3, D, 16, seed=D, width=10)
    new = [5, 7, 40, 0, 1] if packed else [7] * 5
    starts = [1 + x for x in _starts(new)] if packed else None
    shape = (starts[-1] + 2,) if packed else (5, 7)
    k = (torch.randn(*shape, 3, D, generator=s.g) * torch.exp2(torch.randint(-20, 20, (*shape, 3, 1), generator=s.g))).bfloat16()
    # halves of a code's step between the codes: ties
    v = (torch.randint(-28, 29, (*shape, 3, D), generator=s.g) / 4 * torch.exp2(torch.randint(-3, 3, (*shape, 3, 1), generator=s.g))).bfloat16()
    at = (2,) if packed else (2, 1)
    k[at], v[at] = 0.0, v[at] * 2.0 ** -126                # zeros, and blocks below the least scale
    at = (4,) if packed else (0, 3)
    k[at][1, 3], k[at][2] = math.nan, 3.3e38               # one block that is no number; values past the largest that is held
    k[at][0, 5], v[at][0, 1], v[at][1] = -math.inf, math.inf, -0.0
    s.table[2][7] = -1                                     # a page that is not here: its rows are dropped
    table, lengths = s.tables()
    P.paged_write_e2m1(k, v, s.codes, s.scales, s.table, s.lengths, starts)
    M.paged_cache_write(k.cuda(), v.cuda(), s.dev, table, lengths, scales=s.dev_scales, starts=_ints(starts))
    got, got_scales = s.bytes()
    assert torch.equal(got, s.codes) and torch.equal(got_scales, s.scales)
    values = P.e2m1_values(s.codes, s.scales)
    for begin, rows in ((0, 140), (20, 60), (129, 1), (0, 0), (200, 3)):
        read = M.paged_cache_read(s.dev, table, lengths, rows, begin=begin, scales=s.dev_scales)
        plain = P.paged_read(values, s.table, s.lengths, rows, begin).bfloat16()
        assert torch.equal(torch.nan_to_num(read.cpu(), nan=1e9), torch.nan_to_num(plain, nan=1e9))


@pytest.mark.parametrize("new", [1, 80])
def test_rows_past_four_gigabytes(new):
    pages, page, Hkv, D = (2 << 32) // (16 * 8 * 64) + 50, 16, 8, 128
    cache, scales = M.paged_cache(pages, page, Hkv, D, E2M1)
    assert cache.stride(0) > 1 << 32
    length = 40 + new
    table = torch.tensor([[pages - 1, 0, pages // 2 + 1, pages - 2, 7, pages - 9, 8, 9]], dtype=torch.int32).cuda()
    lengths = torch.tensor([length], dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(1, length, Hkv, D, generator=g).bfloat16() for _ in range(2))
    M.paged_cache_write(k.cuda(), v.cuda(), cache, table, lengths, scales=scales)
    read = M.paged_cache_read(cache, table, lengths, length, scales=scales).cpu()
    for half, x in enumerate((k, v)):
        top = x.float().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(1, length, Hkv, 4, 32).flatten(-2)
        assert ((read[half].float() - x.float()).abs() <= top / 3).all()       # half a step of at most 2 of 6, whose scale is twice the least
    q = torch.randn(1, new, 8, D, generator=g).bfloat16()
    out, lse = M.paged_attn_fwd(q.cuda(), cache, table, lengths, 0.1, scales=scales)
    dense = torch.zeros(2, 8, 16, Hkv, D, dtype=torch.bfloat16)
    dense.view(2, 128, Hkv, D)[:, :length] = read[:, 0]
    for b, (o, l, o_off, l_off) in enumerate(P.paged_attention(q, dense, [list(range(8))], [length], 0.1)):
        assert ((out[b].cpu().double() - o).abs() <= o_off).all() and ((lse[b].cpu().double() - l).abs() <= l_off).all()


def test_a_captured_step_follows_lengths_and_table():
    """Write and attend, captured once, replayed while the sequences grow; an eager call and other work between the replays."""
    s = Setting([40, 100], 2, 64, 16, seed=21, spare=12, width=12)
    table, lengths = s.tables()
    q, k, v = (torch.zeros(2, 1, h, 64, dtype=torch.bfloat16).cuda() for h in (4, 2, 2))
    out, lse = torch.empty_like(q), torch.empty(2, 4, 1).cuda()

    def step():
        M.paged_cache_write(k, v, s.dev, table, lengths, scales=s.dev_scales)
        M.paged_attn_fwd(q, s.dev, table, lengths, 0.1, scales=s.dev_scales, out=out, lse=lse)

    spare = [p for p in range(s.codes.shape[1]) if p not in sum(s.table, [])]
    graphed = M.GraphedStep(step)
    s.dev.view(torch.uint8).copy_(s.codes.cuda())                              # (the capture's own runs wrote zeros)
    s.dev_scales.view(torch.uint8).copy_(s.scales.cuda())
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
        P.paged_write_e2m1(new[1], new[2], s.codes, s.scales, s.table, s.lengths)
        _check(s, new[0], *got, 0.1)
        eager = _attend(s, new[0], 0.1)
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])


@pytest.mark.parametrize("new", [1, 90])
def test_the_interpreters_path_and_every_call_give_the_same(monkeypatch, new):
    s = Setting([140, 95], 2, 64, 16, seed=3)
    q = torch.randn(2, new, 4, 64, generator=s.g).bfloat16()
    k = torch.randn(2, 3, 2, 64, generator=s.g).bfloat16().cuda()
    table, lengths = s.tables()
    M.paged_cache_write(k, k, s.dev, table, lengths, scales=s.dev_scales)
    want, want_read, bytes_ = _attend(s, q, 0.1), M.paged_cache_read(s.dev, table, lengths, 150, scales=s.dev_scales), s.bytes()
    again = _attend(s, q, 0.1)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])

    class Declines:
        def __init__(self, host):
            self.written = host.written

        def __getattr__(self, name):
            return lambda *args: None

    monkeypatch.setattr(N, "host", Declines(N.host))
    M.paged_cache_write(k, k, s.dev, table, lengths, scales=s.dev_scales)
    assert all(torch.equal(x, y) for x, y in zip(s.bytes(), bytes_))
    got, got_read = _attend(s, q, 0.1), M.paged_cache_read(s.dev, table, lengths, 150, scales=s.dev_scales)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got_read, want_read)


def test_refusals_say_why():
    s = Setting([40], 2, 64, 16)
    table, lengths = s.tables()
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16).cuda()
    M.paged_attn_fwd(q, s.dev, table, lengths, 0.1, scales=s.dev_scales)
    wide = torch.zeros(*s.scales.shape[:-1], 6, dtype=torch.uint8).cuda().view(E8M0)
    for message, call in [
        ("scales", lambda: M.paged_attn_fwd(q, s.dev, table, lengths, 0.1)),
        ("scales", lambda: M.paged_attn_fwd(q, s.dev, table, lengths, 0.1, scales=s.dev_scales[..., :2])),
        ("scales", lambda: M.paged_attn_fwd(q, s.dev, table, lengths, 0.1, scales=s.dev_scales.view(torch.uint8))),
        ("on 4 bytes", lambda: M.paged_attn_fwd(q, s.dev, table, lengths, 0.1, scales=wide[..., :4])),
        ("aligned", lambda: M.paged_cache_read(s.dev, table, lengths, 3, scales=torch.zeros(s.scales.numel() + 4, dtype=torch.uint8).cuda()
                                               [1:-3].view(E8M0).view(s.scales.shape))),
        ("q must be", lambda: M.paged_attn_fwd(q[..., :32], s.dev, table, lengths, 0.1, scales=s.dev_scales)),
        ("head dimension", lambda: M.paged_attn_fwd(q[..., :48], s.dev[..., :24], table, lengths, 0.1, scales=s.dev_scales)),
        ("k must be", lambda: M.paged_cache_write(q, q, s.dev, table, lengths, scales=s.dev_scales)),
        ("multiple of 32", lambda: M.paged_cache(4, 16, 2, 80, E2M1)),
    ]:
        with pytest.raises(RuntimeError, match=message):
            call()
