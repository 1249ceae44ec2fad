"""Sequences with many new tokens over a paged cache, in every width of the long-chunk kernel and with keys that several workgroups share,
against the 64-bit restatement (oracle/paged_oracle.py)."""
import math

import pytest
import torch

import mercury_artifact_amd as M
from oracle import paged_oracle as P
from test_gpu_paged import Setting, _attend, _check, _starts

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
WIDTHS = [16, 64, 72, 80, 88, 96, 104, 112, 120, 128]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,e4m3", [(D, False) for D in WIDTHS] + [(D, True) for D in WIDTHS if D % 16 == 0])
def test_every_width(D, e4m3, causal):
    """Sequences of two, three and five tiles of 64 keys, 140 rows each: one whole wavefront's rows and more, one past the end."""
    print(f"D {D} e4m3 {e4m3} causal {causal}", flush=True)
    s = Setting([128, 129, 300, 71], 1, D, 16, e4m3, seed=D)
    q = torch.randn(4, 70, 2, D, generator=s.g).bfloat16()
    out, lse = _attend(s, q, D ** -0.5, causal)
    _check(s, q, out, lse, D ** -0.5, causal)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D,lengths,new,Hq,Hkv", [
    (128, [1100], 66, 1, 1),                 # one item, its keys in several pieces
    (96, [1100], 66, 1, 1),
    (80, [1500], 35, 4, 2),
    (64, [2100], 40, 2, 1),
    (128, [1300, 200], 150, 2, 1),           # two tiles of rows, a short sequence that is not cut beside it
    (96, [1024, 1025, 700], 100, 1, 1),
])
def test_keys_that_several_workgroups_share(D, lengths, new, Hq, Hkv, e4m3):
    print(f"D {D} lengths {lengths} new {new} H{Hq}/{Hkv} e4m3 {e4m3}", flush=True)
    s = Setting(lengths, Hkv, D, 16, e4m3, seed=new)
    q = torch.randn(len(lengths), new, Hq, D, generator=s.g).bfloat16()
    for causal in (True, False):
        out, lse = _attend(s, q, D ** -0.5, causal)
        _check(s, q, out, lse, D ** -0.5, causal)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D", [80, 96, 128])
def test_packed_prompts_beside_single_tokens(D, e4m3):
    s = Setting([1200, 40, 333, 9], 2, D, 16, e4m3, seed=D)
    new = [90, 1, 1, 9]
    starts = _starts(new)
    q = torch.randn(starts[-1], 4, D, generator=s.g).bfloat16()
    for most in (90, 1, None):
        out, lse = _attend(s, q, D ** -0.5, starts=starts, most_new=most)
        _check(s, q, out, lse, D ** -0.5, starts=starts)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("D", [80, 128])
def test_pages_that_are_not_here(D, e4m3):
    """Every third page elsewhere, among keys that several workgroups share; the first and the last pages too."""
    s = Setting([1100, 150], 1, D, 16, e4m3, seed=D)
    q = torch.randn(2, 70, 1, D, generator=s.g).bfloat16()
    s.table = [[-1 if i % 3 == 0 or i > 65 else e for i, e in enumerate(row)] for row in s.table]
    out, lse = _attend(s, q, D ** -0.5)
    _check(s, q, out, lse, D ** -0.5)


@pytest.mark.parametrize("D", [80, 96, 104])
def test_a_value_that_is_no_number_in_the_other_widths(D):
    s = Setting([400], 1, D, 16, False, seed=D)
    new, at = 100, 350
    q = torch.randn(1, new, 1, D, generator=s.g).bfloat16()
    page, slot = s.table[0][at // 16], at % 16
    for x in (s.cache, s.dev):
        x[1, page, slot, 0, 3], x[1, page, slot, 0, D - 1] = math.nan, -math.inf
    out, lse = _attend(s, q, 0.1)
    _check(s, q, out, lse, 0.1)
    sees = torch.arange(new) + 300 >= at
    assert torch.isnan(out[0, sees, 0, 3]).all() and (out[0, sees, 0, D - 1] == -math.inf).all() and torch.isfinite(out[0, ~sees]).all()


@pytest.mark.parametrize("D", [80, 128])
def test_scattered_pages_that_no_cache_holds(D):
    """Short items, the first tiles of which come from all over gigabytes: what the loop's first products read has to have arrived."""
    B, page, Hkv, Hq, new = 24, 16, 8, 16, 40
    cache, _ = M.paged_cache(60000, page, Hkv, D)
    g = torch.Generator().manual_seed(D)
    lengths = [65 + (37 * b) % 128 for b in range(B)]
    table = torch.randperm(60000, generator=g)[:B * 12].view(B, 12).int()
    dev = table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
    k, v = (torch.randn(B, 192, Hkv, D, generator=g).bfloat16() for _ in range(2))
    starts = _starts(lengths)
    packed = [torch.cat([x[b, :n] for b, n in enumerate(lengths)]).cuda() for x in (k, v)]
    M.paged_cache_write(*packed, cache, *dev, starts=torch.tensor(starts, dtype=torch.int32).cuda())
    q = torch.randn(B, new, Hq, D, generator=g).bfloat16()
    other = torch.empty(1 << 28, device="cuda")
    dense = torch.stack([k, v]).view(2, B * 12, page, Hkv, D)
    want = P.paged_attention(q, dense, torch.arange(B * 12).view(B, 12).tolist(), lengths, D ** -0.5)
    for i in range(3):
        other.fill_(i)                     # (1 GiB: nothing of the cache stays in the chip's)
        out, lse = M.paged_attn_fwd(q.cuda(), cache, *dev, D ** -0.5)
        out, lse = out.cpu().double(), lse.cpu().double()
        for b, (o, l, o_off, l_off) in enumerate(want):
            assert ((out[b] - o).abs() <= o_off).all() and ((lse[b] - l).abs() <= l_off).all(), b


def test_e4m3_keys_and_values_past_four_gigabytes():
    """Both halves written and read at places of more than 32 bits."""
    pages, page, Hkv, D = (1 << 32) // (16 * 8 * 128) + 40, 16, 8, 128
    cache, scales = M.paged_cache(pages, page, Hkv, D, E4M3)
    table = torch.tensor([[pages - 1, 0, pages // 2 + 1]], dtype=torch.int32).cuda()
    lengths = torch.tensor([41], dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(1, 41, Hkv, D, generator=g).bfloat16(), torch.randn(1, 41, Hkv, D, generator=g).bfloat16()
    M.paged_cache_write(k.cuda(), v.cuda(), cache, table, lengths, scales=scales)
    read = M.paged_cache_read(cache, table, lengths, 41, scales=scales).cpu()
    want = torch.zeros(2, 3, page, Hkv, D, dtype=torch.float64)
    want_scales = torch.ones(2, 3, page, Hkv)
    P.paged_write(k, v, want, [[2, 0, 1]], [41], want_scales)
    assert torch.equal(read, P.paged_read(want, [[2, 0, 1]], [41], 41, 0, want_scales).bfloat16())
    q = torch.randn(1, 3, 8, D, generator=g).bfloat16()
    out, lse = M.paged_attn_fwd(q.cuda(), cache, table, lengths, 0.1, scales=scales)
    for o, l, o_off, l_off in P.paged_attention(q, want, [[2, 0, 1]], [41], 0.1, True, want_scales):
        assert ((out[0].cpu().double() - o).abs() <= o_off).all() and ((lse[0].cpu().double() - l).abs() <= l_off).all()
