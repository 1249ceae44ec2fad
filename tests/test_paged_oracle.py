"""The 64-bit restatement of the paged cache against things that are not it: torch's own conversion to e4m3, attention of
torch over the gathered rows, and the restatement of dense block attention."""
import math

import pytest
import torch

import oracle as O
from oracle import paged_oracle as P


def test_quantised_rows_are_torchs_conversion_of_the_scaled_row():
    g = torch.Generator().manual_seed(1)
    for exponent in (-130, -60, -9, 0, 7, 100, 118):
        x = (torch.randn(64, generator=g).double() * 2.0 ** exponent).bfloat16()
        codes, scale = P.quantise_row(x)
        assert math.frexp(scale)[0] == 0.5 and scale >= 2.0 ** -126
        top = x.double().abs().max().item()
        assert top <= 448 * scale and (top > 224 * scale or scale == 2.0 ** -126)
        want = (x.double() / scale).float().to(torch.float8_e4m3fn).double()
        assert torch.equal(codes, want)
        normal = codes.abs() >= 2.0 ** -6
        assert ((codes * scale - x.double()).abs()[normal] <= 2.0 ** -4 * x.double().abs()[normal]).all()
        assert torch.equal((codes * scale).bfloat16().double(), codes * scale) or exponent < -100
    codes, scale = P.quantise_row(torch.tensor([448.0, -1.0]))
    assert scale == 1.0 and codes.tolist() == [448.0, -1.0]
    assert P.quantise_row(torch.tensor([450.0, 1.0]))[1] == 2.0
    assert P.quantise_row(torch.zeros(4))[1] == 1.0
    assert math.isnan(P.quantise_row(torch.tensor([1.0, math.inf]))[1])


@pytest.mark.parametrize("causal", [False, True])
def test_attention_over_pages_is_attention_over_the_gathered_rows(causal):
    g = torch.Generator().manual_seed(2)
    cache = torch.randn(2, 5, 16, 2, 8, generator=g).bfloat16()
    table, lengths = [[3, 0], [4, 1]], [20, 32]
    q = torch.randn(2, 3, 4, 8, generator=g).bfloat16()
    chunk = P.paged_read(cache, table, lengths, 32)
    for b, (out, lse, _, _) in enumerate(P.paged_attention(q, cache, table, lengths, 0.3, causal)):
        kv = chunk[:, b:b + 1, :lengths[b]]
        want, want_lse = O.block_attention(q[b:b + 1].double(), kv[0], kv[1], 0.3, causal=causal)
        assert (out - want[0]).abs().max() < 1e-6 and (lse - want_lse[0]).abs().max() < 1e-6


def test_written_rows_are_read_back():
    g = torch.Generator().manual_seed(3)
    k, v = torch.randn(5, 2, 8, generator=g).bfloat16(), torch.randn(5, 2, 8, generator=g).bfloat16()
    table, lengths, starts = [[1, 2], [0, -1]], [18, 2], [0, 3, 5]
    cache = torch.zeros(2, 3, 16, 2, 8, dtype=torch.bfloat16)
    P.paged_write(k, v, cache, table, lengths, starts=starts)
    got = P.paged_read(cache, table, lengths, 3, begin=15)
    assert torch.equal(got[0, 0], k[:3].double()) and torch.equal(got[1, 0], v[:3].double()) and (got[:, 1] == 0).all()
    assert torch.equal(P.paged_read(cache, table, lengths, 2)[0, 1], k[3:].double())
    assert (cache != 0).sum() == 2 * 5 * 2 * 8
