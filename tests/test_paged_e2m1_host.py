"""The paged cache in four bits without a GPU: its 64-bit restatement, and what the C entries refuse of it."""
import math

import pytest
import torch

import mercury_artifact_amd as M
from mercury_artifact_amd import _native as N
from oracle import paged_oracle as P

E2M1, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
OK, EINVAL, EHEADDIM, EALIGN, EUNSUPPORTED = 0, -1, -3, -4, -6
AT = 0x10000


def test_a_block_is_the_nearest_of_all_codes():
    """Against the bit layout: one bit of sign, two of an exponent with bias 1, one of a fraction."""
    def value(code):
        sign, e, f = code >> 3, code >> 1 & 3, code & 1
        return (-1) ** sign * (f / 2 if e == 0 else (1 + f / 2) * 2 ** (e - 1))

    assert [value(c) for c in range(8)] == list(P.E2M1)
    g = torch.Generator().manual_seed(1)
    for exponent in (-128, -126, -60, 0, 5, 100, 126):
        x = (torch.randn(32, generator=g).double() * 2.0 ** exponent).bfloat16()
        codes, byte = P.quantise_block(x)
        scale = 2.0 ** (byte - 127)
        top = x.double().abs().max().item()
        assert 1 <= byte <= 252 and (top <= 6 * scale or byte == 252) and (top > 3 * scale or byte == 1)
        for c, v in zip(codes, x.tolist()):
            assert abs(value(c) * scale - v) <= min(abs(value(d) * scale - v) for d in range(16)) and (value(c) < 0) <= (v < 0)
    assert P.quantise_block(torch.zeros(32)) == ([0] * 32, 127)
    assert P.quantise_block(torch.tensor([1.0, math.inf])) == ([0, 0], 255)
    ties = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0])
    assert P.quantise_block(ties) == ([7, 0, 2, 2, 4, 4, 6, 6, 8, 14], 127)
    assert P.quantise_block(torch.tensor([6.03125]))[1] == 128


def test_bytes_hold_what_they_say():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(96, generator=g).bfloat16()
    codes, scales = P.quantise_e2m1(x)
    assert codes.shape == (48,) and scales.shape == (3,)
    values = P.e2m1_values(codes, torch.cat([scales, torch.tensor([255], dtype=torch.uint8)]))
    assert values.shape == (96,) and ((values - x.double()).abs() <= x.abs().max().double() / 3).all()
    assert values[0].item() == (-1) ** (codes[0].item() >> 3 & 1) * P.E2M1[codes[0].item() & 7] * 2.0 ** (scales[0].item() - 127)
    assert values[65].item() == (-1) ** (codes[32].item() >> 7) * P.E2M1[codes[32].item() >> 4 & 7] * 2.0 ** (scales[2].item() - 127)


def test_the_cache_that_is_made():
    cache, scales = M.paged_cache(5, 16, 3, 96, E2M1, device="cpu")
    assert cache.shape == (2, 5, 16, 3, 48) and cache.dtype == E2M1 and cache.stride(2) == 48
    assert scales.shape == (2, 5, 16, 3, 4) and scales.dtype == E8M0 and scales.stride(2) == 4
    with pytest.raises(RuntimeError, match="multiple of 32"):
        M.paged_cache(5, 16, 3, 80, E2M1, device="cpu")
    x = torch.zeros(1, 1, 3, 96, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU only"):
        M.paged_cache_write(x, x, cache, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), scales=scales)


def _strides(Hkv, D, page):
    return (Hkv * page * D // 2, D // 2, page * D // 2, Hkv * page, 1, page)


def _read(ks=AT, vs=AT, D=64, cache=None, rows=8):
    o = (2 * rows * 2 * 128, rows * 2 * 128, 2 * 128, 128)
    return N.lib().mhip_paged_cache_read(AT, AT, ks, vs, AT, AT, AT, 2, 0, rows, 2, D, 9, 16, 4, 4, *(_strides(2, D, 16) if cache is None else cache),
                                         *o, N.MHIP_E2M1, None)


def test_what_the_entries_refuse():
    for D in (0, 16, 48, 80, 112, 160):
        assert _read(D=D, cache=(4096, 64, 1024, 32, 1, 16)) == EHEADDIM
    assert _read(ks=None) == EINVAL and _read(vs=None) == EINVAL
    assert _read(ks=AT + 2) == EALIGN
    assert _read(cache=(1024, 40, 512, 32, 1, 16)) == EALIGN
    assert _read(cache=(1024, 16, 512, 32, 1, 16)) == EUNSUPPORTED               # rows over one another
    assert _read(cache=(1 << 40, 1 << 26, 32, 32, 1, 16)) == EUNSUPPORTED        # 16 rows past what an offset reaches
    assert _read(rows=0) == OK
