"""What the C entries over a paged cache refuse, before anything is launched (no GPU needed; pointers are never followed)."""
import pytest

from mercury_artifact_amd import _native as N

OK, EINVAL, EDTYPE, EHEADDIM, EALIGN, EUNSUPPORTED = 0, -1, -2, -3, -4, -6
P = 0x10000


@pytest.fixture(scope="module")
def lib():
    return N.lib()


def _cache(Hkv, D, page):
    return (Hkv * page * D, D, page * D, Hkv * page, 1, page)


def _write(lib, k=P, v=P, kc=P, vc=P, ks=P, vs=P, table=P, lengths=P, starts=None, B=2, n=3, T=0, Hkv=2, D=64, pages=9, page=16, width=4,
           tokens=None, cache=None, dtype=0):
    tokens = (n * Hkv * D, Hkv * D, D) if tokens is None else tokens
    return lib.mhip_paged_cache_write(k, v, kc, vc, ks, vs, table, lengths, starts, B, n, T, Hkv, D, pages, page, width, width,
                                      *tokens, *tokens, *(_cache(Hkv, D, page) if cache is None else cache), dtype, None)


def _read(lib, kc=P, vc=P, ks=P, vs=P, table=P, lengths=P, out=P, B=2, begin=0, rows=8, Hkv=2, D=64, pages=9, page=16, width=4,
          cache=None, o=None, dtype=0):
    o = (B * rows * Hkv * D, rows * Hkv * D, Hkv * D, D) if o is None else o
    return lib.mhip_paged_cache_read(kc, vc, ks, vs, table, lengths, out, B, begin, rows, Hkv, D, pages, page, width, width,
                                     *(_cache(Hkv, D, page) if cache is None else cache), *o, dtype, None)


def _attn(lib, q=P, kc=P, vc=P, ks=P, vs=P, table=P, lengths=P, starts=None, out=P, lse=P, B=2, n=3, T=0, most=3, Hq=4, Hkv=2, D=64,
          pages=9, page=16, width=4, tokens=None, cache=None, scale=0.1, mask=1, dtype=0, ws=P):
    tokens = (n * Hq * D, Hq * D, D) if tokens is None else tokens
    return lib.mhip_paged_attn_fwd(q, kc, vc, ks, vs, table, lengths, starts, out, lse, B, n, T, most, Hq, Hkv, D, pages, page, width, width,
                                   *tokens, *(_cache(max(Hkv, 1), D, page) if cache is None else cache), *tokens, scale, mask, dtype, ws, None)


@pytest.mark.parametrize("call", [_write, _read, _attn])
def test_what_all_three_refuse(lib, call):
    for D in (0, 4, 100, 136):
        assert call(lib, D=D, cache=(4096, 256, 1024, 32, 1, 16)) == EHEADDIM
    assert call(lib, D=72, dtype=1) == EHEADDIM
    assert call(lib, dtype=2) == EDTYPE
    assert call(lib, B=-1) == EINVAL
    assert call(lib, pages=-1) == EINVAL
    assert call(lib, page=0, cache=_cache(2, 64, 16)) == EINVAL
    assert call(lib, page=8) == EUNSUPPORTED
    assert call(lib, page=24) == EUNSUPPORTED
    assert call(lib, page=1 << 20, width=1 << 11, cache=_cache(2, 64, 16)) == EUNSUPPORTED
    assert call(lib, width=-1) == EINVAL
    assert call(lib, Hkv=0) == EINVAL
    for missing in ("kc", "vc", "table", "lengths"):
        assert call(lib, **{missing: None}) == EINVAL
    assert call(lib, dtype=1, ks=None) == EINVAL
    assert call(lib, dtype=1, vs=None) == EINVAL
    assert call(lib, kc=P + 8) == EALIGN
    assert call(lib, table=P + 2) == EALIGN
    assert call(lib, dtype=1, ks=P + 2) == EALIGN
    assert call(lib, cache=(2048, 68, 1024, 32, 1, 16)) == EALIGN
    assert call(lib, cache=(2048, 0, 1024, 32, 1, 16)) == EUNSUPPORTED          # rows over one another
    assert call(lib, cache=(1 << 40, 1 << 26, 64, 32, 1, 16)) == EUNSUPPORTED    # 16 rows past what an offset reaches
    assert call(lib, B=0) == OK


def test_write_refuses(lib):
    assert _write(lib, n=-1) == EINVAL
    assert _write(lib, starts=P, T=-1) == EINVAL
    assert _write(lib, k=None) == EINVAL
    assert _write(lib, v=P + 4) == EALIGN
    assert _write(lib, tokens=(384, 132, 64)) == EALIGN
    assert _write(lib, B=1 << 16, n=1 << 16) == EUNSUPPORTED
    assert _write(lib, starts=P, T=1 << 30) == EUNSUPPORTED
    assert _write(lib, starts=P + 2, T=4) == EALIGN
    assert _write(lib, n=0) == OK
    assert _write(lib, pages=0, kc=None, vc=None) == OK


def test_read_refuses(lib):
    assert _read(lib, rows=-1) == EINVAL
    assert _read(lib, begin=-1) == EINVAL
    assert _read(lib, begin=1 << 30, rows=(1 << 30) + 1) == EINVAL
    assert _read(lib, out=None) == EINVAL
    assert _read(lib, out=P + 8) == EALIGN
    assert _read(lib, o=(1024, 512, 68, 64)) == EALIGN
    assert _read(lib, rows=1 << 29) == EUNSUPPORTED
    assert _read(lib, rows=0) == OK


def test_attention_refuses(lib):
    assert _attn(lib, Hq=5) == EINVAL
    assert _attn(lib, Hq=0) == EINVAL
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert _attn(lib, scale=scale) == EINVAL
    assert _attn(lib, mask=2) == EINVAL
    assert _attn(lib, most=-1) == EINVAL
    for missing in ("q", "out", "lse", "ws"):
        assert _attn(lib, **{missing: None}) == EINVAL
    assert _attn(lib, q=P + 8) == EALIGN
    assert _attn(lib, out=P + 8) == EALIGN
    assert _attn(lib, lse=P + 2) == EALIGN
    assert _attn(lib, ws=P + 8) == EALIGN
    assert _attn(lib, tokens=(384, 132, 64)) == EALIGN
    assert _attn(lib, starts=P, T=1 << 29) == EUNSUPPORTED
    assert _attn(lib, n=0) == OK
    assert lib.mhip_paged_attn_workspace_bytes(2, 1, 2, 1, 0, 5, 2, 64) == EINVAL
    assert lib.mhip_paged_attn_workspace_bytes(2, 1, 2, -1, 1, 4, 2, 64) == EINVAL
    assert lib.mhip_paged_attn_workspace_bytes(2, 1, 2, 1, 0, 4, 2, 136) == EHEADDIM
    assert lib.mhip_paged_attn_workspace_bytes(2, 1, 2, 1, 0, 4, 2, 64) > 0


def test_no_cpu_fallback():
    import torch

    import mercury_artifact_amd as M

    cache, _ = M.paged_cache(2, 16, 2, 64, device="cpu")
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: M.paged_attn_fwd(x, cache, table, lengths, 0.1), lambda: M.paged_cache_write(x, x, cache, table, lengths),
                 lambda: M.paged_cache_read(cache, table, lengths, 1)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    with pytest.raises(RuntimeError, match="bfloat16 or float8"):
        M.paged_cache(2, 16, 2, 64, dtype=torch.float16, device="cpu")


def test_positions_stay_below_the_last_ints(lib):
    for call in (_write, _read, _attn):
        assert call(lib, width=(1 << 27) - (1 << 12) + 1) == EUNSUPPORTED
    assert _attn(lib, B=0, width=(1 << 27) - (1 << 12)) == OK


def test_a_call_that_no_launch_takes_is_refused(lib):
    """A launch counts its threads in 32 bits; none of these may come as far as launching."""
    for starts in (None, P):
        many = dict(starts=starts, B=1, n=0 if starts else 1 << 28, T=1 << 28 if starts else 0, Hkv=1, tokens=(0, 128, 128))
        assert _write(lib, D=128, **many) == EUNSUPPORTED
        many["n"], many["T"] = many["n"] * 2, many["T"] * 2
        for dtype in (0, 1):
            assert _write(lib, D=64, dtype=dtype, **many) == EUNSUPPORTED
    for dtype in (0, 1):
        assert _read(lib, B=1, rows=1 << 29, Hkv=1, D=128, dtype=dtype) == EUNSUPPORTED
        assert _read(lib, B=1, rows=(1 << 30) - 129, Hkv=1, D=64, dtype=dtype) == EUNSUPPORTED
        # items of 256 rows: as many sequences
        assert _attn(lib, B=1 << 23, n=65, Hq=1, Hkv=1, dtype=dtype) == EUNSUPPORTED
        assert _attn(lib, starts=P, B=1 << 23, n=0, T=4, most=65, Hq=1, Hkv=1, tokens=(0, 64, 64), dtype=dtype) == EUNSUPPORTED
        assert _attn(lib, starts=P, B=1 << 20, n=0, T=4, most=65, Hq=8, Hkv=8, tokens=(0, 512, 64), dtype=dtype) == EUNSUPPORTED


def test_rows_of_a_sequence_and_a_tile_are_ints(lib):
    for T in (2 ** 31 - 65, 2 ** 31 - 256):
        assert _attn(lib, starts=P, B=1, n=0, T=T, most=1, Hq=1, Hkv=1, tokens=(0, 64, 64)) == EUNSUPPORTED
        assert _attn(lib, B=1, n=T, Hq=1, Hkv=1, tokens=(0, 64, 64)) == EUNSUPPORTED
