"""What the C entries for keys' weights and eviction refuse, before anything is launched (no GPU needed; pointers are never followed)."""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mercury_artifact_amd as M
from mercury_artifact_amd import _native as N

OK, EINVAL, EDTYPE, EHEADDIM, EALIGN, EUNSUPPORTED = 0, -1, -2, -3, -4, -6
P = 0x10000


@pytest.fixture(scope="module")
def lib():
    return N.lib()


def _cache(Hkv, D, page):
    return (Hkv * page * D, D, page * D, Hkv * page, 1, page)


def _weigh(lib, q=P, kc=P, ks=P, table=P, lengths=P, starts=None, lse=P, w=P, out=P, B=2, n=3, T=0, most=3, Hq=4, Hkv=2, D=64, pages=9, page=16,
           width=4, tokens=None, cache=None, scale=0.1, decay=1.0, mask=1, dtype=0,
           ws=P):
    tokens = (n * Hq * D, Hq * D, D) if tokens is None else tokens
    at = (Hkv * page, 1, page)
    return lib.mhip_paged_attn_weights(q, kc, ks, table, lengths, starts, lse, w, out, B, n, T, most, Hq, Hkv, D, pages, page, width, width,
                                       *tokens, *(_cache(max(Hkv, 1), D, page) if cache is None else cache), *at, *at, scale, decay, mask, dtype, ws, None)


def _evict(lib, kc=P, vc=P, ks=P, vs=P, table=P, out_table=None, lengths=P, w=P, kept=P, left=P, B=2, Hkv=2, D=64, pages=9, page=16, width=4,
           out_pages=0, keep=10, recent=2, limit=12, cache=None, dtype=0):
    return lib.mhip_paged_cache_evict(kc, vc, ks, vs, table, out_table, lengths, w, kept, left, B, Hkv, D, pages, page, width, out_pages, width,
                                      out_pages, keep, recent, limit, *(_cache(max(Hkv, 1), D, page) if cache is None else cache),
                                      Hkv * page, 1, page, dtype, None)


@pytest.mark.parametrize("call", [_weigh, _evict])
def test_what_both_refuse(lib, call):
    for D in (0, 4, 100, 136):
        assert call(lib, D=D, cache=(4096, 256, 1024, 32, 1, 16)) == EHEADDIM
    assert call(lib, D=72, dtype=1) == EHEADDIM
    assert call(lib, D=80, dtype=3, cache=(4096, 256, 1024, 32, 1, 16)) == EHEADDIM
    assert call(lib, dtype=2) == EDTYPE
    assert call(lib, B=-1) == EINVAL
    assert call(lib, pages=-1) == EINVAL
    assert call(lib, page=8) == EUNSUPPORTED
    assert call(lib, page=1 << 20, width=1 << 11, cache=_cache(2, 64, 16)) == EUNSUPPORTED
    assert call(lib, width=-1) == EINVAL
    assert call(lib, Hkv=0) == EINVAL
    for missing in ("kc", "table", "lengths", "w"):
        assert call(lib, **{missing: None}) == EINVAL
    for dtype in (1, 3):
        assert call(lib, dtype=dtype, ks=None) == EINVAL
        assert call(lib, dtype=dtype, ks=P + 2) == EALIGN
    assert call(lib, kc=P + 8) == EALIGN
    assert call(lib, table=P + 2) == EALIGN
    assert call(lib, w=P + 2) == EALIGN
    assert call(lib, cache=(2048, 68, 1024, 32, 1, 16)) == EALIGN
    assert call(lib, cache=(2048, 0, 1024, 32, 1, 16)) == EUNSUPPORTED
    assert call(lib, B=0) == OK


def test_weights_refuse(lib):
    assert _weigh(lib, Hq=5) == EINVAL
    assert _weigh(lib, Hq=0) == EINVAL
    for scale in (0.0, -1.0, math.nan, math.inf):
        assert _weigh(lib, scale=scale) == EINVAL
    for decay in (-1.0, math.nan, math.inf):
        assert _weigh(lib, decay=decay) == EINVAL
    assert _weigh(lib, mask=2) == EINVAL
    assert _weigh(lib, most=-1) == EINVAL
    assert _weigh(lib, n=-1) == EINVAL
    for missing in ("q", "lse", "out"):
        assert _weigh(lib, **{missing: None}) == EINVAL
    assert _weigh(lib, q=P + 8) == EALIGN
    assert _weigh(lib, lse=P + 2) == EALIGN
    assert _weigh(lib, out=P + 2) == EALIGN
    assert _weigh(lib, tokens=(384, 132, 64)) == EALIGN
    assert _weigh(lib, starts=P, T=1 << 29) == EUNSUPPORTED
    assert _weigh(lib, B=1 << 16, n=1 << 16) == EUNSUPPORTED
    assert _weigh(lib, width=0, table=None) == OK
    many = dict(n=40, tokens=(40 * 4 * 64, 256, 64))
    assert _weigh(lib, ws=None, **many) == EINVAL
    assert _weigh(lib, ws=P + 8, **many) == EALIGN
    size = lib.mhip_paged_attn_weights_workspace_bytes
    assert size(1, 2, 1, 0, 4, 2) == 0 and size(40, 80, 40, 0, 4, 2) > 0 and size(0, 80, 40, 1, 4, 2) > 0 and size(0, 80, 1, 1, 4, 2) == 0
    assert size(1, 2, 1, 0, 5, 2) == EINVAL and size(1, 2, -1, 1, 4, 2) == EINVAL


def test_eviction_refuses(lib):
    assert _evict(lib, recent=-1) == EINVAL
    assert _evict(lib, recent=11) == EINVAL
    assert _evict(lib, keep=13) == EINVAL
    assert _evict(lib, limit=0x7fff0001) == EUNSUPPORTED
    for missing in ("vc", "kept", "left"):
        assert _evict(lib, **{missing: None}) == EINVAL
    assert _evict(lib, kept=P + 2) == EALIGN
    assert _evict(lib, left=P + 2) == EALIGN
    assert _evict(lib, out_table=P + 2, out_pages=1) == EALIGN
    assert _evict(lib, out_table=P, out_pages=0) == EINVAL
    assert _evict(lib, out_table=P, out_pages=1, limit=17) == EINVAL
    assert _evict(lib, out_table=P, out_pages=-1) == EINVAL
    # a launch counts its threads in 32 bits
    assert _evict(lib, B=1 << 22, Hkv=1) == EUNSUPPORTED
    assert _evict(lib, B=1 << 20, Hkv=1, out_table=P, out_pages=1 << 10, limit=1 << 14, keep=2) == EUNSUPPORTED


def test_no_cpu_fallback_no_gradients_no_fake_tensors():
    cache, _ = M.paged_cache(2, 16, 2, 64, device="cpu")
    weights = M.paged_weights(2, 16, 2, device="cpu")
    assert weights.shape == (2, 16, 2) and weights.stride() == (32, 1, 16) and (weights == 0).all()
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q, lse = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 1)
    calls = [lambda w: M.paged_attn_weights(q, cache, table, lengths, 0.1, lse, w), lambda w: M.paged_cache_evict(cache, table, lengths, w, 1)]
    for call in calls:
        with pytest.raises(RuntimeError, match="GPU only"):
            call(weights)
        with pytest.raises(RuntimeError, match="no gradients, which weights asks for"):
            call(weights.clone().requires_grad_())
        with FakeTensorMode():
            fake = torch.zeros(2, 16, 2)
        with pytest.raises(RuntimeError, match="no fake form"):
            call(fake)
