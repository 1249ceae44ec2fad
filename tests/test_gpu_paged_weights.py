"""Attention over a paged cache: a value that is no number reaches every row that sees it, however little the row's weight for it is."""
import math

import pytest
import torch

import mercury_artifact_amd as M

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new,Hq", [(1, 2), (8, 2), (12, 4), (30, 2), (90, 2)])
@pytest.mark.parametrize("where", ["before", "among"])
def test_a_value_that_is_no_number_with_a_weight_of_nothing(e4m3, new, Hq, where):
    """Scores lie 200 apart, so that in 32 bits the key's weight is zero: the rows that see it get NaN, the others do not.  `before`: in
    a tile that every row sees whole; `among`: among the new tokens, where rows of one tile differ."""
    length, D, page = 300, 64, 16
    at = 40 if where == "before" else length - new + new // 2
    g = torch.Generator().manual_seed(new)
    cache, scales = M.paged_cache(20, page, 1, D, E4M3 if e4m3 else torch.bfloat16)
    table = torch.randperm(20, generator=g)[:19].int().view(1, 19).cuda()
    lengths = torch.tensor([length], dtype=torch.int32).cuda()
    k, v = torch.randn(1, length, 1, D, generator=g), torch.randn(1, length, 1, D, generator=g)
    k[..., 0] = 10.0
    k[0, at, 0, 0] = -10.0
    q = torch.zeros(1, new, Hq, D)
    q[..., 0] = 10.0
    v[0, at, 0, 9] = math.nan
    M.paged_cache_write(k.bfloat16().cuda(), v.bfloat16().cuda(), cache, table, lengths, scales=scales)
    out, lse = M.paged_attn_fwd(q.bfloat16().cuda(), cache, table, lengths, 1.0, scales=scales)
    out, lse = out.cpu()[0], lse.cpu()[0]
    sees = torch.arange(new) + length - new >= at
    if where == "among" and new == 1:
        assert sees.all()                  # the one new token, whose own key it is
        assert torch.isnan(out[:, :, 9]).all()
        return
    assert torch.isnan(out[sees][:, :, 9]).all() and torch.isfinite(out[~sees]).all() and torch.isfinite(lse).all()
    if not e4m3:                           # (an e4m3 row with a NaN is NaN in all of its columns)
        out[:, :, 9] = 0.0
        assert torch.isfinite(out).all()
