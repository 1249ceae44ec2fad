"""Sizes of the tensors of a paged cache that no C int holds (views of a few bytes): refused by name, not taken modulo 2^32."""
import pytest
import torch

import mercury_artifact_amd as M

pytestmark = pytest.mark.gpu

MANY = 2 ** 32 + 1


def _rows(*shape):
    """A contiguous last dimension of 8, the others over one another."""
    return torch.zeros(8, dtype=torch.bfloat16, device="cuda").expand(*shape, 8)


def test_sizes_that_no_c_int_holds():
    table, lengths = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    starts = torch.zeros(2, dtype=torch.int32, device="cuda")
    cache, _ = M.paged_cache(1, 16, 1, 8)
    heads = cache.expand(2, 1, 16, MANY, 8)
    for call in [
        lambda: M.paged_cache_read(heads, table, lengths, 0),
        lambda: M.paged_cache_read(_rows(2, MANY, 16, 1), table, lengths, 0),
        lambda: M.paged_cache_read(_rows(2, 1, MANY + 15, 1), table, lengths, 0),
        lambda: M.paged_cache_read(cache, table.expand(1, MANY), lengths, 0),
        lambda: M.paged_cache_write(_rows(1, 0, MANY), _rows(1, 0, MANY), heads, table, lengths),
        lambda: M.paged_cache_write(_rows(MANY, 1), _rows(MANY, 1), cache, table, lengths, starts=starts),
        lambda: M.paged_attn_fwd(_rows(1, 0, MANY), cache, table, lengths, 0.1),
        lambda: M.paged_attn_fwd(_rows(1, 0, MANY), heads, table, lengths, 0.1),
        lambda: M.paged_attn_fwd(_rows(1, MANY, 1), cache, table, lengths, 0.1, out=_rows(1, MANY, 1)),
        lambda: M.paged_attn_fwd(_rows(MANY, 1), cache, table, lengths, 0.1, starts=starts, most_new=1, out=_rows(MANY, 1)),
    ]:
        with pytest.raises(RuntimeError, match=r"is no whole number from 0 to 2\^31 - 1|contiguous rows"):
            call()
