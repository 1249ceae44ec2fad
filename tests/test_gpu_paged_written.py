"""What the interpreter's path of the operators over a paged cache reports as written: each tensor that it writes, once, and no other."""
import pytest
import torch

import mercury_artifact_amd as M
from mercury_artifact_amd import _native as N

pytestmark = pytest.mark.gpu

E4M3, E2M1 = torch.float8_e4m3fn, torch.float4_e2m1fn_x2


@pytest.mark.parametrize("kind", [torch.bfloat16, E4M3, E2M1], ids=["bf16", "e4m3", "e2m1"])
def test_the_interpreters_path_counts_what_it_writes(monkeypatch, kind):
    cache, scales = M.paged_cache(8, 16, 2, 64, kind)
    weights, other = M.paged_weights(8, 16, 2), M.paged_weights(8, 16, 2)
    table = torch.tensor([[3, 1, 5, 0]], dtype=torch.int32).cuda()
    out_table = torch.tensor([[2, 4, 6, 7]], dtype=torch.int32).cuda()
    lengths = torch.tensor([60], dtype=torch.int32).cuda()
    k, q = torch.randn(1, 60, 2, 64).bfloat16().cuda(), torch.randn(1, 3, 4, 64).bfloat16().cuda()
    written = []

    class Declines:
        def __init__(self, host):
            self.host = host

        def written(self, *tensors):
            written.extend(t for t in tensors if t is not None)
            self.host.written(*tensors)

        def __getattr__(self, name):
            return lambda *args: None

    N.lib()                                              # (loading it asks the host module for its version)
    monkeypatch.setattr(N, "host", Declines(N.host))
    given = {"scales": scales}
    made = {}
    held = [t for t in (cache, scales) if t is not None]

    def attend():
        made["out"], made["lse"] = M.paged_attn_fwd(q, cache, table, lengths, 0.1, **given)

    for call, changed in [
        (lambda: M.paged_cache_write(k, k, cache, table, lengths, **given), lambda: held),
        (lambda: made.update(read=M.paged_cache_read(cache, table, lengths, 60, **given)), lambda: [made["read"]]),
        (attend, lambda: [made["out"], made["lse"]]),
        (lambda: M.paged_attn_weights(q, cache, table, lengths, 0.1, made["lse"], weights, **given), lambda: [weights]),
        (lambda: M.paged_attn_weights(q, cache, table, lengths, 0.1, made["lse"], weights, out=other, **given), lambda: [other]),
        (lambda: M.paged_cache_evict(cache, table, lengths, weights, 50, out_table=out_table, **given), lambda: [*held, weights]),
        (lambda: M.paged_cache_evict(cache, table, lengths, weights, 50, **given), lambda: [*held, weights]),
    ]:
        tensors = [*held, weights, other, table, out_table, lengths, q, k]
        before = [t._version for t in tensors]
        written.clear()
        call()
        assert len(written) == len(changed()) and all(any(w is c for c in changed()) for w in written)
        assert [t._version > n for t, n in zip(tensors, before)] == [any(t is c for c in changed()) for t in tensors]
