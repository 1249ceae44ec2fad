"""What the operators over a paged cache do with tensors that autograd or a trace looks after (no GPU needed: they say so before anything else)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad

import mercury_artifact_amd as M
from mercury_artifact_amd import _native as N

E4M3 = torch.float8_e4m3fn


def _data(device="cpu"):
    cache, scales = M.paged_cache(2, 16, 2, 64, E4M3, device=device)
    table = torch.tensor([[1]], dtype=torch.int32, device=device)
    lengths = torch.tensor([5], dtype=torch.int32, device=device)
    return cache, scales, table, lengths, torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device=device)


def _calls(asks, device="cpu"):
    """Name of the tensor that asks for a gradient, call."""
    cache, scales, table, lengths, x = _data(device)
    lse, chunk = torch.zeros(1, 2, 1, device=device), torch.zeros(2, 1, 3, 2, 64, dtype=torch.bfloat16, device=device)
    return [
        ("q", lambda: M.paged_attn_fwd(asks(x), cache, table, lengths, 0.1, scales=scales)),
        ("scales", lambda: M.paged_attn_fwd(x, cache, table, lengths, 0.1, scales=asks(scales))),
        ("out", lambda: M.paged_attn_fwd(x, cache, table, lengths, 0.1, scales=scales, out=asks(x))),
        ("lse", lambda: M.paged_attn_fwd(x, cache, table, lengths, 0.1, scales=scales, lse=asks(lse))),
        ("cache", lambda: M.paged_attn_fwd(x, asks(x.new_zeros(2, 2, 16, 2, 64)), table, lengths, 0.1)),
        ("k", lambda: M.paged_cache_write(asks(x), x, cache, table, lengths, scales=scales)),
        ("v", lambda: M.paged_cache_write(x, asks(x), cache, table, lengths, scales=scales)),
        ("scales", lambda: M.paged_cache_write(x, x, cache, table, lengths, scales=asks(scales))),
        ("cache", lambda: M.paged_cache_write(x, x, asks(x.new_zeros(2, 2, 16, 2, 64)), table, lengths)),
        ("cache", lambda: M.paged_cache_read(asks(x.new_zeros(2, 2, 16, 2, 64)), table, lengths, 3)),
        ("scales", lambda: M.paged_cache_read(cache, table, lengths, 3, scales=asks(scales))),
        ("out", lambda: M.paged_cache_read(cache, table, lengths, 3, scales=scales, out=asks(chunk))),
    ]


def _refused(device):
    for name, call in _calls(lambda t: t.detach().requires_grad_(), device):
        with pytest.raises(RuntimeError, match=f"no gradients, which {name} asks for"):
            call()
    with forward_ad.dual_level():
        for name, call in _calls(lambda t: forward_ad.make_dual(t.detach(), torch.ones_like(t)), device):
            with pytest.raises(RuntimeError, match=f"no gradients, which {name} asks for"):
                call()


def test_a_gradient_that_is_asked_for_is_refused():
    _refused("cpu")


def test_without_gradients_the_call_goes_on():
    with torch.no_grad():
        for _, call in _calls(lambda t: t.detach().requires_grad_()):
            with pytest.raises(RuntimeError, match="GPU only"):
                call()


@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_fake_tensors_are_refused(device):
    with FakeTensorMode():
        for _, call in _calls(lambda t: t, device):
            with pytest.raises(RuntimeError, match="no fake form"):
                call()


@pytest.mark.gpu
def test_a_gradient_that_is_asked_for_is_refused_on_the_gpu():
    _refused("cuda")
    with torch.no_grad():
        for _, call in _calls(lambda t: t.detach().requires_grad_(), "cuda"):
            call()
    torch.cuda.synchronize()


class _Declines:
    """A host module that leaves every call to the Python functions, but for counting writes."""

    def __init__(self, host):
        self.written = host.written

    def __getattr__(self, name):
        return lambda *args: None


@pytest.mark.gpu
@pytest.mark.parametrize("compiled", [True, False])
def test_what_is_written_counts_as_written(monkeypatch, compiled):
    """Autograd compares a tensor's count of writes with what it saved of it."""
    cache, scales, table, lengths, x = _data("cuda")
    lse, chunk = torch.zeros(1, 2, 1, device="cuda"), torch.zeros(2, 1, 3, 2, 64, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(x)
    if not compiled:
        N.lib()
        monkeypatch.setattr(N, "host", _Declines(N.host))
    read = (table, lengths, x)
    for call, changed in [
        (lambda: M.paged_cache_write(x, x, cache, table, lengths, scales=scales), (cache, scales)),
        (lambda: M.paged_cache_read(cache, table, lengths, 3, scales=scales, out=chunk), (chunk,)),
        (lambda: M.paged_attn_fwd(x, cache, table, lengths, 0.1, scales=scales, out=out, lse=lse), (out, lse)),
    ]:
        tensors = (*read, cache, scales, lse, chunk, out)
        before = [t._version for t in tensors]
        call()
        for t, n in zip(tensors, before):
            assert (t._version > n) == any(t is c for c in changed)


@pytest.mark.gpu
def test_a_saved_view_of_the_cache_that_is_written_over_is_noticed():
    cache, _ = M.paged_cache(2, 16, 2, 64)
    cache.zero_()
    _, _, table, lengths, x = _data("cuda")
    factor = torch.ones((), device="cuda", requires_grad=True)
    y = (cache[0, 1].float() * 1.0 * factor).sum() + (cache[1, 1] * factor.bfloat16()).float().sum()
    M.paged_cache_write(x, x, cache, table, lengths)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
