"""A paged K/V cache: new tokens written into it, rows of it read back as a chunk, attention of new tokens over it, and the keys
that had least of it evicted.

The ring steps take a rank's K/V as dense ``(2, B, S, Hkv, D)`` chunks, every sequence of one length.  Sequences that grow
token by token, each at its own length, lie in pages instead: ``cache`` is ``(2, pages, page_size, Hkv, D)`` -- keys and
values, as in a chunk -- in bfloat16, or in float8_e4m3fn with one float32 scale for each row, ``scales``
``(2, pages, page_size, Hkv)``, or in float4_e2m1fn_x2, two columns to an element (the even one in its low half), so that the last
dimension is D / 2, with a float8_e8m0fnu scale for each 32 columns, ``scales`` ``(2, pages, page_size, Hkv, 4)`` whatever D is;
``page_table`` ``(B, pages of a sequence)`` and ``lengths`` ``(B,)`` (int32, on the GPU) say
where a sequence's tokens lie and how many there are.  An entry outside ``[0, pages)`` is a page that is not here.  A rank
that holds some pages of a sequence attends over those alone, and the ranks' ``(out, lse)`` merge as the results of
different chunks do (``merge_many``, ``update_out_and_lse``).

New tokens come as ``(B, n, heads, D)``, or packed as ``(T, heads, D)`` with ``starts`` ``(B + 1,)``: rows ``starts[b]`` up to
``starts[b + 1]`` belong to sequence b, rows outside of all are left alone.  They are the last ones of their sequence:
``lengths`` counts them.  Nothing here waits for the GPU or looks at the values of tables, lengths and starts on the host.
A step of generation within a budget: ``paged_cache_write``, ``paged_attn_fwd``, ``paged_attn_weights``, ``paged_cache_evict``.
They compute no gradients, and refuse tensors that require one unless ``torch.no_grad()`` is on; nor do they take fake tensors.  The reference has no counterpart;
an operator that is asked for something it does not do raises ``RuntimeError``.
"""
from __future__ import annotations

import operator
from typing import Optional, Tuple

import torch
from torch._subclasses.fake_tensor import FakeTensor

from . import _native as N

__all__ = ["paged_cache", "paged_weights", "paged_cache_write", "paged_cache_read", "paged_attn_fwd", "paged_attn_weights", "paged_cache_evict"]


def paged_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                device="cuda") -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """An empty cache ``(2, pages, page_size, kv_heads, head_dim)`` (float4_e2m1fn_x2: head_dim / 2) and, in 8 or 4 bits, its
    scales.  In memory the rows of one head of a page lie together, which is how attention reads them; the operators take any
    other order too."""
    if dtype not in (torch.bfloat16, torch.float8_e4m3fn, torch.float4_e2m1fn_x2):
        raise RuntimeError("a paged cache is bfloat16 or float8_e4m3fn or float4_e2m1fn_x2")
    four = dtype == torch.float4_e2m1fn_x2
    if four and head_dim % 32:
        raise RuntimeError(f"a float4_e2m1fn_x2 cache has a multiple of 32 columns, not {head_dim}")
    cache = torch.empty((2, pages, kv_heads, page_size, head_dim // 2 if four else head_dim), dtype=dtype, device=device).transpose(2, 3)
    if dtype == torch.bfloat16:
        return cache, None
    if four:
        return cache, torch.empty((2, pages, kv_heads, page_size, 4), dtype=torch.float8_e8m0fnu, device=device).transpose(2, 3)
    return cache, torch.empty((2, pages, kv_heads, page_size), dtype=torch.float32, device=device).transpose(2, 3)


def paged_weights(pages: int, page_size: int, kv_heads: int, device="cuda") -> torch.Tensor:
    """What attention the keys of a cache have had, ``(pages, page_size, kv_heads)`` in float32: nothing yet."""
    return torch.zeros((pages, kv_heads, page_size), dtype=torch.float32, device=device).transpose(1, 2)


def _check_plain(**tensors):
    """Nothing that only a registered operator could do: a derivative, or shapes without data."""
    for name, t in tensors.items():
        if isinstance(t, FakeTensor):
            raise RuntimeError(f"the operators over a paged cache have no fake form, and {name} is a fake tensor: keep them out of traced programs")
        if t is not None and ((torch.is_grad_enabled() and t.requires_grad) or torch.autograd.forward_ad.unpack_dual(t).tangent is not None):
            raise RuntimeError(f"the operators over a paged cache compute no gradients, which {name} asks for: "
                               "call them under torch.no_grad(), or with detached tensors")


def _check_cache(cache, scales, page_table, lengths, starts=None):
    N.require_cuda(cache, scales, page_table, lengths, starts)
    if cache.dim() != 5 or cache.shape[0] != 2 or cache.stride(-1) != 1:
        raise RuntimeError("cache must be (2, pages, page_size, kv_heads, head_dim) with a contiguous last dimension")
    if cache.dtype == torch.float8_e4m3fn:
        if scales is None or scales.shape != cache.shape[:-1] or scales.dtype != torch.float32:
            raise RuntimeError(f"a float8_e4m3fn cache needs float32 scales {tuple(cache.shape[:-1])}")
    elif cache.dtype == torch.float4_e2m1fn_x2:
        if scales is None or scales.shape != (*cache.shape[:-1], 4) or scales.dtype != torch.float8_e8m0fnu:
            raise RuntimeError(f"a float4_e2m1fn_x2 cache needs float8_e8m0fnu scales {(*cache.shape[:-1], 4)}")
        if scales.stride(-1) != 1 or any(x % 4 for x in scales.stride()[:4]):
            raise RuntimeError("the four scales of a row must lie together, on 4 bytes")
    elif cache.dtype != torch.bfloat16:
        raise RuntimeError(f"unsupported cache dtype {cache.dtype}: bfloat16 or float8_e4m3fn or float4_e2m1fn_x2")
    elif scales is not None:
        raise RuntimeError("a bfloat16 cache has no scales")
    B = lengths.shape[0] if lengths.dim() == 1 else -1
    if B < 0 or lengths.dtype != torch.int32 or not lengths.is_contiguous():
        raise RuntimeError("lengths must be a contiguous int32 (B,) tensor")
    if page_table.dim() != 2 or page_table.shape[0] != B or page_table.dtype != torch.int32 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise RuntimeError("page_table must be an int32 (B, pages of a sequence) tensor with contiguous rows")
    if starts is not None and (starts.shape != (B + 1,) or starts.dtype != torch.int32 or not starts.is_contiguous()):
        raise RuntimeError("starts must be a contiguous int32 (B + 1,) tensor")
    for name, size in zip(("pages", "rows of a page", "K/V heads", "columns"), cache.shape[1:]):
        _whole(f"the number of {name}", size)
    _whole("the number of sequences", B)
    _whole("the number of entries of page_table", page_table.shape[1])
    for t in (scales, page_table, lengths, starts):
        if t is not None and t.device != cache.device:
            raise RuntimeError("cache, scales, page_table, lengths and starts must be on one device")
    return B


def _sizes(cache):
    """Pages, rows of a page, K/V heads, columns."""
    _, pages, page_size, Hkv, D = cache.shape
    return pages, page_size, Hkv, 2 * D if cache.dtype == torch.float4_e2m1fn_x2 else D


def _check_tokens(name, t, B, starts, heads, head_dim, device):
    """Whether t holds new tokens: (B, n, heads, head_dim), or (T, heads, head_dim) with starts.  Returns n, T."""
    N.require_cuda(t)
    if t.dim() != (4 if starts is None else 3) or (starts is None and t.shape[0] != B):
        raise RuntimeError(f"{name} must be (B, new tokens, heads, head_dim), or (all new tokens, heads, head_dim) with starts")
    if t.shape[-2] != heads or t.shape[-1] != head_dim or t.stride(-1) != 1 or t.dtype != torch.bfloat16 or t.device != device:
        raise RuntimeError(f"{name} must be bfloat16 with {heads} heads of {head_dim}, a contiguous last dimension, on the cache's device")
    _whole("the number of heads", heads)
    n = 0 if starts is not None else _whole("the number of new tokens of a sequence", t.shape[1])
    return n, _whole("the number of new tokens", t.shape[0] if starts is not None else t.shape[0] * n)


def _whole(name, x, bits=31):
    """x as a number that a C int (or one of as many bits) holds."""
    try:
        whole = operator.index(x)
    except TypeError:
        whole = -1
    if not 0 <= whole < 2 ** bits:
        raise RuntimeError(f"invalid {name}: {x!r} is no whole number from 0 to 2^{bits} - 1")
    return whole


def _token_strides(t):
    return t.stride()[:3] if t.dim() == 4 else (0, *t.stride()[:2])


def _cache_args(cache, scales):
    """Pointers of keys, values and their scales, and the strides."""
    size = cache.element_size()
    k, v = cache.data_ptr(), cache.data_ptr() + cache.stride(0) * size if cache.numel() else cache.data_ptr()
    if scales is None:
        return (k, v, None, None), (*cache.stride()[1:4], 0, 0, 0)
    ks, each = scales.data_ptr(), 4 // scales.element_size()             # (strides of four bytes: a float, or a row of four)
    strides = [x // each for x in scales.stride()[:4]]
    return (k, v, ks, ks + strides[0] * 4 if scales.numel() else ks), (*cache.stride()[1:4], *strides[1:])


def _dtype(cache):
    return {torch.bfloat16: N.MHIP_BF16, torch.float8_e4m3fn: N.MHIP_E4M3, torch.float4_e2m1fn_x2: N.MHIP_E2M1}[cache.dtype]


def paged_cache_write(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                      scales: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None) -> None:
    """The keys and values of the new tokens (bfloat16) into their rows of the cache.  In e4m3 each row gets a scale of its
    own, the least power of two that keeps its largest value within 448; a row with an infinity or a NaN gets the scale NaN
    and reads back as NaN.  In e2m1 the same goes for each 32 columns, whose largest value is kept within 6 (values past 6 * 2^125
    count as that).  Rows of pages that are not here are dropped.  No two new tokens of a call may lie in one row
    (sequences that share the page they write to)."""
    if N.host.paged_cache_write(k, v, cache, page_table, lengths, scales, starts):
        return
    _check_plain(k=k, v=v, cache=cache, scales=scales)
    B = _check_cache(cache, scales, page_table, lengths, starts)
    pages, page_size, Hkv, D = _sizes(cache)
    n, T = _check_tokens("k", k, B, starts, Hkv, D, cache.device)
    _check_tokens("v", v, B, starts, Hkv, D, cache.device)
    if k.shape != v.shape:
        raise RuntimeError(f"shape mismatch: k {tuple(k.shape)} v {tuple(v.shape)}")
    pointers, strides = _cache_args(cache, scales)
    with torch.cuda.device(cache.device):
        code = N.lib().mhip_paged_cache_write(
            N.ptr(k), N.ptr(v), *pointers, N.ptr(page_table), N.ptr(lengths), N.ptr(starts),
            B, n, T, Hkv, D, pages, page_size, page_table.shape[1], page_table.stride(0),
            *_token_strides(k), *_token_strides(v), *strides, _dtype(cache), N.stream_of(cache))
    N.check(code, "mhip_paged_cache_write")
    N.host.written(cache, scales)


def paged_cache_read(cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, rows: int, begin: int = 0,
                     scales: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows ``begin`` up to ``begin + rows`` of every sequence as a chunk ``(2, B, rows, Hkv, D)`` in bfloat16, as the ring
    steps take it; zeros past a sequence's end and where a page is not here."""
    done = N.host.paged_cache_read(cache, page_table, lengths, rows, begin, scales, out)
    if done is not None:
        return done
    _check_plain(cache=cache, scales=scales, out=out)
    B = _check_cache(cache, scales, page_table, lengths)
    pages, page_size, Hkv, D = _sizes(cache)
    rows, begin = _whole("rows", rows), _whole("begin", begin)
    if out is None:
        out = torch.empty((2, B, rows, Hkv, D), dtype=torch.bfloat16, device=cache.device)
    elif out.shape != (2, B, rows, Hkv, D) or out.dtype != torch.bfloat16 or out.stride(-1) != 1 or out.device != cache.device:
        raise RuntimeError("out must be (2, B, rows, kv_heads, head_dim) bfloat16 with a contiguous last dimension, on the cache's device")
    pointers, strides = _cache_args(cache, scales)
    with torch.cuda.device(cache.device):
        code = N.lib().mhip_paged_cache_read(
            *pointers, N.ptr(page_table), N.ptr(lengths), N.ptr(out), B, begin, rows, Hkv, D, pages, page_size,
            page_table.shape[1], page_table.stride(0), *strides, *out.stride()[:4], _dtype(cache), N.stream_of(cache))
    N.check(code, "mhip_paged_cache_read")
    N.host.written(out)
    return out


def paged_attn_fwd(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, softmax_scale: float,
                   causal: bool = True, scales: Optional[torch.Tensor] = None, starts: Optional[torch.Tensor] = None,
                   most_new: Optional[int] = None, out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                   ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of the new tokens over their sequences' keys, their own among them: ``out`` like q in bfloat16 and ``lse``
    (B, Hq, n) -- packed: (Hq, T) -- in float32.  ``causal``: new token i of n sees the keys up to ``lengths - n + i``, else all
    of them.  Rows that see no key get 0 and -inf.  ``most_new``: with ``starts``, about how many new tokens a sequence has at
    most (default: all of them in one).  Results are right whatever it says; it chooses the form of the kernels, and those round
    differently.  With up to 16 rows (new tokens times query heads of a K/V head) the values' weights are carried as two bfloat16
    numbers (not over a cache in e2m1), with more they are rounded to bfloat16 once; with up to 64 rows the scales of a cache are applied in float32, with more
    a row times its scale is rounded to bfloat16, which is exact for powers of two.  ``out`` may be q itself."""
    done = N.host.paged_attn_fwd(q, cache, page_table, lengths, softmax_scale, causal, scales, starts, most_new, out, lse)
    if done is not None:
        return done
    _check_plain(q=q, cache=cache, scales=scales, out=out, lse=lse)
    B = _check_cache(cache, scales, page_table, lengths, starts)
    pages, page_size, Hkv, D = _sizes(cache)
    Hq = q.shape[-2] if q.dim() >= 2 else 0
    n, T = _check_tokens("q", q, B, starts, Hq, D, cache.device)
    if Hkv == 0 or Hq == 0 or Hq % Hkv != 0:
        raise RuntimeError("number of query heads must be a multiple of the number of KV heads")
    if out is None:
        out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    else:
        _check_tokens("out", out, B, starts, Hq, D, cache.device)
        if out.shape != q.shape:
            raise RuntimeError("out must have the shape of q")
    shape = (B, Hq, n) if starts is None else (Hq, T)
    if lse is None:
        lse = torch.empty(shape, dtype=torch.float32, device=q.device)
    else:
        N.require_cuda(lse)
        if lse.shape != shape or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != cache.device:
            raise RuntimeError(f"lse must be a contiguous float32 {shape} tensor on the cache's device")
    most = n if starts is None else T if most_new is None else min(_whole("most_new", most_new, 63), T)
    size = N.lib().mhip_paged_attn_workspace_bytes(B, n, T, most, int(starts is not None), Hq, Hkv, D)
    if size < 0:
        N.check(int(size), "mhip_paged_attn_workspace_bytes")
    workspace = torch.empty((int(size),), dtype=torch.uint8, device=q.device)
    pointers, strides = _cache_args(cache, scales)
    with torch.cuda.device(cache.device):
        code = N.lib().mhip_paged_attn_fwd(
            N.ptr(q), *pointers, N.ptr(page_table), N.ptr(lengths), N.ptr(starts), N.ptr(out), N.ptr(lse),
            B, n, T, most, Hq, Hkv, D, pages, page_size, page_table.shape[1], page_table.stride(0),
            *_token_strides(q), *strides, *_token_strides(out), float(softmax_scale),
            N.MASK_CAUSAL if causal else N.MASK_NONE, _dtype(cache), N.ptr(workspace), N.stream_of(cache))
    N.check(code, "mhip_paged_attn_fwd")
    N.host.written(out, lse)
    return out, lse


def _check_weights(name, t, cache):
    N.require_cuda(t)
    if t.shape != cache.shape[1:4] or t.dtype != torch.float32 or t.device != cache.device:
        raise RuntimeError(f"{name} must be float32 {tuple(cache.shape[1:4])}, on the cache's device")


def paged_attn_weights(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, softmax_scale: float,
                       lse: torch.Tensor, weights: torch.Tensor, causal: bool = True, scales: Optional[torch.Tensor] = None,
                       starts: Optional[torch.Tensor] = None, most_new: Optional[int] = None, decay: float = 1.0,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What attention each key has had: ``weights`` ``(pages, page_size, Hkv)`` in float32 become ``decay`` times what they were --
    nothing for the keys of the new tokens -- plus the key's weight in the attention of every new token that sees it, summed over the
    query heads of its K/V head.  ``q``, ``lse`` and the other arguments are those of ``paged_attn_fwd``; ``lse`` may be merged over the
    ranks that hold parts of a sequence.  Rows whose ``lse`` is -inf weigh nothing, sequences without new tokens keep their weights, and
    entries that belong to no key are left as they are.  No two sequences of a call may share a page.  Scores are rounded as those of
    ``paged_attn_fwd`` with the same ``most_new``: where that rounds a row times its scale to bfloat16 (exact for powers of two), this does, too.
    ``out``: takes the results in place of ``weights`` (and is returned)."""
    done = N.host.paged_attn_weights(q, cache, page_table, lengths, softmax_scale, lse, weights, causal, scales, starts, most_new, decay, out)
    if done is not None:
        return done
    _check_plain(q=q, cache=cache, scales=scales, lse=lse, weights=weights, out=out)
    B = _check_cache(cache, scales, page_table, lengths, starts)
    pages, page_size, Hkv, D = _sizes(cache)
    Hq = q.shape[-2] if q.dim() >= 2 else 0
    n, T = _check_tokens("q", q, B, starts, Hq, D, cache.device)
    if Hkv == 0 or Hq == 0 or Hq % Hkv != 0:
        raise RuntimeError("number of query heads must be a multiple of the number of KV heads")
    shape = (B, Hq, n) if starts is None else (Hq, T)
    N.require_cuda(lse)
    if lse.shape != shape or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != cache.device:
        raise RuntimeError(f"lse must be a contiguous float32 {shape} tensor on the cache's device")
    _check_weights("weights", weights, cache)
    if out is None:
        out = weights
    else:
        _check_weights("out", out, cache)
    most = n if starts is None else T if most_new is None else min(_whole("most_new", most_new, 63), T)
    size = N.lib().mhip_paged_attn_weights_workspace_bytes(n, T, most, int(starts is not None), Hq, Hkv)
    if size < 0:
        N.check(int(size), "mhip_paged_attn_weights_workspace_bytes")
    workspace = torch.empty((int(size),), dtype=torch.uint8, device=q.device)
    (k, _, ks, _), strides = _cache_args(cache, scales)
    with torch.cuda.device(cache.device):
        code = N.lib().mhip_paged_attn_weights(
            N.ptr(q), k, ks, N.ptr(page_table), N.ptr(lengths), N.ptr(starts), N.ptr(lse), N.ptr(weights), N.ptr(out),
            B, n, T, most, Hq, Hkv, D, pages, page_size, page_table.shape[1], page_table.stride(0), *_token_strides(q), *strides,
            *weights.stride(), *out.stride(), float(softmax_scale), float(decay), N.MASK_CAUSAL if causal else N.MASK_NONE, _dtype(cache),
            N.ptr(workspace), N.stream_of(cache))
    N.check(code, "mhip_paged_attn_weights")
    N.host.written(out)
    return out


def paged_cache_evict(cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, weights: torch.Tensor, keep: int, recent: int = 0,
                      limit: Optional[int] = None, scales: Optional[torch.Tensor] = None, out_table: Optional[torch.Tensor] = None,
                      ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Sequences of more than ``limit`` (default: ``keep``) tokens are cut to ``keep``: each K/V head keeps the keys of the ``recent``
    last tokens and, of the others, those with the largest ``weights`` (NaN above all, of equal ones the first).  They move, in their
    order, with values, scales and weights, to the first rows of the sequence -- in its own pages, which no two sequences may share, or
    in those of ``out_table`` ``(B, at least limit / page_size)``, where the rows of sequences that are not cut go too; no page of it
    may hold a sequence's rows or be there twice.  Returns their old positions, ``kept`` ``(B, Hkv, limit)`` in int32 with -1 behind them, and the new
    lengths, ``left`` ``(B,)``; ``lengths`` itself is not written.  A sequence of which a page is not here is left as it is, with -1
    in all of ``kept``: it has no rows in the pages of ``out_table`` either, so it goes on with its row of ``page_table``."""
    limit = keep if limit is None else limit
    done = N.host.paged_cache_evict(cache, page_table, lengths, weights, keep, recent, limit, scales, out_table)
    if done is not None:
        return done
    _check_plain(cache=cache, scales=scales, weights=weights)
    B = _check_cache(cache, scales, page_table, lengths)
    pages, page_size, Hkv, D = _sizes(cache)
    _check_weights("weights", weights, cache)
    keep, recent, limit = _whole("keep", keep), _whole("recent", recent), _whole("limit", limit)
    if not recent <= keep <= limit:
        raise RuntimeError(f"keep ({keep}) must be from recent ({recent}) to limit ({limit})")
    if out_table is not None:
        N.require_cuda(out_table)
        if out_table.dim() != 2 or out_table.shape[0] != B or out_table.dtype != torch.int32 or (out_table.shape[1] > 1 and out_table.stride(1) != 1) or out_table.device != cache.device:
            raise RuntimeError("out_table must be an int32 (B, pages of a sequence) tensor with contiguous rows, on the cache's device")
        if _whole("the number of entries of out_table", out_table.shape[1]) * page_size < limit:
            raise RuntimeError(f"out_table must have pages for {limit} rows of a sequence")
    kept = torch.empty((B, Hkv, limit), dtype=torch.int32, device=cache.device)
    left = torch.empty((B,), dtype=torch.int32, device=cache.device)
    pointers, strides = _cache_args(cache, scales)
    with torch.cuda.device(cache.device):
        code = N.lib().mhip_paged_cache_evict(
            *pointers, N.ptr(page_table), N.ptr(out_table), N.ptr(lengths), N.ptr(weights), N.ptr(kept), N.ptr(left),
            B, Hkv, D, pages, page_size, page_table.shape[1], 0 if out_table is None else out_table.shape[1],
            page_table.stride(0), 0 if out_table is None else out_table.stride(0), keep, recent, limit, *strides, *weights.stride(),
            _dtype(cache), N.stream_of(cache))
    N.check(code, "mhip_paged_cache_evict")
    N.host.written(cache, scales, weights)
    return kept, left
