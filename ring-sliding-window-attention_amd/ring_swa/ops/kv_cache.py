"""Serving from an 8-bit paged cache: the token-by-token continuation of a sequence whose prompt the
sliding-window and streaming-LLM functions have computed.  No counterpart in the upstream package,
which computes whole sequences only.

A cache holds e4m3 codes times one power of two per (page, kv head); a page holds ``page_size``
tokens of one sequence, and the caller's ``page_table`` (int32 ``[batch, max_pages]``, on the device)
says which::

    cache = KVCache.empty(num_pages, heads_kv, head_dim, device="cuda")
    out = ring_streaming_llm_attn(q, k, v, window, num_sink_tokens=4)           # the prompt
    kv_cache_append(cache, k, v, page_table, held)                              # held = 0
    held += k.shape[1]
    while True:                                                                 # a token at a time
        kv_cache_append(cache, k, v, page_table, held)
        held += 1
        out, lse = kv_cache_attn(q, cache, page_table, held, window, num_sink_tokens=4, return_lse=True)
        kv_cache_weights(q, cache, page_table, held, lse, weights, window, num_sink_tokens=4)
        ...                                                                     # now and then:
        held, weights, kept = kv_cache_evict(cache, weights, page_table, held, new_page_table, budget)

Lengths and page ids stay on the device, nothing is read back.  Rows are ``[batch, seq, heads, dim]``,
or packed ``[tokens, heads, dim]`` with ``cu_seqlens`` (int32 ``[batch + 1]``; sequences may bring
different numbers of rows, none among them; rows that are no sequence's are passed over), as in the
attention functions.  The new rows' keys are
in the cache already when their queries attend: row ``i`` of ``n`` is token ``seqlens - n + i``.  A
page id outside the cache (``-1``) is a page that is not there: seen by nobody, never written, so the
pages that a window has left behind can be given back.  There is no backward.

A compiled program makes these calls between its graphs (``fullgraph=True`` refuses them); in a traced one, and to a
dispatch mode, they are the operators ``ring_swa::cache_append``, ``cache_attn``, ``cache_weights`` and ``cache_evict``.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from .. import _lib

PAGE_SIZES = (16, 32, 64, 128, 256)


class KVCache(NamedTuple):
    """The tensors of a cache: ``k`` e4m3 ``[pages, kv_heads, page_size, dim]``, ``v`` e4m3 ``[pages,
    kv_heads, page_size / 16, dim, 16]`` (the 16 keys of a group are adjacent: what the matrix
    instruction reads), ``k_scale`` and ``v_scale`` e8m0 ``[pages, kv_heads]``.  Strides of pages and
    heads are free (multiples of 16 for ``k`` and ``v``), so several layers' caches may share a tensor."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, num_pages: int, heads_kv: int, head_dim: int, page_size: int = 64,
              device=None) -> "KVCache":
        """A cache of ``num_pages`` pages with nothing in them."""
        assert page_size in PAGE_SIZES, f"page_size must be one of {PAGE_SIZES}"
        k = torch.empty(num_pages, heads_kv, page_size, head_dim, dtype=torch.float8_e4m3fn, device=device)
        v = torch.empty(num_pages, heads_kv, page_size // 16, head_dim, 16, dtype=torch.float8_e4m3fn,
                        device=device)
        scales = (torch.zeros(num_pages, heads_kv, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
                  for _ in range(2))
        return cls(k, v, *scales)

    @property
    def page_size(self) -> int:
        return self.k.shape[2]


def _dense_from(t: torch.Tensor, dim: int) -> bool:
    """Are the dimensions of ``t`` from ``dim`` on without gaps?  (A stride over one element is never used.)"""
    step = 1
    for d in range(t.dim() - 1, dim - 1, -1):
        if t.shape[d] != 1 and t.stride(d) != step:
            return False
        step *= t.shape[d]
    return True


def _calls(cache):
    """The native module where it may take the call (it answers None to what it leaves to Python)."""
    return _lib.torch_calls() if cache[0].is_cuda else None


@torch._disable_dynamo
def _uncompiled(call, *args, **kwargs):
    """Compiled programs make the calls between their graphs, as they make those of the attention functions.  (In a
    graph, PyTorch's default compiler refuses operators that write beside e8m0 tensors, and others copy the cache.)"""
    return call(*args, **kwargs)


# What the native module leaves to Python goes through operators that PyTorch knows, so that whatever looks on (a
# tracer, a dispatch mode) sees one operation with what it reads and writes, and not a launch behind its back.
_ops = torch.library.Library("ring_swa", "DEF")
_CACHE = "Tensor k, Tensor v, Tensor k_scale, Tensor v_scale"
_WRITTEN_CACHE = "Tensor(a!) k, Tensor(b!) v, Tensor(c!) k_scale, Tensor(d!) v_scale"


def _operator(schema, fake):
    """Registers the function under it: ``schema``, and ``fake`` for tensors without data."""
    def register(fn):
        name = schema[:schema.index("(")]
        _ops.define(schema)
        _ops.impl(name, fn, "CompositeExplicitAutograd")
        torch.library.register_fake("ring_swa::" + name, fake, lib=_ops)
        return getattr(torch.ops.ring_swa, name).default
    return register


def _no_grad(*tensors) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("the cache has no backward: call this under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the cache has no forward derivative: call this on tensors without tangents")


def _fit(*sizes) -> None:
    """(the parameter block would cut them to 32 bits without a word; what is too large below that, the library refuses)"""
    assert max(sizes) < 1 << 31, "sizes must be below 2^31"


def _cache_params(cache, page_table, seqlens, rows, cu_seqlens):
    """The fields that every call sets, from its cache, table, lengths and rows (a tensor, or None)."""
    k, v, k_scale, v_scale = cache
    assert k.dim() == 4 and v.dim() == 5, "expected k [pages, heads, page, dim], v [pages, heads, page / 16, dim, 16]"
    pages, heads, size, dim = k.shape
    assert heads > 0 and size in PAGE_SIZES, f"expected heads, and page_size one of {PAGE_SIZES}"
    assert v.shape == (pages, heads, size // 16, dim, 16), "v must be [pages, heads, page / 16, dim, 16]"
    assert k_scale.shape == v_scale.shape == (pages, heads), "scales must be [pages, heads]"
    assert k.dtype == v.dtype == torch.float8_e4m3fn, "k and v must be float8_e4m3fn"
    assert k_scale.dtype == v_scale.dtype == torch.float8_e8m0fnu, "scales must be float8_e8m0fnu"
    assert _dense_from(k, 2) and _dense_from(v, 2), "the rows of a (page, head) must be dense"
    assert page_table.dim() == 2 and page_table.dtype == torch.int32, "page_table must be int32 [batch, max_pages]"
    assert _dense_from(page_table, 1), "the entries of a row of page_table must be adjacent"
    batch = page_table.shape[0]
    assert seqlens.dtype == torch.int32 and seqlens.shape == (batch,) and seqlens.is_contiguous(), (
        "seqlens must be a contiguous int32 tensor [batch]")
    dev = _lib.require_device(k, v, k_scale, v_scale, page_table, seqlens)
    _fit(*k.shape, *page_table.shape)
    p = _lib.CacheParams()  # (zero-initialised)
    p.head_dim, p.batch, p.heads_q, p.heads_kv = dim, batch, heads, heads
    p.page_size, p.num_pages, p.max_pages = size, pages, page_table.shape[1]
    p.k, p.v, p.k_scale, p.v_scale = k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr()
    p.k_stride, p.v_stride = k.stride()[:2], v.stride()[:2]
    p.k_scale_stride, p.v_scale_stride = k_scale.stride(), v_scale.stride()
    p.page_table, p.page_table_stride = page_table.data_ptr(), page_table.stride(0)
    p.seqlens = seqlens.data_ptr()
    if rows is not None:
        assert rows.shape[-1] == dim, "head_dim mismatch"
        _fit(*rows.shape)
        _lib.require_device(k, rows)
        p.dtype = _lib.dtype_code(rows)
        if cu_seqlens is None:
            assert rows.dim() == 4, "expected [batch, seq, heads, dim]"
            assert rows.shape[0] == batch, "batch mismatch"
            p.seqlen_q = rows.shape[1]
        else:
            assert rows.dim() == 3, "expected [tokens, heads, dim]"
            assert cu_seqlens.dtype == torch.int32 and cu_seqlens.shape == (batch + 1,) and \
                cu_seqlens.is_contiguous(), "cu_seqlens must be a contiguous int32 tensor [batch + 1]"
            _lib.require_device(k, cu_seqlens)
            p.total_q = rows.shape[0]
            p.cu_seqlens_q = cu_seqlens.data_ptr()
    return p, dev


def _strides3(t: torch.Tensor, packed: bool):
    st = t.stride()
    return (0, st[0], st[1]) if packed else st[:3]


def _window(window_size) -> int:
    return max(-1, min(int(window_size), 1 << 28))  # (2^28 is unbounded)


def _sinks(num_sink_tokens) -> int:
    return min(int(num_sink_tokens), 1 << 28)


def _scale(softmax_scale) -> Optional[float]:
    return None if softmax_scale is None else float(softmax_scale)


def _query_params(p, q, heads_kv, softmax_scale, window_size, num_sink_tokens, packed):
    assert q.shape[-2] % heads_kv == 0, "Number of query heads must be divisible by number of key/value heads"
    assert q.stride(-1) == 1, "last dimension must be contiguous"
    assert num_sink_tokens >= 0
    p.heads_q = q.shape[-2]
    p.softmax_scale = float(q.shape[-1] ** (-0.5) if softmax_scale is None else softmax_scale)
    p.window_left = _window(window_size)
    p.num_sink = _sinks(num_sink_tokens)
    p.q, p.q_stride = q.data_ptr(), _strides3(q, packed)


def kv_cache_append(
    cache: KVCache,
    k: torch.Tensor,
    v: torch.Tensor,
    page_table: torch.Tensor,
    seqlens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
) -> None:
    """Write the keys and values of new tokens behind the ``seqlens`` tokens that the sequences hold.

    ``k``, ``v``: ``[batch, seq, kv_heads, dim]``, or packed ``[tokens, kv_heads, dim]`` with
    ``cu_seqlens``; bf16 or fp16.  The scale of a (page, head) is the smallest power of two at which
    its largest finite value is within e4m3's range of 448; where the page holds tokens from before it
    never shrinks, and if it grows their codes are rounded anew (only those that fall below the
    smallest normal code change).  Infinities and NaN are stored as NaN.  Tokens beyond the last page
    of ``page_table``, or whose page is not there, are dropped.  ``seqlens`` is left alone; two
    sequences of one call must not have a page written in common."""
    if torch.compiler.is_dynamo_compiling():
        return _uncompiled(kv_cache_append, cache, k, v, page_table, seqlens, cu_seqlens)
    calls = _calls(cache)
    if calls is not None and calls.cache_append(cache, k, v, page_table, seqlens, cu_seqlens):
        return
    _no_grad(*cache, k, v)
    _append(*cache, k, v, page_table, seqlens, cu_seqlens)


@_operator(f"cache_append({_WRITTEN_CACHE}, Tensor new_k, Tensor new_v, Tensor page_table, Tensor seqlens, "
           "Tensor? cu_seqlens) -> ()", lambda *_: None)
def _append(k, v, k_scale, v_scale, new_k, new_v, page_table, seqlens, cu_seqlens):
    p, dev = _cache_params((k, v, k_scale, v_scale), page_table, seqlens, new_k, cu_seqlens)
    assert new_k.shape == new_v.shape and new_k.dtype == new_v.dtype, "k and v must have the same shape and dtype"
    assert new_k.shape[-2] == p.heads_kv, "k and v must have the cache's heads"
    _lib.require_device(new_k, new_v)
    assert new_k.stride(-1) == 1 and new_v.stride(-1) == 1, "last dimension must be contiguous"
    packed = cu_seqlens is not None
    p.new_k, p.new_v = new_k.data_ptr(), new_v.data_ptr()
    p.new_k_stride, p.new_v_stride = _strides3(new_k, packed), _strides3(new_v, packed)
    _lib.launch(dev, _lib.lib().rswa_cache_append, p)


def kv_cache_attn(
    q: torch.Tensor,
    cache: KVCache,
    page_table: torch.Tensor,
    seqlens: torch.Tensor,
    window_size: int = -1,
    cu_seqlens: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    *,
    num_sink_tokens: int = 0,
    return_lse: bool = False,
):
    """Attention of the sequences' last tokens over their caches; same mask as ``ring_streaming_llm_attn``.

    ``q``: ``[batch, seq, heads, dim]``, or packed ``[tokens, heads, dim]`` with ``cu_seqlens``; bf16 or
    fp16.  ``seqlens`` counts all tokens of a sequence, those of ``q`` among them.  Each query sees its
    own token and the ``window_size`` before it (negative: all) and the first ``num_sink_tokens``.
    Codes are read in the type of ``q``: what bf16 rows have written beyond fp16's range is infinite to
    fp16 queries.  A NaN or an infinite value reaches the rows that see it and no others.  Rows ahead of
    a pack's first sequence and behind its last are not written.  Returns the output, shape and dtype of
    ``q``, and with ``return_lse`` the log-sum-exp, fp32 ``[batch, heads, seq]`` (``[heads, tokens]`` of a
    pack), as ``merge_attn_out`` takes it.  Rows that see nothing: 0 and ``-inf``."""
    if torch.compiler.is_dynamo_compiling():
        return _uncompiled(kv_cache_attn, q, cache, page_table, seqlens, window_size, cu_seqlens, softmax_scale,
                           num_sink_tokens=num_sink_tokens, return_lse=return_lse)
    calls = _calls(cache)
    if calls is not None:
        got = calls.cache_attn(q, cache, page_table, seqlens, window_size, cu_seqlens, softmax_scale,
                               num_sink_tokens, return_lse)
        if got is not None:
            return got
    _no_grad(*cache, q)
    out, lse = _attn(q, *cache, page_table, seqlens, _window(window_size), cu_seqlens, _scale(softmax_scale),
                     _sinks(num_sink_tokens), bool(return_lse))
    return (out, lse) if return_lse else out


def _results(q, packed, return_lse):
    out = q.new_empty(q.shape)
    if not return_lse:
        return out, q.new_empty(0, dtype=torch.float32)
    qs = q.shape
    return out, q.new_empty((qs[1], qs[0]) if packed else (qs[0], qs[2], qs[1]), dtype=torch.float32)


@_operator(f"cache_attn(Tensor q, {_CACHE}, Tensor page_table, Tensor seqlens, int window_size, Tensor? cu_seqlens, "
           "float? softmax_scale, int num_sink_tokens, bool return_lse) -> (Tensor, Tensor)",
           lambda q, *rest: _results(q, rest[7] is not None, rest[10]))
def _attn(q, k, v, k_scale, v_scale, page_table, seqlens, window_size, cu_seqlens, softmax_scale, num_sink_tokens,
          return_lse):
    """(``lse`` is an empty tensor where it is not wanted)"""
    p, dev = _cache_params((k, v, k_scale, v_scale), page_table, seqlens, q, cu_seqlens)
    packed = cu_seqlens is not None
    _query_params(p, q, p.heads_kv, softmax_scale, window_size, num_sink_tokens, packed)
    out, lse = _results(q, packed, return_lse)
    if q.numel() > 0:
        if p.max_pages == 0:  # no keys at all
            out.zero_()
            lse.fill_(float("-inf"))
            return out, lse
        p.out, p.out_stride = out.data_ptr(), _strides3(out, packed)
        if return_lse:
            p.lse, p.lse_stride = lse.data_ptr(), _strides3(lse, packed)
        L = _lib.lib()
        size = int(L.rswa_cache_attn_workspace_bytes(p))
        if size:
            workspace = q.new_empty(size, dtype=torch.uint8)
            p.workspace, p.workspace_bytes = workspace.data_ptr(), size
        _lib.launch(dev, L.rswa_cache_attn, p)
    return out, lse


def kv_cache_weights(
    q: torch.Tensor,
    cache: KVCache,
    page_table: torch.Tensor,
    seqlens: torch.Tensor,
    lse: torch.Tensor,
    weights: torch.Tensor,
    window_size: int = -1,
    cu_seqlens: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    *,
    num_sink_tokens: int = 0,
) -> None:
    """Add to ``weights`` how much attention each cached key got from ``q``: the softmax weights
    summed over the rows that see it and the query heads of its kv head's group.

    ``lse`` is what ``kv_cache_attn(..., return_lse=True)`` returned for the same arguments; ``weights``
    fp32 ``[batch, kv_heads, n]``, entry ``j`` that of token ``j`` (tokens from ``n`` on are passed over)."""
    if torch.compiler.is_dynamo_compiling():
        return _uncompiled(kv_cache_weights, q, cache, page_table, seqlens, lse, weights, window_size, cu_seqlens,
                           softmax_scale, num_sink_tokens=num_sink_tokens)
    calls = _calls(cache)
    if calls is not None and calls.cache_weights(q, cache, page_table, seqlens, lse, weights, window_size, cu_seqlens,
                                                 softmax_scale, num_sink_tokens):
        return
    _no_grad(*cache, q, lse, weights)
    _weights(weights, q, *cache, page_table, seqlens, lse, _window(window_size), cu_seqlens, _scale(softmax_scale),
             _sinks(num_sink_tokens))


@_operator(f"cache_weights(Tensor(a!) weights, Tensor q, {_CACHE}, Tensor page_table, Tensor seqlens, Tensor lse, "
           "int window_size, Tensor? cu_seqlens, float? softmax_scale, int num_sink_tokens) -> ()", lambda *_: None)
def _weights(weights, q, k, v, k_scale, v_scale, page_table, seqlens, lse, window_size, cu_seqlens, softmax_scale,
             num_sink_tokens):
    p, dev = _cache_params((k, v, k_scale, v_scale), page_table, seqlens, q, cu_seqlens)
    packed = cu_seqlens is not None
    _query_params(p, q, p.heads_kv, softmax_scale, window_size, num_sink_tokens, packed)
    qs = q.shape
    assert lse.dtype == torch.float32 and tuple(lse.shape) == (
        (qs[1], qs[0]) if packed else (qs[0], qs[2], qs[1])), (
        "lse must be fp32 [batch, heads, seq] ([heads, tokens] when packed)")
    _weights_params(p, k, weights)
    _lib.require_device(q, lse)
    if q.numel() > 0 and p.max_pages > 0:
        p.lse, p.lse_stride = lse.data_ptr(), _strides3(lse, packed)
        _lib.launch(dev, _lib.lib().rswa_cache_weights, p)


def _weights_params(p, k, weights):
    assert weights.dtype == torch.float32 and weights.dim() == 3 and weights.shape[:2] == (p.batch, p.heads_kv), (
        "weights must be fp32 [batch, kv_heads, n]")
    assert _dense_from(weights, 2), "last dimension must be contiguous"
    _fit(weights.shape[2])
    span = weights.shape[2]  # of what the inner of the two strides has walked over
    for size, step in sorted(zip(weights.shape[:2], weights.stride()), key=lambda d: d[1]):
        assert size <= 1 or step >= span, "the sums of different heads overlap"
        span += max(0, size - 1) * step
    _lib.require_device(k, weights)
    p.weights, p.weights_stride, p.weights_len = weights.data_ptr(), weights.stride()[:2], weights.shape[2]


def kv_cache_evict(
    cache: KVCache,
    weights: torch.Tensor,
    page_table: torch.Tensor,
    seqlens: torch.Tensor,
    new_page_table: torch.Tensor,
    budget: int,
    *,
    num_sink_tokens: int = 0,
    num_recent: int = 0,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cut every sequence to at most ``budget`` tokens, for each kv head by itself.

    Kept are the first ``num_sink_tokens``, the last ``num_recent``, and of the others those with the
    largest ``weights`` (of equal ones the earlier; NaN counts as the least), in their order.  Tokens whose
    page is not there are not kept, and a sequence's new length does not count them.  The others move
    to the pages of ``new_page_table`` (int32 ``[batch, n]``, room for ``budget`` tokens), each page at the
    scale that fits its values; the old pages are only read, so that sequences may share them, and none
    of them may be among the new ones, nor a new one in two rows.  Tokens without a weight (``n`` below the
    length) weigh 0.  Returns the new ``seqlens``, the kept tokens' weights (shape of
    ``weights``, zeros behind) and their old numbers, int32 ``[batch, kv_heads, budget]`` (``-1`` behind).
    From then on a token's number is its place among the kept ones, for windows too."""
    if torch.compiler.is_dynamo_compiling():
        return _uncompiled(kv_cache_evict, cache, weights, page_table, seqlens, new_page_table, budget,
                           num_sink_tokens=num_sink_tokens, num_recent=num_recent)
    calls = _calls(cache)
    if calls is not None:
        got = calls.cache_evict(cache, weights, page_table, seqlens, new_page_table, budget, num_sink_tokens,
                                num_recent)
        if got is not None:
            return got
    _fit(budget)
    assert budget > 0 and num_sink_tokens >= 0 and num_recent >= 0
    assert num_sink_tokens + num_recent <= budget, "budget must hold the sinks and the recent tokens"
    _no_grad(*cache, weights)
    return _evict(*cache, weights, page_table, seqlens, new_page_table, int(budget), int(num_sink_tokens), int(num_recent))


def _cut(weights, seqlens, heads, budget):
    """Lengths, weights and numbers of what stays."""
    return (torch.empty_like(seqlens), weights.new_empty(weights.shape),
            seqlens.new_empty((seqlens.shape[0], heads, budget)))


@_operator(f"cache_evict({_WRITTEN_CACHE}, Tensor weights, Tensor page_table, Tensor seqlens, Tensor new_page_table, "
           "int budget, int num_sink_tokens, int num_recent) -> (Tensor, Tensor, Tensor)",
           lambda k, v, ks, vs, weights, table, seqlens, new, budget, *_: _cut(weights, seqlens, k.shape[1], budget))
def _evict(k, v, k_scale, v_scale, weights, page_table, seqlens, new_page_table, budget, num_sink_tokens, num_recent):
    p, dev = _cache_params((k, v, k_scale, v_scale), page_table, seqlens, None, None)
    _weights_params(p, k, weights)
    assert new_page_table.dim() == 2 and new_page_table.dtype == torch.int32 and \
        new_page_table.shape[0] == p.batch, "new_page_table must be int32 [batch, n]"
    assert _dense_from(new_page_table, 1), "the entries of a row of new_page_table must be adjacent"
    _fit(new_page_table.shape[1])
    _lib.require_device(k, new_page_table)
    new_seqlens, new_weights, kept = _cut(weights, seqlens, p.heads_kv, budget)
    p.num_sink, p.num_recent, p.budget = num_sink_tokens, num_recent, budget
    p.new_page_table, p.new_page_table_stride = new_page_table.data_ptr(), new_page_table.stride(0)
    p.new_max_pages = new_page_table.shape[1]
    p.new_seqlens, p.new_weights, p.kept = new_seqlens.data_ptr(), new_weights.data_ptr(), kept.data_ptr()
    _lib.launch(dev, _lib.lib().rswa_cache_evict, p)
    return new_seqlens, new_weights, kept
