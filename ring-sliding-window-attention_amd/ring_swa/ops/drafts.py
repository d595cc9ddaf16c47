"""A step of drafted tokens over the 8-bit paged cache.  No counterpart in the upstream package.

A draft model proposes, for each sequence, a tree of tokens that may follow; the target model looks at all of them at
once, and those that its probabilities take are kept, as if it had drawn them one by one::

    tree = draft_tree(parents)                                   # once a step
    position = held[:, None] + tree.depths                       # of every node
    for layer in ...:
        out = kv_cache_tree_attn(q, k, v, tree, cache, page_table, held, window, num_sink_tokens=4)
    path, accepted, token = verify_drafts(tree, tokens, target, draft, uniforms)
    for layer in ...:
        kv_cache_accept(cache, k, v, path, page_table, held)     # the keys and values of what is kept
    held += accepted                                             # token is the next tree's root

Nodes are rows of their sequence, parents ahead of their children: ``[batch, nodes, ...]``, or packed ``[tokens, ...]``
with ``cu_seqlens``, as in the other calls over the cache; trees of different sizes are packed, or padded with nodes that
are not there.  Node 0 is the root, the token chosen last, whose key is not in the cache yet.  The nodes' own keys and values
are taken as they are, in 16 bits: a draft that is not kept never touches the cache, and no page's scale grows with it.

All is found on the device; nothing is read back.  There is no backward.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from .. import _lib
from .kv_cache import (KVCache, _CACHE, _WRITTEN_CACHE, _cache_params, _calls, _dense_from, _fit, _new_rows, _no_grad,
                       _operator, _query_params, _results, _scale, _sinks, _strides3, _uncompiled, _window)

MAX_NODES = 1024


class DraftTree(NamedTuple):
    """What ``draft_tree`` makes of ``parents``: ``parents`` int32, -2 for nodes that are not there; ``depths`` int32, the
    number of a node's ancestors, -1 for nodes that are not there; ``ancestors`` int64 ``[..., words]``, bit ``j % 64`` of
    word ``j / 64`` set for ``j`` = the node itself and its ancestors.  Trees of a batch may share memory (stride 0)."""

    parents: torch.Tensor
    depths: torch.Tensor
    ancestors: torch.Tensor


def _ints(t, rows, what):
    """An int32 tensor of ``rows`` entries in a row; the stride between sequences."""
    assert t.dtype == torch.int32 and tuple(t.shape) == tuple(rows), f"{what} must be int32 {list(rows)}"
    assert _dense_from(t, t.dim() - 1), f"{what}: the entries of a sequence must be adjacent"
    return t.stride(0) if t.dim() == 2 else 0


def _cu(cu_seqlens, like):
    assert cu_seqlens.dtype == torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.shape[0] >= 1 and \
        cu_seqlens.is_contiguous(), "cu_seqlens must be a contiguous int32 tensor [batch + 1]"
    _lib.require_device(like, cu_seqlens)
    return cu_seqlens.shape[0] - 1, cu_seqlens.data_ptr()


def draft_tree(
    parents: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    *,
    max_nodes: Optional[int] = None,
) -> DraftTree:
    """Depths and ancestors of the nodes of trees.

    ``parents``: int32 ``[batch, nodes]``, or packed ``[tokens]`` with ``cu_seqlens`` and ``max_nodes``, the most nodes
    that a sequence may have (at most 1024).  A parent is a lower node of the sequence, or -1: the last cached token.  A
    node whose chain of parents does not fall step by step and end at -1 is not there (padding: -2), nor is one from
    ``max_nodes`` on.  Rows of a pack that are no sequence's are left as ``torch.empty`` has them."""
    if torch.compiler.is_dynamo_compiling():
        return _uncompiled(draft_tree, parents, cu_seqlens, max_nodes=max_nodes)
    if max_nodes is None:
        assert cu_seqlens is None, "a pack needs max_nodes"
        max_nodes = max(1, parents.shape[-1])
    calls = _calls((parents,))
    if calls is not None:
        got = calls.draft_tree(parents, cu_seqlens, max_nodes)
        if got is not None:
            return DraftTree(*got)
    return DraftTree(*_tree(parents, cu_seqlens, int(max_nodes)))


def _tree_of(parents, max_nodes):
    return (parents.new_empty(parents.shape), parents.new_empty(parents.shape),
            parents.new_empty((*parents.shape, (max_nodes + 63) // 64), dtype=torch.int64))


@_operator("draft_tree(Tensor parents, Tensor? cu_seqlens, int max_nodes) -> (Tensor, Tensor, Tensor)",
           lambda parents, cu, max_nodes: _tree_of(parents, max_nodes))
def _tree(parents, cu_seqlens, max_nodes):
    assert 1 <= max_nodes <= MAX_NODES, f"max_nodes must be between 1 and {MAX_NODES}"
    dev = _lib.require_device(parents)
    p = _lib.TreeParams()
    assert parents.dim() == (2 if cu_seqlens is None else 1), "parents must be [batch, nodes], or [tokens] with cu_seqlens"
    _fit(*parents.shape)
    p.parents, p.parents_stride = parents.data_ptr(), _ints(parents, parents.shape, "parents")
    if cu_seqlens is None:
        p.batch, p.nodes = parents.shape
        assert p.nodes <= max_nodes, f"more than max_nodes ({max_nodes}) nodes"
    else:
        p.batch, p.cu_seqlens = _cu(cu_seqlens, parents)
        p.total = parents.shape[0]
    p.max_nodes = max_nodes
    made = _tree_of(parents, max_nodes)
    p.tree_parents, p.depths, p.ancestors = (t.data_ptr() for t in made)
    _lib.launch(dev, _lib.lib().rswa_draft_tree, p)
    return made


def kv_cache_tree_attn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    tree: DraftTree,
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
    """Attention of a tree's nodes over their sequences' caches and over each other.

    ``q``: ``[batch, nodes, heads, dim]``, ``k``, ``v``: ``[batch, nodes, kv_heads, dim]`` (packed ``[tokens, ...]`` with
    ``cu_seqlens``), bf16 or fp16; ``tree``: of ``draft_tree`` for the same rows (depths are below their number).  ``seqlens`` counts the tokens in the
    cache, the nodes not among them; node ``i`` is token ``seqlens + depth(i)``.  It sees the cached tokens, itself and its
    ancestors, of these the ``window_size`` before it (negative: all) and the first ``num_sink_tokens``.  Everything else
    is as in ``kv_cache_attn``; nodes that are not there: 0 and ``-inf``."""
    if torch.compiler.is_dynamo_compiling():
        return _uncompiled(kv_cache_tree_attn, q, k, v, tree, cache, page_table, seqlens, window_size, cu_seqlens,
                           softmax_scale, num_sink_tokens=num_sink_tokens, return_lse=return_lse)
    calls = _calls(cache)
    if calls is not None:
        got = calls.cache_tree_attn(q, k, v, tree, cache, page_table, seqlens, window_size, cu_seqlens, softmax_scale,
                                    num_sink_tokens, return_lse)
        if got is not None:
            return got
    _no_grad(*cache, q, k, v)
    _, depths, ancestors = tree
    out, lse = _tree_attn(q, k, v, depths, ancestors, *cache, page_table, seqlens, _window(window_size), cu_seqlens,
                          _scale(softmax_scale), _sinks(num_sink_tokens), bool(return_lse))
    return (out, lse) if return_lse else out


@_operator(f"cache_tree_attn(Tensor q, Tensor new_k, Tensor new_v, Tensor depths, Tensor ancestors, {_CACHE}, "
           "Tensor page_table, Tensor seqlens, int window_size, Tensor? cu_seqlens, float? softmax_scale, "
           "int num_sink_tokens, bool return_lse) -> (Tensor, Tensor)",
           lambda q, *rest: _results(q, rest[11] is not None, rest[14]))
def _tree_attn(q, new_k, new_v, depths, ancestors, k, v, k_scale, v_scale, page_table, seqlens, window_size, cu_seqlens,
               softmax_scale, num_sink_tokens, return_lse):
    """(``lse`` is an empty tensor where it is not wanted)"""
    c, dev = _cache_params((k, v, k_scale, v_scale), page_table, seqlens, q, cu_seqlens)
    packed = cu_seqlens is not None
    _query_params(c, q, c.heads_kv, softmax_scale, window_size, num_sink_tokens, packed)
    assert new_k.shape[:-2] == q.shape[:-2] and new_k.shape[-1] == q.shape[-1] and new_k.dtype == q.dtype, (
        "q, k and v must have the same rows, head_dim and dtype")
    _new_rows(c, new_k, new_v, packed)
    rows = q.shape[:-2]
    p = _lib.DraftParams()
    p.depths, p.depths_stride = depths.data_ptr(), _ints(depths, rows, "depths")
    assert ancestors.dtype == torch.int64 and tuple(ancestors.shape[:-1]) == tuple(rows), (
        f"ancestors must be int64 {[*rows, 'words']}")
    words = ancestors.shape[-1]
    assert 1 <= words <= MAX_NODES // 64 and (packed or rows[1] <= 64 * words), (
        f"ancestors must have a bit for every node, and at most {MAX_NODES}")
    assert _dense_from(ancestors, ancestors.dim() - 2), "ancestors: the words of a sequence must be adjacent"
    p.ancestors, p.ancestors_stride, p.words = ancestors.data_ptr(), 0 if packed else ancestors.stride(0), words
    _lib.require_device(q, new_k, depths, ancestors)
    out, lse = _results(q, packed, return_lse)
    if q.numel() > 0:
        c.out, c.out_stride = out.data_ptr(), _strides3(out, packed)
        if return_lse:
            c.lse, c.lse_stride = lse.data_ptr(), _strides3(lse, packed)
        p.cache = c
        L = _lib.lib()
        size = int(L.rswa_cache_tree_attn_workspace_bytes(p))
        if size:
            workspace = q.new_empty(size, dtype=torch.uint8)
            p.cache.workspace, p.cache.workspace_bytes = workspace.data_ptr(), size
        _lib.launch(dev, L.rswa_cache_tree_attn, p)
    return out, lse


def verify_drafts(
    tree: DraftTree,
    tokens: torch.Tensor,
    target: torch.Tensor,
    draft: Optional[torch.Tensor],
    uniforms: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which nodes the target's probabilities take, and the token behind them.

    ``tokens``: int32 or int64 ``[batch, nodes]`` (packed ``[tokens]`` with ``cu_seqlens``; the root's is not looked at);
    ``target``: ``[batch, nodes, vocab]``, the probabilities behind each node, fp32, bf16 or fp16; ``draft``: the same of
    the draft model, which the children of a node were drawn from, independently, or None: the children were named outright
    (its likeliest tokens, say); ``uniforms``: fp32 ``[batch, nodes]``, numbers from [0, 1).  With ``p`` and ``q`` the rows of
    the node reached, its children are tried in their order: with ``draft`` a token ``x`` is taken if ``uniform * S * q(x) <
    p(x)``, S = 1 for the first, and a rejected one leaves ``max(0, p - S * q)`` for ``p`` and its sum for S; without, if
    ``uniform * S < p(x)``, and a rejected one leaves ``p`` without it and ``S - p(x)`` for S.  What is left of ``p`` when no child
    is taken is what the next token is drawn from: the least ``x`` at which its running sum is above the root's uniform times its
    sum (``p`` itself, where nothing is left of it).  So tokens are distributed as if drawn from the target one after the other,
    if rows sum to 1.  They are not made to: a token's distribution is off (in total variation) by no more than what the
    target's sum differs from 1, and the draft's for each child tried (rows rounded to 16 bits: some 1e-3); without ``draft`` a
    child that has all of S is taken, whatever is left of ``p`` beside it.  Sums and comparisons are in 64 bits;
    probabilities that are not positive count as 0, and none may be infinite.  At most 2^22 tokens of vocabulary, and fewer
    than 2^16 sequences.

    Returns the nodes taken, root first (int32 ``[batch, nodes]``, of a pack ``[batch, 64 * words]``; -1 behind), their
    number (int32 ``[batch]``) and the next token (type of ``tokens``; -1 where the target has no probabilities, or the
    root is not there, whose number of nodes is 0 then)."""
    if torch.compiler.is_dynamo_compiling():
        return _uncompiled(verify_drafts, tree, tokens, target, draft, uniforms, cu_seqlens)
    calls = _calls((target,))
    if calls is not None:
        got = calls.verify_drafts(tree, tokens, target, draft, uniforms, cu_seqlens)
        if got is not None:
            return got
    _no_grad(*(t for t in (target, draft, uniforms) if t is not None))
    return _verify(tree[0], tokens, target, draft, uniforms, cu_seqlens, 64 * tree[2].shape[-1])


def _choice(tokens, cu_seqlens, max_nodes):
    batch, width = tokens.shape if cu_seqlens is None else (cu_seqlens.shape[0] - 1, max_nodes)
    return (tokens.new_empty((batch, width), dtype=torch.int32), tokens.new_empty(batch, dtype=torch.int32),
            tokens.new_empty(batch))


@_operator("verify_drafts(Tensor parents, Tensor tokens, Tensor target, Tensor? draft, Tensor uniforms, "
           "Tensor? cu_seqlens, int max_nodes) -> (Tensor, Tensor, Tensor)",
           lambda parents, tokens, target, draft, uniforms, cu, max_nodes: _choice(tokens, cu, max_nodes))
def _verify(parents, tokens, target, draft, uniforms, cu_seqlens, max_nodes):
    packed = cu_seqlens is not None
    assert target.dim() == (2 if packed else 3) and target.shape[-1] > 0, (
        "target must be [batch, nodes, vocab], or [tokens, vocab] with cu_seqlens")
    assert target.dtype in (torch.float32, torch.bfloat16, torch.float16), "target must be fp32, bf16 or fp16"
    assert 1 <= max_nodes <= MAX_NODES, f"ancestors must have a bit for every node, and at most {MAX_NODES}"
    dev = _lib.require_device(*(t for t in (target, draft, parents, tokens, uniforms) if t is not None))
    rows = target.shape[:-1]
    _fit(*target.shape)
    p = _lib.VerifyParams()
    p.dtype = _lib.dtype_code(target)
    assert tokens.dtype in (torch.int32, torch.int64), "tokens must be int32 or int64"
    p.token_bytes = tokens.element_size()
    p.parents, p.parents_stride = parents.data_ptr(), _ints(parents, rows, "parents")
    assert tokens.shape == rows and _dense_from(tokens, tokens.dim() - 1), "tokens must be like parents"
    assert uniforms.dtype == torch.float32 and uniforms.shape == rows and _dense_from(uniforms, uniforms.dim() - 1), (
        "uniforms must be fp32, and like parents")
    p.tokens, p.tokens_stride = tokens.data_ptr(), 0 if packed else tokens.stride(0)
    p.uniforms, p.uniforms_stride = uniforms.data_ptr(), 0 if packed else uniforms.stride(0)
    if packed:
        p.batch, p.cu_seqlens = _cu(cu_seqlens, target)
        p.total = rows[0]
    else:
        p.batch, p.nodes = rows
    for t in (target, draft):
        if t is not None:
            assert t.shape == target.shape and t.dtype == target.dtype, "target and draft must be alike"
            assert t.stride(-1) == 1 or t.shape[-1] == 1, "last dimension must be contiguous"
    p.vocab, p.max_nodes = target.shape[-1], max_nodes
    strides = (lambda t: (0, t.stride(0))) if packed else (lambda t: t.stride()[:2])
    p.target, p.target_stride = target.data_ptr(), strides(target)
    if draft is not None:
        p.draft, p.draft_stride = draft.data_ptr(), strides(draft)
    made = _choice(tokens, cu_seqlens, max_nodes)
    p.path, p.accepted, p.next_token = (t.data_ptr() for t in made)
    p.path_len = made[0].shape[1]
    L = _lib.lib()
    size = int(L.rswa_verify_drafts_workspace_bytes(p))
    workspace = target.new_empty(size, dtype=torch.uint8)
    p.workspace, p.workspace_bytes = workspace.data_ptr(), size
    _lib.launch(dev, L.rswa_verify_drafts, p)
    return made


def kv_cache_accept(
    cache: KVCache,
    k: torch.Tensor,
    v: torch.Tensor,
    path: torch.Tensor,
    page_table: torch.Tensor,
    seqlens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
) -> None:
    """``kv_cache_append`` of the rows that ``path`` names: ``k[b, path[b, 0]]``, ``k[b, path[b, 1]]``, ... go behind the
    ``seqlens`` tokens that the sequence holds, as many as there are ahead of the row's first entry that is no row of the
    sequence (-1, say).

    ``k``, ``v``: ``[batch, nodes, kv_heads, dim]``, or packed with ``cu_seqlens``; ``path``: int32 ``[batch, n]``, as
    ``verify_drafts`` returns it (a slice ``path[:, :n]`` that holds every path saves a little)."""
    if torch.compiler.is_dynamo_compiling():
        return _uncompiled(kv_cache_accept, cache, k, v, path, page_table, seqlens, cu_seqlens)
    calls = _calls(cache)
    if calls is not None and calls.cache_accept(cache, k, v, path, page_table, seqlens, cu_seqlens):
        return
    _no_grad(*cache, k, v)
    _accept(*cache, k, v, path, page_table, seqlens, cu_seqlens)


@_operator(f"cache_accept({_WRITTEN_CACHE}, Tensor new_k, Tensor new_v, Tensor path, Tensor page_table, Tensor seqlens, "
           "Tensor? cu_seqlens) -> ()", lambda *_: None)
def _accept(k, v, k_scale, v_scale, new_k, new_v, path, page_table, seqlens, cu_seqlens):
    p = _lib.DraftParams()
    c, dev = _cache_params((k, v, k_scale, v_scale), page_table, seqlens, new_k, cu_seqlens)
    _new_rows(c, new_k, new_v, cu_seqlens is not None)
    assert path.dim() == 2, "path must be int32 [batch, n]"
    _fit(path.shape[1])
    p.path, p.path_stride = path.data_ptr(), _ints(path, (c.batch, path.shape[1]), "path")
    p.path_len = path.shape[1]
    _lib.require_device(k, path)
    p.cache = c
    _lib.launch(dev, _lib.lib().rswa_cache_accept, p)
