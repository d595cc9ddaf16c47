"""The cache operators of this repository as they are measured: serving from an 8-bit paged cache.

``kv_cache_append`` (new keys and values into pages of e4m3 with a power-of-two scale per page and head),
``kv_cache_attn`` (window + sink attention of new queries over the cache), ``kv_cache_weights`` (running sums of
the softmax weights of every cached key) and ``kv_cache_evict`` (keeps the sinks, the recent and the heaviest
keys).  A case is one call.  Where ``own`` is false the same call is computed with elementary torch operations.

The cache: ``k`` e4m3 ``[pages, kv_heads, page, dim]``, ``v`` e4m3 ``[pages, kv_heads, page / 16, dim, 16]``
(the 16 keys of a group are adjacent), ``k_scale`` / ``v_scale`` e8m0 ``[pages, kv_heads]``; a sequence's pages
are named by its row of ``page_table``.  Keys and values are N(0, 1) (projected activations after normalisation)
with an amplitude of its own for every page; sink keys are four times as large, which is what makes a token a
sink.  Pages lie in no order, as an allocator leaves them.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_E4M3 = torch.float8_e4m3fn
_E8M0 = torch.float8_e8m0fnu


def listed():
    return [
        # The smallest call: one sequence's new token goes into the cache.  Launch and host work.
        dict(name="append_token_1", kind="append", batch=1, new=1, shortest=5000, longest=5000, lens=0,
             packed=False, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # A decode batch appends one token per sequence, at ragged lengths.
        dict(name="append_token_128", kind="append", batch=128, new=1, shortest=16, longest=32768, lens=1,
             packed=False, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # A pack of prompts goes into an empty cache.
        dict(name="append_prompts_32k", kind="append", batch=8, new=16384, shortest=0, longest=0, lens=2,
             packed=True, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # One sequence answers: a single token over a cache of an ordinary length.
        dict(name="attn_token_1", kind="attn", batch=1, new=1, shortest=4001, longest=4001, lens=0,
             packed=False, heads=32, kv_heads=8, dim=128, page=64, window=-1, sinks=0, lse=False,
             dtype="bf16"),
        # A full decode batch with ragged caches, every key attended.
        dict(name="attn_token_64", kind="attn", batch=64, new=1, shortest=256, longest=32768, lens=3,
             packed=False, heads=32, kv_heads=8, dim=128, page=64, window=-1, sinks=0, lse=False,
             dtype="bf16"),
        # A streaming model with sinks and a window: odd group (28 over 4 heads), head_dim 64, fp16, small pages.
        dict(name="attn_stream_128", kind="attn", batch=128, new=1, shortest=2048, longest=65536, lens=4,
             packed=False, heads=28, kv_heads=4, dim=64, page=16, window=4092, sinks=4, lse=False,
             dtype="fp16"),
        # Five drafted tokens a sequence are verified at once.
        dict(name="attn_draft_16", kind="attn", batch=16, new=5, shortest=1000, longest=16384, lens=5,
             packed=False, heads=32, kv_heads=8, dim=128, page=32, window=4096, sinks=4, lse=True,
             dtype="bf16"),
        # The largest: a chunk of a long prompt against all that came before it.
        dict(name="attn_chunk_2k", kind="attn", batch=1, new=2048, shortest=32768, longest=32768, lens=0,
             packed=False, heads=32, kv_heads=8, dim=128, page=64, window=-1, sinks=0, lse=False,
             dtype="bf16"),
        # A decode batch keeps the running sums that eviction goes by.
        dict(name="weights_token_32", kind="weights", batch=32, new=1, shortest=1024, longest=16384, lens=6,
             packed=False, heads=32, kv_heads=8, dim=128, page=64, window=-1, sinks=0, dtype="bf16"),
        # The last 64 tokens of a long prompt say which of its keys are kept.
        dict(name="weights_prompt_64", kind="weights", batch=1, new=64, shortest=32001, longest=32001, lens=0,
             packed=False, heads=32, kv_heads=8, dim=128, page=64, window=-1, sinks=0, dtype="bf16"),
        # A decode batch is cut back to its budget after 128 tokens.
        dict(name="evict_slack_32", kind="evict", batch=32, shortest=2100, longest=2176, lens=7, budget=2048,
             sinks=4, recent=512, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # Long prompts are cut down to an eighth.
        dict(name="evict_prompt_4", kind="evict", batch=4, shortest=20000, longest=32768, lens=8, budget=4096,
             sinks=4, recent=64, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16"),
    ]


# heads / kv heads, drawn with equal odds
_HEADS = [(4, 4), (8, 2), (12, 12), (16, 4), (28, 4), (32, 8), (32, 32), (32, 1)]


def _spread(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max(work(c)["flops"] for c in listed())
    most_bytes = max(work(c)["bytes"] for c in listed())
    while True:
        case = _draw_any(rng)
        w = work(case)
        if w["flops"] <= most and w["bytes"] <= most_bytes and _plain_bytes(case) <= 12e9:
            return case


def _draw_any(rng):
    kind = rng.choice(["append", "attn", "attn", "attn", "weights", "evict"])
    heads, kv_heads = rng.choice(_HEADS)
    case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128, 128]),
                page=rng.choice([16, 32, 64, 64, 128, 256]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                batch=_spread(rng, 1, 128), lens=rng.randrange(1 << 20))
    shortest = _spread(rng, 1, 16384)
    longest = _spread(rng, shortest, 32768)
    if kind == "evict":
        budget = _spread(rng, 16, longest)
        sinks = min(budget, rng.choice([0, 1, 4]))
        case.update(shortest=shortest, longest=longest, budget=budget, sinks=sinks,
                    recent=rng.randrange(0, budget - sinks + 1))
        return case
    new = rng.choice([1, 1, _spread(rng, 2, 16), _spread(rng, 17, 2048)])
    case.update(new=new, packed=rng.random() < 0.4, shortest=shortest, longest=longest)
    if kind != "append":
        bounded = rng.random() < 0.6
        case.update(window=_spread(rng, 16, 8192) if bounded else -1, sinks=rng.choice([0, 1, 4]) if bounded else 0)
    if kind == "attn":
        case["lse"] = rng.random() < 0.4
    return case


# ---- lengths ----------------------------------------------------------------------------------
def _lengths(case):
    """Tokens held before the call and new tokens, per sequence.  Lengths are spread over their logarithm; in a
    pack the new tokens are, too (continuous batching: some sequences answer, others bring a chunk)."""
    rng = random.Random(case["lens"])
    held = [_spread(rng, case["shortest"], case["longest"]) if case["longest"] else 0 for _ in range(case["batch"])]
    if case["kind"] == "evict":
        return held, [0] * case["batch"]
    new = [_spread(rng, 1, case["new"]) if case["packed"] else case["new"] for _ in range(case["batch"])]
    if case["packed"]:
        new[0] = case["new"]
    if case["kind"] != "append":  # the queries' own keys are in the cache already
        held = [max(h, n) - n for h, n in zip(held, new)]
    return held, new


def _pages(tokens, page):
    return -(-tokens // page)


def _seen(case):
    """Cached keys that a call's queries attend, and (query, key) pairs, over all sequences."""
    keys = pairs = 0
    for h, n in zip(*_lengths(case)):
        w, s = case["window"], case["sinks"]
        if w < 0:
            keys += h + n
            pairs += n * h + n * (n + 1) // 2
            continue
        first = max(0, h - w)
        keys += h + n - first + min(s, first)
        for i in range(n):
            lo = max(0, h + i - w)
            pairs += h + i + 1 - lo + min(s, lo)
    return keys, pairs


def work(case):
    held, new = _lengths(case)
    hq, hk, d, n = case["heads"], case["kv_heads"], case["dim"], sum(new)
    if case["kind"] == "append":
        return {"bytes": 2 * n * hk * d * 3, "flops": 2 * 2 * n * hk * d}
    if case["kind"] == "evict":
        kept = sum(min(h, case["budget"]) for h in held)
        return {"bytes": kept * hk * (4 * d + 4) + 8 * hk * sum(held), "flops": 2 * 2 * kept * hk * d}
    keys, pairs = _seen(case)
    if case["kind"] == "weights":
        return {"bytes": keys * hk * (d + 8) + n * hq * (2 * d + 4), "flops": 2 * d * hq * pairs}
    return {"bytes": keys * hk * 2 * d + n * hq * (4 * d + 4 * case["lse"]), "flops": 4 * d * hq * pairs}


def _plain_bytes(case):
    """The largest tensors of the plain form."""
    held, new = _lengths(case)
    most = max(h + n for h, n in zip(held, new))
    kv = case["batch"] * most * case["kv_heads"] * case["dim"] * 4
    if case["kind"] in ("attn", "weights"):
        return max(kv, case["batch"] * case["heads"] * max(new) * most * 4)
    return kv


# ---- inputs -----------------------------------------------------------------------------------
def _exponents(amax):
    """The least e with ``amax <= 448 * 2**e`` (448: the largest e4m3 value), within [-120, 120]."""
    m, x = torch.frexp(amax)  # amax = m * 2**x, m in [0.5, 1); 448 = 0.875 * 2**9
    return torch.where(amax > 0, x - 9 + (m > 0.875), -120).clamp(-120, 120)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev, dtype = torch.device("cuda"), _DTYPES[case["dtype"]]
    held, new = _lengths(case)
    b, hq, hk, d, p = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    evict = case["kind"] == "evict"
    source = [_pages(h + n, p) for h, n in zip(held, new)]
    target = [_pages(min(h, case["budget"]), p) for h in held] if evict else [0] * b
    total = sum(source) + sum(target) + 1

    # the pool: values with an amplitude for every page and head, at the scale that fits them
    k = torch.empty(total, hk, p, d, dtype=_E4M3, device=dev)
    v = torch.empty(total, hk, p // 16, d, 16, dtype=_E4M3, device=dev)
    k_scale, v_scale = (torch.empty(total, hk, dtype=torch.uint8, device=dev) for _ in range(2))
    order = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    firsts = [sum(source[:i]) for i in range(b)]
    first_pages = order[torch.tensor(firsts, device=dev)].long()
    step = max(1, (1 << 27) // (hk * p * d))
    for t, scale, sink in ((k, k_scale, 4.0), (v, v_scale, 1.0)):
        for at in range(0, total, step):
            part = t[at:at + step]
            x = torch.randn(part.shape, generator=gen, device=dev)
            x *= torch.rand(part.shape[0], hk, *[1] * (x.dim() - 2), generator=gen, device=dev) + 0.5
            if sink != 1.0:
                mine = first_pages[(first_pages >= at) & (first_pages < at + x.shape[0])] - at
                x[mine, :, :4] *= sink
            e = _exponents(x.flatten(2).abs().amax(-1))
            part.copy_((x * torch.exp2(-e.float()).reshape(-1, hk, *[1] * (x.dim() - 2))).to(_E4M3))
            scale[at:at + step] = (e + 127).to(torch.uint8)

    def table(counts, at):
        rows = torch.full((b, max(1, max(counts))), -1, dtype=torch.int32, device=dev)
        n = torch.tensor(counts, device=dev)[:, None]
        place = torch.arange(rows.shape[1], device=dev)[None]
        start = torch.tensor([at + sum(counts[:i]) for i in range(b)], device=dev)[:, None]
        return torch.where(place < n, order[(start + place).clamp(max=total - 1)], rows)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    s = {"case": case, "cache": (k, v, k_scale.view(_E8M0), v_scale.view(_E8M0)),
         "page_table": table(source, 0), "held": ints(held), "seqlens": ints([h + n for h, n in zip(held, new)])}
    packed = case.get("packed", False)
    s["cu_seqlens"] = ints([sum(new[:i]) for i in range(b + 1)]) if packed else None
    lead = (sum(new),) if packed else (b, max(new))

    def rows(heads):
        return torch.randn(*lead, heads, d, generator=gen, device=dev).to(dtype)

    if case["kind"] == "append":
        s["new_k"], s["new_v"] = rows(hk), rows(hk)
    elif case["kind"] == "attn":
        s["q"] = rows(hq)
    elif case["kind"] == "weights":
        s["q"] = rows(hq)
        lse = _scores(s).logsumexp(-1).flatten(1, 2)
        s["lse"] = (_packed_rows(s, lse).t() if packed else lse).contiguous()
        # what a few earlier calls have left: sums of the size of one call's
        n = s["page_table"].shape[1] * p
        s["weights"] = torch.rand(b, hk, n, generator=gen, device=dev) * (4 * max(new) * (hq // hk) / n)
    else:
        s["new_page_table"] = table(target, sum(source))
        # sums of softmax weights: a heavy tail, and keys that nothing has attended
        n = s["page_table"].shape[1] * p
        w = torch.exp(2 * torch.randn(b, hk, n, generator=gen, device=dev)) / n
        s["weights"] = w * (torch.rand(b, hk, n, generator=gen, device=dev) > 0.05)
    return s


# ---- the calls --------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    kind = s["case"]["kind"]
    if kind == "append":
        return _append(s)
    if kind == "attn":
        out, lse = _attention(s)
        return (out, lse) if s["case"]["lse"] else out
    return _weights(s) if kind == "weights" else _evict(s)


def _own(s):
    path = os.path.join(os.getcwd(), "ring-sliding-window-attention_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import ring_swa

    c, cache = s["case"], ring_swa.KVCache(*s["cache"])
    if c["kind"] == "append":
        ring_swa.kv_cache_append(cache, s["new_k"], s["new_v"], s["page_table"], s["held"], s["cu_seqlens"])
        return tuple(cache)
    if c["kind"] == "attn":
        return ring_swa.kv_cache_attn(s["q"], cache, s["page_table"], s["seqlens"], c["window"], s["cu_seqlens"],
                                      num_sink_tokens=c["sinks"], return_lse=c["lse"])
    if c["kind"] == "weights":
        ring_swa.kv_cache_weights(s["q"], cache, s["page_table"], s["seqlens"], s["lse"], s["weights"], c["window"],
                                  s["cu_seqlens"], num_sink_tokens=c["sinks"])
        return s["weights"]
    seqlens, weights, kept = ring_swa.kv_cache_evict(
        cache, s["weights"], s["page_table"], s["held"], s["new_page_table"], c["budget"],
        num_sink_tokens=c["sinks"], num_recent=c["recent"])
    return tuple(cache) + (seqlens, weights, kept)


# ---- plain forms ------------------------------------------------------------------------------
def _codes(pool, *at):
    return pool.view(torch.uint8)[at].view(_E4M3).float()


def _power(scale):
    return torch.exp2(scale.view(torch.uint8).float() - 127)


def _rows_of(s, lead):
    """Sequence and place within the new tokens of each new row, flattened."""
    dev = s["held"].device
    if s["cu_seqlens"] is None:
        at = torch.arange(lead[0] * lead[1], device=dev)
        return at // lead[1], at % lead[1]
    at = torch.arange(lead[0], device=dev)
    seq = torch.searchsorted(s["cu_seqlens"], at.to(torch.int32), right=True) - 1
    return seq, at - s["cu_seqlens"][seq]


def _append(s):
    k, v, k_scale, v_scale = s["cache"]
    p = s["case"]["page"]
    new_k, new_v = s["new_k"].flatten(0, -3), s["new_v"].flatten(0, -3)
    seq, i = _rows_of(s, s["new_k"].shape)
    at = s["held"][seq] + i
    page, slot = s["page_table"][seq, at // p].long(), at % p
    # a sequence's first page may hold older rows, all others start with this call
    first = s["page_table"].gather(1, (s["held"].long() // p)[:, None])[:, 0].long()
    older = s["held"] % p
    for_old = torch.arange(p, device=k.device)[None] < older[:, None]  # [b, p]
    started = torch.zeros(k.shape[0], 1, dtype=torch.bool, device=k.device)
    started[first] = (older > 0)[:, None]
    _append_one(k, k_scale, new_k, page, first, started, (page, slot), for_old[:, None, :, None])
    _append_one(v, v_scale, new_v, page, first, started, (page, slot // 16, slot % 16),
                for_old.unflatten(1, (p // 16, 16))[:, None, :, None, :])
    return k, v, k_scale, v_scale


def _append_one(pool, scale, rows, page, first, started, place, for_old):
    x = rows.float()
    amax = torch.where(x.isfinite(), x.abs(), 0).amax(-1)  # [rows, heads]
    most = torch.zeros(scale.shape, device=x.device).scatter_reduce_(0, page[:, None].expand_as(amax), amax, "amax")
    old = scale.view(torch.uint8).int() - 127
    touched = torch.zeros(scale.shape[0], 1, dtype=torch.bool, device=x.device)
    touched[page] = True
    e = torch.where(started, torch.maximum(_exponents(most), old), _exponents(most))
    e = torch.where(touched, e, old)
    codes = pool.view(torch.uint8)
    held = codes[first]
    ratio = torch.exp2((old - e)[first].float()).reshape(*held.shape[:2], *[1] * (held.dim() - 2))
    again = (held.view(_E4M3).float() * ratio).to(_E4M3).view(torch.uint8)
    codes[first] = torch.where(for_old, again, held)
    code = (x * torch.exp2(-e[page].float())[..., None]).to(_E4M3).view(torch.uint8)
    if len(place) == 2:
        codes[place[0], :, place[1]] = code
    else:
        codes[place[0], :, place[1], :, place[2]] = code
    scale.view(torch.uint8).copy_((e + 127).to(torch.uint8))


def _keys(s):
    """All keys that the table names, ``[b, kv_heads, places, dim]`` in 32 bits."""
    k, _, k_scale, _ = s["cache"]
    pages = s["page_table"].clamp(min=0).long()
    x = _codes(k, pages) * _power(k_scale)[pages][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _values(s):
    _, v, _, v_scale = s["cache"]
    pages = s["page_table"].clamp(min=0).long()
    x = _codes(v, pages) * _power(v_scale)[pages][..., None, None, None]  # [b, n, h, p / 16, d, 16]
    return x.permute(0, 2, 1, 3, 5, 4).flatten(2, 4)


def _padded(s, x, heads_at):
    """Packed rows as ``[b, most, ...]``, rows behind a sequence's last one repeated from somewhere."""
    cu = s["cu_seqlens"].long()
    most = s["case"]["new"]
    at = (cu[:-1, None] + torch.arange(most, device=x.device)).clamp(max=x.shape[heads_at] - 1)
    return x.index_select(heads_at, at.flatten()).unflatten(heads_at, at.shape)


def _scores(s):
    """Scaled scores ``[b, kv_heads, group, new, places]``, -inf where nothing is seen."""
    c = s["case"]
    packed = s["cu_seqlens"] is not None
    q = (_padded(s, s["q"], 0) if packed else s["q"]).float()
    b, n, hq, d = q.shape
    keys = _keys(s)
    hk = keys.shape[1]
    q = q.transpose(1, 2).reshape(b, hk, hq // hk * n, d)
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()).mul_(d ** -0.5)
    scores = scores.view(b, hk, hq // hk, n, -1)
    new = s["cu_seqlens"].diff() if packed else torch.full_like(s["seqlens"], n)
    at = (s["seqlens"] - new)[:, None] + torch.arange(n, device=q.device)  # [b, n]
    j = torch.arange(scores.shape[-1], device=q.device)
    seen = (j <= at[..., None]) & (j < s["seqlens"][:, None, None])
    if c["window"] >= 0:
        seen &= (j >= at[..., None] - c["window"]) | (j < c["sinks"])
    return scores.masked_fill_(~seen[:, None, None], float("-inf"))


def _packed_rows(s, x):
    """``[b, heads, new, ...]`` as the rows of a pack, ``[tokens, heads, ...]``."""
    seq, i = _rows_of(s, s["q"].shape)
    return x[seq, :, i]


def _attention(s):
    scores = _scores(s)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top.isfinite(), top, 0)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log())[..., 0].flatten(1, 2)  # [b, heads, new]
    out = torch.matmul(p.flatten(2, 3), _values(s)).view(*p.shape[:-1], -1)
    out = torch.where(total > 0, out / total, 0).flatten(1, 2)  # [b, heads, new, d]
    if s["cu_seqlens"] is None:
        out = out.transpose(1, 2)
    else:
        out, lse = _packed_rows(s, out), _packed_rows(s, lse).t()
    return out.to(s["q"].dtype).contiguous(), lse.contiguous()


def _weights(s):
    scores = _scores(s)
    b, hk, g, n, _ = scores.shape
    if s["cu_seqlens"] is None:
        lse, mine = s["lse"], None
    else:
        lse = _padded(s, s["lse"], 1).transpose(0, 1)  # [b, heads, new]
        new = s["cu_seqlens"].diff()
        mine = torch.arange(n, device=lse.device) < new[:, None]
    p = scores.sub_(lse.reshape(b, hk, g, n)[..., None]).exp_()
    if mine is not None:
        p.masked_fill_(~mine[:, None, None, :, None], 0)
    s["weights"] += p.sum((2, 3))
    return s["weights"]


def _evict(s):
    c, (k, v, k_scale, v_scale) = s["case"], s["cache"]
    p, budget, lens = c["page"], c["budget"], s["held"]
    w = s["weights"]
    j = torch.arange(w.shape[-1], device=w.device)
    n = lens[:, None, None]
    rank = torch.where((j < c["sinks"]) | (j >= n - c["recent"]), float("inf"), w)
    rank = torch.where(j < n, rank, float("-inf"))
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    count = lens.clamp(max=budget)
    place = torch.arange(order.shape[-1], device=w.device)
    there = place < count[:, None, None]  # [b, 1, budget]
    kept = torch.where(there, order, w.shape[-1]).sort(-1).values
    weights = torch.where(there, w.gather(-1, kept.clamp(max=w.shape[-1] - 1)), 0)
    weights = torch.nn.functional.pad(weights, (0, w.shape[-1] - weights.shape[-1]))
    kept = torch.where(there, kept, -1)
    if kept.shape[-1] < budget:
        kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[-1]), value=-1)
    # the kept rows, [b, heads, places of the new pages, dim], zeros behind the last
    pages = s["new_page_table"].shape[1]
    at = torch.nn.functional.pad(kept, (0, max(0, pages * p - budget)), value=-1)[..., :pages * p]
    real = at >= 0
    at = at.clamp(min=0)
    source = s["page_table"].long().gather(1, (at // p).flatten(1)).view_as(at).clamp(min=0)
    h = torch.arange(k.shape[1], device=w.device)[None, :, None]
    slot = at % p
    target = s["new_page_table"].long()
    for_k = _codes(k, source, h, slot) * _power(k_scale)[source, h][..., None]
    places = torch.arange(k.shape[-1], device=w.device)
    for_v = _codes(v, *(t[..., None] for t in (source, h, slot // 16)), places, slot[..., None] % 16)
    for_v = for_v * _power(v_scale)[source, h][..., None]
    _evict_one(k, k_scale, for_k, real, target, p)
    _evict_one(v, v_scale, for_v, real, target, p)
    return k, v, k_scale, v_scale, count.to(torch.int32), weights, kept.to(torch.int32)


def _evict_one(pool, scale, x, real, target, p):
    x = x.unflatten(2, (-1, p)).transpose(1, 2)  # [b, pages, heads, p, dim]
    real = real.unflatten(2, (-1, p)).transpose(1, 2)[..., None]
    amax = torch.where(x.isfinite() & real, x.abs(), 0).amax((-1, -2))
    e = _exponents(amax)
    code = (x * torch.exp2(-e.float())[..., None, None]).to(_E4M3).view(torch.uint8)
    if pool.dim() == 5:
        code, real = code.unflatten(3, (-1, 16)).transpose(-1, -2), real.unflatten(3, (-1, 16)).transpose(-1, -2)
    bytes_ = pool.view(torch.uint8)
    mine = real.flatten(2).any(-1)  # pages that get a row, [b, pages]
    code = torch.where(real, code, bytes_[target.clamp(min=0)])
    bytes_[target[mine]] = code[mine]
    scale.view(torch.uint8)[target[mine]] = (e[mine] + 127).to(torch.uint8)


# ---- in 64 bits -------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "append":
        return _exact_append(s)
    if kind == "evict":
        return _exact_evict(s)
    return _exact_attention(s)


def _exact_scale(amax):
    e = -120
    if amax > 0:
        e = max(-120, min(120, math.ceil(math.log2(amax / 448))))
        while amax > 448 * 2.0 ** e and e < 120:
            e += 1
        while e > -120 and amax <= 448 * 2.0 ** (e - 1):
            e -= 1
    return 2.0 ** e


def _exact_row(s, which, b, h, j):
    """Codes of places ``j`` of a sequence's head, ``[places, dim]``, and their pages' scales."""
    p = s["case"]["page"]
    pool, scale = s["cache"][which], s["cache"][2 + which]
    page = s["page_table"][b].long()[j // p]
    if which == 0:
        codes = pool.view(torch.uint8)[page, h, j % p]
    else:
        codes = pool.view(torch.uint8)[page, h, (j % p) // 16, :, j % 16]
    return codes.view(_E4M3).double(), torch.pow(2.0, scale.view(torch.uint8)[page, h].double() - 127)


def _exact_append(s):
    """Scales exactly; codes as the quotients that they round."""
    case, p = s["case"], s["case"]["page"]
    held, new = _lengths(case)
    if sum(_pages(n, p) + 1 for n in new) * case["kv_heads"] > 12000:
        return None
    outs = [t.double() for t in s["cache"][:2]]
    scales = [torch.pow(2.0, t.view(torch.uint8).double() - 127) for t in s["cache"][2:]]
    table = s["page_table"].tolist()
    row = 0
    for b in range(case["batch"]):
        for which, source in ((0, s["new_k"]), (1, s["new_v"])):
            x = (source[row:row + new[b]] if case["packed"] else source[b]).double()
            done = 0
            while done < new[b]:
                at = held[b] + done
                page, lo = table[b][at // p], at % p
                n = min(p - lo, new[b] - done)
                part = x[done:done + n].transpose(0, 1)  # [heads, n, dim]
                for h, most in enumerate(part.abs().amax((1, 2)).tolist()):
                    old = float(scales[which][page, h])
                    now = max(_exact_scale(most), old) if lo else _exact_scale(most)
                    if which == 0:
                        outs[0][page, h, :lo] *= old / now
                        outs[0][page, h, lo:lo + n] = part[h] / now
                    else:
                        view = outs[1][page, h].transpose(1, 2).reshape(p, -1).clone()
                        view[:lo] *= old / now
                        view[lo:lo + n] = part[h] / now
                        outs[1][page, h] = view.view(p // 16, 16, -1).transpose(1, 2)
                    scales[which][page, h] = now
                done += n
        row += new[b]
    return (*outs, *scales)


def _exact_evict(s):
    case, p = s["case"], s["case"]["page"]
    held, _ = _lengths(case)
    if sum(_pages(min(n, case["budget"]), p) for n in held) * case["kv_heads"] > 12000:
        return None
    outs = [t.double() for t in s["cache"][:2]]
    scales = [torch.pow(2.0, t.view(torch.uint8).double() - 127) for t in s["cache"][2:]]
    weights = torch.zeros_like(s["weights"], dtype=torch.float64)
    target = s["new_page_table"].tolist()
    for b in range(case["batch"]):
        n, budget = held[b], case["budget"]
        for h in range(case["kv_heads"]):
            w = s["weights"][b, h, :n].double()
            must = set(range(min(n, case["sinks"]))) | set(range(max(0, n - case["recent"]), n))
            values = w.tolist()
            rest = sorted((j for j in range(n) if j not in must), key=lambda j: (-values[j], j))
            keep = sorted(list(must) + rest[:max(0, budget - len(must))]) if n > budget else list(range(n))
            j = torch.tensor(keep, device=w.device)
            weights[b, h, :len(keep)] = w[j]
            for which in (0, 1):
                codes, power = _exact_row(s, which, b, h, j)
                x = codes * power[:, None]
                for i in range(_pages(len(keep), p)):
                    part = x[i * p:(i + 1) * p]
                    now = _exact_scale(float(part.abs().max()))
                    page = target[b][i]
                    scales[which][page, h] = now
                    if which == 0:
                        outs[0][page, h, :part.shape[0]] = part / now
                    else:
                        view = outs[1][page, h].transpose(1, 2).reshape(p, -1).clone()
                        view[:part.shape[0]] = part / now
                        outs[1][page, h] = view.view(p // 16, 16, -1).transpose(1, 2)
    return (*outs, *scales, None, weights, None)


def _exact_attention(s):
    """One sequence and kv head at a time, over the keys that its queries can see."""
    case = s["case"]
    held, new = _lengths(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["batch"] * hk > 4096:
        return None
    q = s["q"]
    dev = q.device
    weights = case["kind"] == "weights"
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    lse = torch.zeros(*((hq, q.shape[0]) if case["packed"] else (q.shape[0], hq, q.shape[1])), dtype=torch.float64,
                      device=dev)
    sums = s["weights"].double() if weights else None
    row = 0
    for b in range(case["batch"]):
        n, end = new[b], held[b] + new[b]
        rows = slice(row, row + n)
        mine = q[rows] if case["packed"] else q[b]
        place = held[b] + torch.arange(n, device=dev)
        j = torch.arange(end, device=dev)
        hidden = j[None] > place[:, None]
        if case["window"] >= 0:
            hidden |= (j[None] < place[:, None] - case["window"]) & (j[None] >= case["sinks"])
        for h in range(hk):
            heads = slice(h * (hq // hk), (h + 1) * (hq // hk))
            codes, power = _exact_row(s, 0, b, h, j)
            x = mine[:, heads].double().transpose(0, 1)  # [group, n, dim]
            z = x @ (codes * power[:, None]).T / math.sqrt(d)
            z = z.masked_fill(hidden, -math.inf)
            if weights:
                given = (s["lse"][heads, rows] if case["packed"] else s["lse"][b, heads]).double()
                sums[b, h, :end] += torch.exp(z - given[..., None]).sum((0, 1))
                continue
            codes, power = _exact_row(s, 1, b, h, j)
            norm = torch.logsumexp(z, -1)
            o = (torch.exp(z - norm[..., None]) @ (codes * power[:, None])).transpose(0, 1)
            if case["packed"]:
                out[rows, heads], lse[heads, rows] = o, norm
            else:
                out[b, :, heads], lse[b, heads] = o, norm
        row += n
    if weights:
        return sums
    return (out, lse) if case["lse"] else out
