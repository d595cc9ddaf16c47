"""The drafting operators of this repository as they are measured: a step of drafted tokens over the 8-bit paged cache.

``draft_tree`` (parents of drafted tokens to depths and ancestor bits), ``kv_cache_tree_attn`` (attention of a tree of
drafted tokens over the cache and over each other), ``verify_drafts`` (which of the drafts the target's probabilities
take, from given random numbers, and the token behind them), ``kv_cache_accept`` (the taken drafts' keys and values
into the cache) and ``kv_cache_read`` (a cached range back in 16 bits).  A case is one call.  Where ``own`` is false
the same call is computed with elementary torch operations.

A tree's nodes are rows of their sequence in an order in which parents come first.  ``parents`` (int32) names a node's
parent, -1 that of a node behind the last cached token; a node whose chain does not end at -1, or does not fall, is not
there (padding has -2).  Node 0 is the last token that was chosen, whose keys are not in the cache yet; the others are
drafts.  ``ancestors`` (int64) has a bit for each node, set for the node itself and its ancestors, 64 to a word.

The cache: ``k`` e4m3 ``[pages, kv_heads, page, dim]``, ``v`` e4m3 ``[pages, kv_heads, page / 16, dim, 16]`` (the 16
keys of a group are adjacent), ``k_scale`` / ``v_scale`` e8m0 ``[pages, kv_heads]``; a sequence's pages are named by its
row of ``page_table``.  Keys and values are N(0, 1) (projected activations after normalisation) with an amplitude of its
own for every page; sink keys are four times as large.  Pages lie in no order, as an allocator leaves them.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_E4M3 = torch.float8_e4m3fn
_E8M0 = torch.float8_e8m0fnu


def listed():
    return [
        # The smallest tree: one sequence, 32 drafts.  Launch and host work.
        dict(name="tree_1", kind="tree", batch=1, nodes=32, width=16, lens=0, packed=False),
        # A serving batch with trees of different sizes in a pack, chains of hundreds among what it has to hold.
        dict(name="tree_packed_256", kind="tree", batch=256, nodes=512, width=8, lens=1, packed=True),
        # One sequence answers: 32 drafts over a cache of an ordinary length.
        dict(name="attn_1", kind="attn", batch=1, nodes=32, width=16, lens=0, packed=False, shortest=4001, longest=4001,
             heads=32, kv_heads=8, dim=128, page=64, window=-1, sinks=0, lse=False, dtype="bf16"),
        # A streaming model with sinks and a window, ragged trees in a pack: odd group (28 over 4 heads), head_dim 64,
        # fp16, small pages.
        dict(name="attn_stream_64", kind="attn", batch=64, nodes=24, width=6, lens=2, packed=True, shortest=2048,
             longest=65536, heads=28, kv_heads=4, dim=64, page=16, window=4092, sinks=4, lse=True, dtype="fp16"),
        # The largest: a full batch with 64 drafts a sequence (padded trees) and every key attended.
        dict(name="attn_32", kind="attn", batch=32, nodes=64, width=24, lens=3, packed=False, shortest=512, longest=16384,
             heads=32, kv_heads=8, dim=128, page=64, window=-1, sinks=0, lse=False, dtype="bf16"),
        # A chain of five drafts behind the last token, one sequence, 32-bit probabilities.
        dict(name="verify_chain_1", kind="verify", batch=1, nodes=6, width=1, lens=0, packed=False, vocab=131072,
             sampled=True, dtype="fp32"),
        # Trees of drafts drawn from the draft model: rejected siblings leave a residual that the next is tried against.
        dict(name="verify_tree_32", kind="verify", batch=32, nodes=32, width=10, lens=4, packed=False, vocab=32768,
             sampled=True, dtype="fp32"),
        # Trees of a draft model's likeliest tokens (no probabilities to divide by), ragged in a pack, 16 bits, odd vocabulary.
        dict(name="verify_top_64", kind="verify", batch=64, nodes=40, width=10, lens=5, packed=True, vocab=50001,
             sampled=False, dtype="bf16"),
        # One sequence's accepted drafts go into the cache.
        dict(name="accept_1", kind="accept", batch=1, nodes=32, lens=0, packed=False, shortest=5000, longest=5000, heads=32,
             kv_heads=8, dim=128, page=64, dtype="bf16"),
        # A batch's accepted drafts, paths of 1 to 12 among trees of up to 64.
        dict(name="accept_128", kind="accept", batch=128, nodes=64, lens=6, packed=False, shortest=16, longest=32768, heads=32,
             kv_heads=8, dim=128, page=64, dtype="bf16"),
        # A page or two of one sequence back in 16 bits.
        dict(name="read_1", kind="read", batch=1, rows=100, lens=0, packed=False, shortest=1000, longest=1000, heads=32,
             kv_heads=8, dim=128, page=64, dtype="bf16"),
        # Cached prefixes of a pack of sequences, as the attention functions take them.
        dict(name="read_prefixes_16", kind="read", batch=16, rows=16384, lens=7, packed=True, shortest=16384, longest=32768,
             heads=32, kv_heads=8, dim=128, page=64, dtype="bf16"),
    ]


# heads / kv heads, drawn with equal odds
_HEADS = [(4, 4), (8, 2), (12, 12), (16, 4), (28, 4), (32, 8), (32, 32), (32, 1)]


def _spread(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {name: max(work(c)[name] for c in listed()) for name in ("bytes", "flops")}
    while True:
        case = _draw_any(rng)
        w = work(case)
        if all(w[name] <= most[name] for name in most) and _plain_bytes(case) <= (6e8 if case["kind"] == "verify" else 12e9):
            return case


def _draw_any(rng):
    kind = rng.choice(["tree", "attn", "attn", "attn", "verify", "verify", "accept", "read"])
    case = dict(kind=kind, batch=_spread(rng, 1, 128), lens=rng.randrange(1 << 20), packed=rng.random() < 0.4)
    if kind == "tree":
        case.update(nodes=_spread(rng, 1, 512), width=_spread(rng, 1, 64))
        return case
    if kind == "verify":
        case.update(nodes=_spread(rng, 1, 64), width=_spread(rng, 1, 16), vocab=_spread(rng, 100, 200000),
                    sampled=rng.random() < 0.6, dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]))
        return case
    heads, kv_heads = rng.choice(_HEADS)
    shortest = _spread(rng, 1, 16384)
    case.update(heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128, 128]), page=rng.choice([16, 32, 64, 64, 128, 256]),
                dtype=rng.choice(["bf16", "bf16", "fp16"]), shortest=shortest, longest=_spread(rng, shortest, 32768))
    if kind == "accept":
        case.update(nodes=_spread(rng, 1, 64))
        return case
    if kind == "read":
        case.update(rows=_spread(rng, 1, 16384))
        return case
    bounded = rng.random() < 0.5
    case.update(nodes=_spread(rng, 1, 200), width=_spread(rng, 1, 32), window=_spread(rng, 4, 8192) if bounded else -1,
                sinks=rng.choice([0, 1, 4]) if bounded else 0, lse=rng.random() < 0.4)
    return case


# ---- lengths ----------------------------------------------------------------------------------
def _lengths(case):
    """Cached tokens, rows (nodes, or tokens to read) and nodes that are there, per sequence.  Lengths are spread over
    their logarithm; in a pack the rows are, too, and in a batch the trees are padded."""
    rng = random.Random(case["lens"])
    held = [_spread(rng, case["shortest"], case["longest"]) if "shortest" in case else 0 for _ in range(case["batch"])]
    if case["kind"] == "read":
        most = [min(case["rows"], h) for h in held]
        if case["packed"]:
            rows = [_spread(rng, 1, m) for m in most]
        else:
            rows = [min(most)] * case["batch"]
        return held, rows, rows
    sizes = [_spread(rng, max(1, case["nodes"] // 4), case["nodes"]) for _ in range(case["batch"])]
    sizes[0] = case["nodes"]
    return held, sizes if case["packed"] else [case["nodes"]] * case["batch"], sizes


def _path_lengths(case, sizes):
    rng = random.Random(case["lens"] + 1)
    return [rng.randint(1, min(12, n)) for n in sizes]


def _words(case):
    return -(-case["nodes"] // 64)


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    held, rows, sizes = _lengths(case)
    n = sum(sizes)
    if case["kind"] == "tree":
        return {"bytes": sum(rows) * (4 + 8 + 8 * _words(case)), "flops": 0}
    if case["kind"] == "verify":  # the rows of the last node, which the next token is drawn from
        size = _DTYPES[case["dtype"]].itemsize * case["vocab"]
        return {"bytes": case["batch"] * size * (2 if case["sampled"] else 1), "flops": 3 * case["batch"] * case["vocab"]}
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "accept":
        taken = sum(_path_lengths(case, sizes))
        return {"bytes": 2 * taken * hk * d * 3, "flops": 2 * 2 * taken * hk * d}
    if case["kind"] == "read":
        return {"bytes": 2 * n * hk * d * 3, "flops": 2 * n * hk * d}
    keys = pairs = 0
    for h, m in zip(held, sizes):  # (at the depth of m at most; of the tree itself each row sees at least its own node)
        w, s = case["window"], case["sinks"]
        lo, least = (0, 0) if w < 0 else (max(0, h - w), min(h, max(0, h + m - w)))
        keys += h - lo + min(s, lo)
        pairs += m * (h - least + min(s, least) + 1)
    return {"bytes": keys * hk * 2 * d + n * (hq * (4 * d + 4 * case["lse"]) + hk * 4 * d), "flops": 4 * d * hq * pairs}


def _plain_bytes(case):
    """The largest tensors of the plain form and of the inputs."""
    held, rows, _ = _lengths(case)
    if case["kind"] == "tree":
        return case["batch"] * case["nodes"] ** 2
    if case["kind"] == "verify":
        return 4 * sum(rows) * case["vocab"]
    most = max(held) + max(rows)
    kv = case["batch"] * most * case["kv_heads"] * case["dim"] * 4
    return max(kv, case["batch"] * case["heads"] * max(rows) * most * 4) if case["kind"] == "attn" else kv


# ---- inputs -----------------------------------------------------------------------------------
def _exponents(amax):
    """The least e with ``amax <= 448 * 2**e`` (448: the largest e4m3 value), within [-120, 120]."""
    m, x = torch.frexp(amax)  # amax = m * 2**x, m in [0.5, 1); 448 = 0.875 * 2**9
    return torch.where(amax > 0, x - 9 + (m > 0.875), -120).clamp(-120, 120)


def _trees(case, seed):
    """Parents, depths and ancestor words of every row, as the host has them when it has drafted: each node's parent is
    one of the ``width`` nodes ahead of it (1: a chain), and of a tree's first nodes all are children of node 0."""
    _, rows, sizes = _lengths(case)
    rng = random.Random(seed)
    words = _words(case)
    parents, depths, bits = [], [], []
    for n, m in zip(rows, sizes):
        base = len(parents)
        for i in range(n):
            if i >= m:
                parents.append(-2)
                depths.append(-1)
                bits.append(0)
                continue
            p = rng.randrange(max(0, i - case["width"]), i) if i else -1
            parents.append(p)
            depths.append(depths[base + p] + 1 if i else 0)
            bits.append((bits[base + p] if i else 0) | 1 << i)
    low = (1 << 64) - 1
    signed = [[w - (1 << 64) if w >> 63 else w for w in (b >> 64 * j & low for j in range(words))] for b in bits]
    shape = (len(parents),) if case["packed"] else (case["batch"], case["nodes"])
    ints = [torch.tensor(x, dtype=torch.int32).view(shape).cuda() for x in (parents, depths)]
    return (*ints, torch.tensor(signed, dtype=torch.int64).view(*shape, words).cuda())


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    held, rows, sizes = _lengths(case)
    s = {"case": case}
    s["cu_seqlens"] = _ints([sum(rows[:i]) for i in range(len(rows) + 1)]) if case["packed"] else None
    if case["kind"] in ("tree", "attn", "verify"):
        s["parents"], s["depths"], s["ancestors"] = _trees(case, seed)
    if case["kind"] == "tree":
        del s["depths"], s["ancestors"]
    elif case["kind"] == "verify":
        _prepare_verify(s, gen)
    else:
        _prepare_cache(s, gen, held, rows, sizes)
    return s


def _prepare_cache(s, gen, held, rows, sizes):
    case, dev = s["case"], torch.device("cuda")
    b, hq, hk, d, p = case["batch"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    accept = case["kind"] == "accept"
    counts = [_pages(h + (12 if accept else 0), p) for h in held]
    total = sum(counts) + 1

    # the pool: values with an amplitude for every page and head, at the scale that fits them
    k = torch.empty(total, hk, p, d, dtype=_E4M3, device=dev)
    v = torch.empty(total, hk, p // 16, d, 16, dtype=_E4M3, device=dev)
    k_scale, v_scale = (torch.empty(total, hk, dtype=torch.uint8, device=dev) for _ in range(2))
    order = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    firsts = torch.tensor([sum(counts[:i]) for i in range(b)], device=dev)
    first_pages = order[firsts.clamp(max=total - 1)].long()
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
    n = torch.tensor(counts, device=dev)[:, None]
    place = torch.arange(max(1, max(counts)), device=dev)[None]
    s["page_table"] = torch.where(place < n, order[(firsts[:, None] + place).clamp(max=total - 1)], -1)
    s["cache"] = (k, v, k_scale.view(_E8M0), v_scale.view(_E8M0))
    s["held"] = _ints(held)

    lead = (sum(rows),) if case["packed"] else (b, rows[0])

    def some(heads):
        return torch.randn(*lead, heads, d, generator=gen, device=dev).to(_DTYPES[case["dtype"]])

    if case["kind"] == "read":
        # the end of each prefix; what is read goes to the rows that the caller has for it
        s["first"] = _ints([h - r for h, r in zip(held, rows)])
        s["k"], s["v"] = (torch.empty(*lead, hk, d, dtype=_DTYPES[case["dtype"]], device=dev) for _ in range(2))
        return
    s["k"], s["v"] = some(hk), some(hk)
    if case["kind"] == "attn":
        s["q"] = some(hq)
        return
    taken = _path_lengths(case, sizes)
    rng = random.Random(gen.initial_seed())
    path = [sorted([0] + rng.sample(range(1, m), t - 1)) + [-1] * (12 - t) for m, t in zip(sizes, taken)]
    s["path"] = _ints(path)


def _prepare_verify(s, gen):
    """Probabilities of two models that agree in part: softmax of logits with a common and an own share.  Drafted tokens
    are drawn from the draft's probabilities at their parent, or are its likeliest in the order of the siblings."""
    case, dev = s["case"], torch.device("cuda")
    parents, vocab = s["parents"], case["vocab"]
    lead, dtype = parents.shape, _DTYPES[case["dtype"]]
    target = torch.empty(*lead, vocab, dtype=dtype, device=dev)
    draft = torch.empty_like(target)
    flat_t, flat_d = target.view(-1, vocab), draft.view(-1, vocab)
    rows = flat_t.shape[0]
    flat = parents.reshape(-1).tolist()
    base = s["cu_seqlens"].tolist() if case["packed"] else list(range(0, rows + 1, case["nodes"]))
    children = [[] for _ in range(rows)]
    for lo, hi in zip(base, base[1:]):
        for j in range(lo, hi):
            if flat[j] >= 0:
                children[lo + flat[j]].append(j)
    most = max(1, max(map(len, children)))
    drafted = torch.tensor([c + [rows] * (most - len(c)) for c in children], device=dev)  # (rows: nobody's)
    tokens = torch.zeros(rows + 1, dtype=torch.int32, device=dev)
    step = max(1, (1 << 26) // vocab)
    for at in range(0, rows, step):
        n = min(step, rows - at)
        common = torch.randn(n, vocab, generator=gen, device=dev) * 3.0
        for to in (flat_t, flat_d):
            to[at:at + n] = torch.softmax(common + torch.randn(n, vocab, generator=gen, device=dev), -1).to(dtype)
        q = flat_d[at:at + n].float()
        if case["sampled"]:
            sums = q.cumsum(-1)
            u = torch.rand(n, most, generator=gen, device=dev) * sums[:, -1:]
            chosen = torch.searchsorted(sums, u, right=True).clamp(max=vocab - 1)
        else:
            chosen = q.topk(min(most, vocab), -1).indices
        mine = drafted[at:at + n, :chosen.shape[1]]
        tokens[mine] = chosen.to(torch.int32)
    s["tokens"] = tokens[:rows].view(lead).clone()
    s["target"] = target
    s["draft"] = draft if case["sampled"] else None
    s["uniforms"] = torch.rand(lead, generator=gen, device=dev)


# ---- the calls --------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    return {"tree": _tree, "attn": _attention, "verify": _verify, "accept": _accept, "read": _read}[s["case"]["kind"]](s)


def _own(s):
    path = os.path.join(os.getcwd(), "ring-sliding-window-attention_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import ring_swa

    c, cu = s["case"], s["cu_seqlens"]
    most = c["nodes"] if c["packed"] and c["kind"] == "tree" else None
    if c["kind"] == "tree":
        tree = ring_swa.draft_tree(s["parents"], cu, max_nodes=most)
        return tree.depths, tree.ancestors
    if c["kind"] == "verify":
        tree = ring_swa.DraftTree(s["parents"], s["depths"], s["ancestors"])
        return ring_swa.verify_drafts(tree, s["tokens"], s["target"], s["draft"], s["uniforms"], cu)
    cache = ring_swa.KVCache(*s["cache"])
    if c["kind"] == "accept":
        ring_swa.kv_cache_accept(cache, s["k"], s["v"], s["path"], s["page_table"], s["held"], cu)
        return tuple(cache)
    if c["kind"] == "read":
        ring_swa.kv_cache_read(cache, s["k"], s["v"], s["page_table"], s["first"], cu)
        return s["k"], s["v"]
    tree = ring_swa.DraftTree(s["parents"], s["depths"], s["ancestors"])
    return ring_swa.kv_cache_tree_attn(s["q"], s["k"], s["v"], tree, cache, s["page_table"], s["held"], c["window"], cu,
                                       num_sink_tokens=c["sinks"], return_lse=c["lse"])


# ---- plain forms ------------------------------------------------------------------------------
def _padded(s, x):
    """Packed rows as ``[b, most, ...]``, rows behind a sequence's last one repeated from somewhere, and which are real."""
    cu = s["cu_seqlens"]
    if cu is None:
        return x, torch.ones(x.shape[:2], dtype=torch.bool, device=x.device)
    cu = cu.long()
    at = cu[:-1, None] + torch.arange(s["case"]["nodes"], device=x.device)
    return x[at.clamp(max=x.shape[0] - 1)], at < cu[1:, None]


def _unpadded(s, x):
    """``[b, most, ...]`` as the call's rows."""
    cu = s["cu_seqlens"]
    if cu is None:
        return x
    at = torch.arange(s["parents"].shape[0], device=x.device)
    seq = torch.searchsorted(cu, at.to(torch.int32), right=True) - 1
    return x[seq, at - cu[seq]]


def _tree(s):
    parents, real = _padded(s, s["parents"])
    b, n = parents.shape
    dev = parents.device
    words = _words(s["case"])
    seen = torch.zeros(b, n, n, dtype=torch.bool, device=dev)
    there = torch.zeros(b, n, dtype=torch.bool, device=dev)
    at = torch.arange(b, device=dev)
    for i in range(n):
        p = parents[:, i].long()
        above = (p >= 0) & (p < i)
        p = p.clamp(0, n - 1)
        there[:, i] = real[:, i] & ((parents[:, i] == -1) | (above & there[at, p]))
        seen[:, i] = seen[at, p] & (above & there[:, i])[:, None]
        seen[:, i, i] = there[:, i]
    depths = torch.where(there, seen.sum(-1) - 1, -1).to(torch.int32)
    bits = torch.nn.functional.pad(seen, (0, 64 * words - n)).view(b, n, words, 64).long()
    return _unpadded(s, depths), _unpadded(s, (bits << torch.arange(64, device=dev)).sum(-1))


def _codes(pool, *at):
    return pool.view(torch.uint8)[at].view(_E4M3).float()


def _power(scale):
    return torch.exp2(scale.view(torch.uint8).float() - 127)


def _cached(s, which):
    """All keys or values that the table names, ``[b, kv_heads, places, dim]`` in 32 bits."""
    pool, scale = s["cache"][which], s["cache"][2 + which]
    pages = s["page_table"].clamp(min=0).long()
    x = _codes(pool, pages)
    x *= _power(scale)[pages].reshape(*pages.shape, -1, *[1] * (x.dim() - 3))
    return x.transpose(1, 2).flatten(2, 3) if which == 0 else x.permute(0, 2, 1, 3, 5, 4).flatten(2, 4)


def _attention(s):
    c = s["case"]
    (q, real), (k, _), (v, _) = (_padded(s, s[x]) for x in "qkv")
    depths, ancestors = _padded(s, s["depths"])[0], _padded(s, s["ancestors"])[0]
    depths = torch.where(real, depths, -1)
    b, n, hq, d = q.shape
    hk, dev = k.shape[2], q.device
    g = hq // hk
    # heads that share keys are rows of one product
    rows = q.float().transpose(1, 2).reshape(b, hk, g * n, d)
    places = s["page_table"].shape[1] * c["page"]
    scores = torch.empty(b, hk, g * n, places + n, device=dev)
    scores[..., :places] = torch.matmul(rows, _cached(s, 0).transpose(2, 3).contiguous())
    scores[..., places:] = torch.matmul(rows, k.float().permute(0, 2, 3, 1).contiguous())
    scores = scores.mul_(d ** -0.5).view(b, hk, g, n, -1)
    held = s["held"][:, None, None]
    j = torch.arange(places, device=dev)
    at = held + depths[..., None]  # [b, n, 1]
    old = (j < held) & (depths[..., None] >= 0)
    bit = torch.arange(n, device=dev)
    new = (ancestors[..., bit // 64] >> (bit % 64) & 1).bool()
    if c["window"] >= 0:
        old &= (j >= at - c["window"]) | (j < c["sinks"])
        place = held + depths[:, None]  # [b, 1, n]
        new &= (place >= at - c["window"]) | (place < c["sinks"])
    seen = torch.cat((old, new & (depths[..., None] >= 0)), -1)[:, None, None]
    scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top.isfinite(), top, 0)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log())[..., 0].flatten(1, 2)  # [b, heads, n]
    p = p.flatten(2, 3)
    out = torch.matmul(p[..., :places], _cached(s, 1)) + torch.matmul(p[..., places:], v.float().transpose(1, 2).contiguous())
    out = torch.where(total > 0, out.view(b, hk, g, n, d) / total, 0).flatten(1, 2).transpose(1, 2)
    out = _unpadded(s, out).to(s["q"].dtype).contiguous()
    if not c["lse"]:
        return out
    lse = _unpadded(s, lse.transpose(1, 2))
    return out, lse.transpose(-1, -2).contiguous()


def _verify(s):
    """All sequences at once, a node after the other, in 64 bits (decisions lie next to borders)."""
    (parents, real), (tokens, _), (uniforms, _) = (_padded(s, s[x]) for x in ("parents", "tokens", "uniforms"))
    b, n = parents.shape
    dev, vocab = parents.device, s["case"]["vocab"]
    at = torch.arange(b, device=dev)
    rows = s["cu_seqlens"][:-1].long() if s["cu_seqlens"] is not None else at * n
    flat_t = s["target"].view(-1, vocab)
    flat_d = s["draft"].view(-1, vocab) if s["draft"] is not None else None
    cur = torch.zeros(b, dtype=torch.long, device=dev)
    path = torch.full((b, n if s["cu_seqlens"] is None else 64 * _words(s["case"])), -1, dtype=torch.int32, device=dev)
    path[:, 0] = 0
    accepted = torch.ones(b, dtype=torch.int32, device=dev)
    a, mass = torch.zeros(b, dtype=torch.float64, device=dev), torch.ones(b, dtype=torch.float64, device=dev)
    p = flat_t[rows].double()
    q = flat_d[rows].double() if flat_d is not None else None
    for i in range(1, n):
        child = real[:, i] & (parents[:, i] == cur)
        x = tokens[:, i].long()
        if q is not None:
            rest = (p[at, x] - a * q[at, x]).clamp(min=0)
            taken = child & (uniforms[:, i].double() * mass * q[at, x] < rest)
        else:
            rest = p[at, x]
            taken = child & (uniforms[:, i].double() * mass < rest)
        left = child & ~taken
        if q is not None:
            a = torch.where(left, a + mass, a)
            mass = torch.where(left, (p - a[:, None] * q).clamp_(min=0).sum(-1), mass)
        else:
            mass = torch.where(left, (mass - rest).clamp(min=0), mass)
            p[at, x] = torch.where(left, 0, rest)
        cur = torch.where(taken, i, cur)
        a, mass = torch.where(taken, 0, a), torch.where(taken, 1, mass)
        path[at, accepted.long().clamp(max=path.shape[1] - 1)] = torch.where(
            taken, i, path[at, accepted.long().clamp(max=path.shape[1] - 1)])
        accepted += taken.to(torch.int32)
        p = torch.where(taken[:, None], flat_t[rows + cur].double(), p)
        if q is not None:
            q = torch.where(taken[:, None], flat_d[rows + cur].double(), q)
    rest = (p - a[:, None] * q).clamp_(min=0) if q is not None else p
    empty = rest.sum(-1, keepdim=True) <= 0
    sums = torch.where(empty, flat_t[rows + cur].double(), rest).cumsum(-1)
    drawn = torch.searchsorted(sums, uniforms[:, :1].double() * sums[:, -1:], right=True)[:, 0].clamp(max=vocab - 1)
    return path, accepted, drawn.to(s["tokens"].dtype)


def _accept(s):
    c, p = s["case"], s["case"]["page"]
    cu = s["cu_seqlens"]
    b = c["batch"]
    dev = s["held"].device
    path = s["path"].long()
    seq = torch.arange(b, device=dev)[:, None].expand_as(path)
    i = torch.arange(path.shape[1], device=dev)[None].expand_as(path)
    mine = path >= 0
    seq, i, node = seq[mine], i[mine], path[mine]
    new_k = s["k"][seq, node] if cu is None else s["k"][cu[seq] + node]
    new_v = s["v"][seq, node] if cu is None else s["v"][cu[seq] + node]
    k, v, k_scale, v_scale = s["cache"]
    at = s["held"][seq] + i
    page, slot = s["page_table"][seq, at // p].long(), at % p
    # a sequence's first page may hold older rows, the next one starts with this call
    first = s["page_table"].gather(1, (s["held"].long() // p)[:, None])[:, 0].long()
    older = s["held"] % p
    for_old = torch.arange(p, device=dev)[None] < older[:, None]  # [b, p]
    started = torch.zeros(k.shape[0], 1, dtype=torch.bool, device=dev)
    started[first] = (older > 0)[:, None]
    _accept_one(k, k_scale, new_k, page, first, started, (page, slot), for_old[:, None, :, None])
    _accept_one(v, v_scale, new_v, page, first, started, (page, slot // 16, slot % 16),
                for_old.unflatten(1, (p // 16, 16))[:, None, :, None, :])
    return k, v, k_scale, v_scale


def _accept_one(pool, scale, rows, page, first, started, place, for_old):
    x = rows.float()
    amax = x.abs().amax(-1)  # [rows, heads]
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


def _read(s):
    p, n = s["case"]["page"], s["k"].shape[-3]
    at = torch.arange(n, device=s["k"].device)
    if s["cu_seqlens"] is None:
        seq = torch.arange(s["case"]["batch"], device=at.device)[:, None]
        token = s["first"][:, None] + at
    else:
        seq = torch.searchsorted(s["cu_seqlens"], at.to(torch.int32), right=True) - 1
        token = s["first"][seq] + at - s["cu_seqlens"][seq]
    page, place = s["page_table"][seq, token // p].long(), token % p
    k, v, k_scale, v_scale = s["cache"]
    x = k.view(torch.uint8)[page, :, place].view(_E4M3).float() * _power(k_scale)[page][..., None]
    s["k"].copy_(x)
    x = v.view(torch.uint8)[page, :, place // 16, :, place % 16].view(_E4M3).float() * _power(v_scale)[page][..., None]
    s["v"].copy_(x)
    return s["k"], s["v"]


# ---- in 64 bits -------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("tree", "verify"):  # (whole numbers, of decisions)
        return None
    return {"attn": _exact_attention, "accept": _exact_accept, "read": _exact_read}[kind](s)


def _exact_row(s, which, b, h, j):
    """Values of places ``j`` of a sequence's head, ``[places, dim]``."""
    p = s["case"]["page"]
    pool, scale = s["cache"][which], s["cache"][2 + which]
    page = s["page_table"][b].long()[j // p]
    if which == 0:
        codes = pool.view(torch.uint8)[page, h, j % p]
    else:
        codes = pool.view(torch.uint8)[page, h, (j % p) // 16, :, j % 16]
    return codes.view(_E4M3).double() * torch.pow(2.0, scale.view(torch.uint8)[page, h].double() - 127)[:, None]


def _exact_attention(s):
    """One sequence and kv head at a time, over its cached tokens and its nodes; who sees whom from the parents."""
    case = s["case"]
    held, rows, _ = _lengths(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["batch"] * hk > 4096:
        return None
    q, dev = s["q"], s["q"].device
    g = hq // hk
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    lse = torch.full(q.shape[:-1], -math.inf, dtype=torch.float64, device=dev)
    row = 0
    for b in range(case["batch"]):
        n, length = rows[b], held[b]
        at = slice(row, row + n) if case["packed"] else b
        parents = s["parents"][at].tolist()
        lines, depth = [], []
        for i, p in enumerate(parents):
            lines.append([] if p < -1 else [i] if p == -1 else lines[p] + [i])
            depth.append(len(lines[i]) - 1)
        place = torch.tensor([length + t for t in depth], device=dev)
        there = torch.tensor([t >= 0 for t in depth], device=dev)
        related = torch.zeros(n, n, dtype=torch.bool)
        for i, line in enumerate(lines):
            related[i, line] = True
        j = torch.arange(length, device=dev)
        hidden = torch.zeros(n, length + n, dtype=torch.bool, device=dev)
        hidden[:, length:] = ~related.to(dev)
        if case["window"] >= 0:
            key_at = torch.cat((j, place))
            hidden |= (key_at[None] < place[:, None] - case["window"]) & (key_at[None] >= case["sinks"])
        hidden |= ~there[:, None]
        for h in range(hk):
            heads = slice(h * g, (h + 1) * g)
            keys = torch.cat((_exact_row(s, 0, b, h, j), s["k"][at][:, h].double()))
            values = torch.cat((_exact_row(s, 1, b, h, j), s["v"][at][:, h].double()))
            z = q[at][:, heads].double().transpose(0, 1) @ keys.T / math.sqrt(d)  # [group, n, keys]
            z = z.masked_fill(hidden, -math.inf)
            norm = torch.logsumexp(z, -1)
            w = torch.exp(z - torch.where(norm.isfinite(), norm, 0)[..., None])
            out[at][:, heads] = (w @ values).transpose(0, 1)
            lse[at][:, heads] = norm.T
        row += n
    lse = lse.transpose(-1, -2).contiguous()
    return (out, lse) if case["lse"] else out


def _exact_scale(amax):
    e = -120
    while e < 120 and amax > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def _exact_accept(s):
    """Scales exactly; codes as the quotients that they round."""
    case, p = s["case"], s["case"]["page"]
    held, rows, _ = _lengths(case)
    if case["batch"] * case["kv_heads"] > 2100:
        return None
    outs = [t.double() for t in s["cache"][:2]]
    scales = [torch.pow(2.0, t.view(torch.uint8).double() - 127) for t in s["cache"][2:]]
    table, paths = s["page_table"].tolist(), s["path"].tolist()
    row = 0
    for b in range(case["batch"]):
        nodes = [i for i in paths[b] if i >= 0]
        for which, source in ((0, s["k"]), (1, s["v"])):
            x = (source[row:row + rows[b]] if case["packed"] else source[b])[nodes].double()
            done = 0
            while done < len(nodes):
                at = held[b] + done
                page, lo = table[b][at // p], at % p
                n = min(p - lo, len(nodes) - done)
                part = x[done:done + n].transpose(0, 1)  # [heads, n, dim]
                for h, most in enumerate(part.abs().amax((1, 2)).tolist()):
                    was = float(scales[which][page, h])
                    now = max(_exact_scale(most), was) if lo else _exact_scale(most)
                    if which == 0:
                        outs[0][page, h, :lo] *= was / now
                        outs[0][page, h, lo:lo + n] = part[h] / now
                    else:
                        view = outs[1][page, h].transpose(1, 2).reshape(p, -1).clone()
                        view[:lo] *= was / now
                        view[lo:lo + n] = part[h] / now
                        outs[1][page, h] = view.view(p // 16, 16, -1).transpose(1, 2)
                    scales[which][page, h] = now
                done += n
        row += rows[b]
    return (*outs, *scales)


def _exact_read(s):
    case = s["case"]
    held, rows, _ = _lengths(case)
    outs = [torch.zeros(s["k"].shape, dtype=torch.float64, device=s["k"].device) for _ in range(2)]
    row = 0
    for b in range(case["batch"]):
        n = rows[b]
        j = torch.arange(held[b] - n, held[b], device=outs[0].device)
        for h in range(case["kv_heads"]):
            for which in range(2):
                mine = outs[which][row:row + n] if case["packed"] else outs[which][b]
                mine[:, h] = _exact_row(s, which, b, h, j)
        row += n
    return tuple(outs)
