"""64-bit restatement of the calls on drafted tokens, one sequence at a time, on whatever device the tensors live.  Test
infrastructure only.  The cache and its helpers are kv_cache_oracle's."""
import math

import torch

from oracle import kv_cache_oracle as O


def lines(parents, max_nodes=1024):
    """For each node of one sequence (a list) the list of its ancestors, root first, and itself; None: not there."""
    found = []
    for i, p in enumerate(parents):
        if i >= max_nodes or not (-1 <= p < i) or (p >= 0 and found[p] is None):
            found.append(None)
        else:
            found.append([i] if p == -1 else found[p] + [i])
    return found


def tree(parents, max_nodes):
    """Parents, depths and ancestor words (as int64) of one sequence, as lists."""
    words = (max_nodes + 63) // 64
    out = ([], [], [])
    for i, line in enumerate(lines(parents, max_nodes)):
        there = line is not None
        out[0].append(parents[i] if there else -2)
        out[1].append(len(line) - 1 if there else -1)
        row = [0] * words
        for j in line or ():
            row[j // 64] |= 1 << (j % 64)
        out[2].append([w - (1 << 64) if w >> 63 else w for w in row])
    return out


def slices(cu_seqlens, batch):
    """What sequence b's rows are in a tensor of rows: an index."""
    if cu_seqlens is None:
        return list(range(batch))
    cu = cu_seqlens.tolist()
    return [slice(lo, hi) for lo, hi in zip(cu, cu[1:])]


def seen(parents, length, window, sinks, cached_there):
    """Who sees whom: bool [nodes, length + nodes]."""
    n = len(parents)
    see = torch.zeros(n, length + n, dtype=torch.bool)
    found = lines(parents)
    for i, line in enumerate(found):
        if line is None:
            continue
        at = length + len(line) - 1
        j = torch.arange(length)
        see[i, :length] = cached_there & ((j >= at - window) | (j < sinks) | (window < 0))
        for j in line:
            place = length + len(found[j]) - 1
            see[i, length + j] = window < 0 or place >= at - window or place < sinks
    return see


def tree_attn(q, k, v, parents, cache, page_table, seqlens, window=-1, cu_seqlens=None, scale=None, sinks=0):
    """out, lse, ``spread``, ``reach`` and ``total`` as kv_cache_oracle.attn; ``parents``: a list of lists."""
    hq, hk, dim = q.shape[-2], k.shape[-2], q.shape[-1]
    g = hq // hk
    scale = dim ** -0.5 if scale is None else scale
    size = cache[0].shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    spread, total = torch.zeros_like(out), torch.zeros_like(out)
    lse = torch.full(q.shape[:-1], -math.inf, dtype=torch.float64, device=q.device)
    reach = torch.zeros(q.shape[:-1], dtype=torch.float64, device=q.device)
    for b, at in enumerate(slices(cu_seqlens, page_table.shape[0])):
        length = max(0, min(int(seqlens[b]), page_table.shape[1] * size))
        n = q[at].shape[0]
        if n == 0:
            continue
        j = torch.arange(length, device=q.device)
        there = O.gather(cache, 0, page_table, b, 0, j)[1].cpu() if length else torch.zeros(0, dtype=torch.bool)
        see = seen(parents[b], length, window, sinks, there).to(q.device)
        any_row = see.any(0)[:, None]
        for h in range(hk):
            mine = slice(h * g, (h + 1) * g)
            old = [O.gather(cache, w, page_table, b, h, j)[0] if length else q.new_zeros(0, dim).double() for w in (0, 1)]
            keys = torch.where(any_row, torch.cat((old[0], k[at][:, h].double())), 0.0)
            values = torch.where(any_row, torch.cat((old[1], v[at][:, h].double())), 0.0)
            x = torch.where(see.any(1)[:, None, None], q[at][:, mine].double(), 0.0)
            z = torch.einsum("ngd,jd->ngj", x, keys) * scale
            r = torch.einsum("ngd,jd->ngj", x.abs(), keys.abs()) * scale
            z = z.masked_fill(~see[:, None], -math.inf)
            norm = torch.logsumexp(z, -1)
            p = torch.exp(z - torch.where(norm.isfinite(), norm, 0.0)[..., None])
            out[at][:, mine] = p @ values
            spread[at][:, mine], total[at][:, mine] = p @ values.abs(), values.abs().sum(0)
            lse[at][:, mine], reach[at][:, mine] = norm, r.masked_fill(~see[:, None], 0.0).amax(-1)
    return out, lse.transpose(-1, -2), spread, reach.transpose(-1, -2), total


def _positive(t):
    t = t.double()
    return torch.where(t > 0, t, 0.0)


def verify(parents, tokens, target, draft, uniforms):
    """Nodes taken and the next token of one sequence: lists of parents and tokens, probabilities [nodes, vocab], draft
    or None, and a list of numbers."""
    if not parents or parents[0] != -1:
        return [], -1
    vocab = target.shape[1]
    path, cur, left = [0], 0, _positive(target[0])
    a, mass = 0.0, 1.0  # left = max(0, p - a q), to be divided by mass
    for i in range(1, len(parents)):
        x = tokens[i]
        if parents[i] != cur or not 0 <= x < vocab:
            continue
        q = float(_positive(draft[cur, x])) if draft is not None else 1.0
        if uniforms[i] * mass * q < float(left[x]):
            path.append(i)
            cur, a, mass = i, 0.0, 1.0
            left = _positive(target[cur])
        elif draft is not None:
            a += mass
            left = torch.clamp(_positive(target[cur]) - a * _positive(draft[cur]), min=0.0)
            mass = math.fsum(left.tolist())
        else:
            mass = max(0.0, mass - float(left[x]))
            left[x] = 0.0
    if not bool((left > 0).any()):
        left = _positive(target[cur])
    if not bool((left > 0).any()):
        return path, -1
    sums = left.cumsum(0)
    past = (sums > uniforms[0] * sums[-1]).nonzero()
    return path, int(past[0]) if past.numel() else int((left > 0).nonzero()[-1])


def accept(cache, k, v, path, page_table, seqlens, cu_seqlens=None):
    """The cache after the call."""
    for b, at in enumerate(slices(cu_seqlens, page_table.shape[0])):
        rows = []
        for i in path[b].tolist():
            if not 0 <= i < k[at].shape[0]:
                break
            rows.append(i)
        if rows:
            cache = O.append(cache, k[at][rows][None], v[at][rows][None], page_table[b:b + 1], seqlens[b:b + 1])
    return cache


def read(cache, page_table, first, rows):
    """Values of tokens first[b], .. of each sequence, rows[b] of them, in 64 bits: lists of [rows, heads, dim], keys and
    values."""
    pages, heads, size, dim = cache[0].shape
    got = []
    for b, n in enumerate(rows):
        start = max(0, int(first[b]))
        j = start + torch.arange(n, device=page_table.device)
        inside = j < page_table.shape[1] * size
        of = []
        for which in (0, 1):
            x = torch.zeros(n, heads, dim, dtype=torch.float64, device=page_table.device)
            for h in range(heads):
                if bool(inside.any()):
                    values, there = O.gather(cache, which, page_table, b, h, j[inside])
                    x[inside, h] = torch.where(there[:, None], values, 0.0)
            of.append(x)
        got.append(of)
    return got
