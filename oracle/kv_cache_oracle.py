"""64-bit restatement of the 8-bit paged cache's calls, one sequence and kv head at a time, on whatever
device the tensors live.  Test infrastructure only.

A cache is the tuple ``(k, v, k_scale, v_scale)`` as the calls take it; codes and scales are compared as
bytes, so the functions that write work on clones and return them."""
import math

import torch

LARGEST = 448.0  # of e4m3


def scale_byte(amax: float) -> int:
    """The byte of the least 2^e with amax <= 448 * 2^e, -120 <= e <= 120."""
    e = -120
    while e < 120 and amax > LARGEST * 2.0 ** e:
        e += 1
    return e + 127


def encode(x: torch.Tensor) -> torch.Tensor:
    """e4m3 codes (uint8) of values within +-448; non-finite ones are NaN.  (64-bit values that are no
    32-bit ones do not occur: a quotient by a power of two is exact.)"""
    x = torch.where(x.isfinite(), x, math.nan).float()
    c = x.to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.where(x.isnan(), torch.full_like(c, 0x7F), c)


def decode(codes: torch.Tensor) -> torch.Tensor:
    return codes.view(torch.float8_e4m3fn).double()


def bytes_of(cache):
    return tuple(t.view(torch.uint8) for t in cache)


def same_bytes(got, want) -> bool:
    """Codes and scales equal, any NaN code as any other."""
    for i, (g, w) in enumerate(zip(bytes_of(got), bytes_of(want))):
        same = g == w
        if i < 2:
            same |= ((g & 0x7F) == 0x7F) & ((w & 0x7F) == 0x7F)
        if not bool(same.all()):
            return False
    return True


def _page_rows(codes, which, page, h):
    """A (page, head)'s codes as ``[place, dim]``, a copy."""
    t = codes[which][page, h]
    return t.clone() if which == 0 else t.transpose(1, 2).reshape(-1, t.shape[1]).clone()


def _put_page_rows(codes, which, page, h, rows):
    if which == 0:
        codes[0][page, h] = rows
    else:
        codes[1][page, h] = rows.view(-1, 16, rows.shape[1]).transpose(1, 2)


def append(cache, k, v, page_table, seqlens, cu_seqlens=None):
    out = tuple(t.clone() for t in cache)
    codes = bytes_of(out)
    pages, heads, size, _ = cache[0].shape
    table = page_table.tolist()
    for b, start in enumerate(seqlens.tolist()):
        start = max(0, start)
        if cu_seqlens is None:
            rows = (k[b], v[b])
        else:
            lo, hi = cu_seqlens[b].item(), cu_seqlens[b + 1].item()
            rows = (k[lo:hi], v[lo:hi])
        done, n = 0, rows[0].shape[0]
        while done < n:
            at = start + done
            place = at % size
            count = min(size - place, n - done)
            page = table[b][at // size] if at // size < len(table[b]) else -1
            if 0 <= page < pages:
                for which in (0, 1):
                    for h in range(heads):
                        x = rows[which][done:done + count, h].double()
                        fine = x[x.isfinite()].abs()
                        byte = scale_byte(fine.max().item() if fine.numel() else 0.0)
                        mine = _page_rows(codes, which, page, h)
                        if place:
                            was = int(codes[2 + which][page, h])
                            byte = max(byte, was)
                            if byte != was:
                                mine[:place] = encode(decode(mine[:place]) * 2.0 ** (was - byte))
                        mine[place:place + count] = encode(x * 2.0 ** (127 - byte))
                        _put_page_rows(codes, which, page, h, mine)
                        codes[2 + which][page, h] = byte
            done += count
    return out


def gather(cache, which, page_table, b, h, tokens):
    """Values of a sequence's tokens ``[n, dim]`` in 64 bits, and which of them are there."""
    codes = bytes_of(cache)
    pages, _, size, dim = cache[0].shape
    page = page_table[b].long()[tokens // size]
    there = (page >= 0) & (page < pages)
    page = page.clamp(0, pages - 1)
    place = tokens % size
    c = codes[0][page, h, place] if which == 0 else codes[1][page, h, place // 16, :, place % 16]
    x = decode(c) * torch.pow(2.0, codes[2 + which][page, h].double() - 127)[:, None]
    return torch.where(there[:, None], x, 0.0), there


def _rows(q, b, cu_seqlens):
    """First row of sequence b, its number of rows, and a view ``[n, heads, dim]``."""
    if cu_seqlens is None:
        return q[b]
    return q[cu_seqlens[b].item():cu_seqlens[b + 1].item()]


def _scores(q, cache, page_table, b, h, length, window, sinks, scale):
    """Scores of a sequence's rows ``[n, group, dim]`` against all its tokens, -inf where not seen; and the
    largest sum over dimensions of scale * |q| |k| among the seen ones (what a dot product's error goes by)."""
    n = q.shape[0]
    dev = q.device
    j = torch.arange(length, device=dev)
    keys, there = gather(cache, 0, page_table, b, h, j)
    pos = length - n + torch.arange(n, device=dev)
    seen = (j[None] <= pos[:, None]) & there[None]
    if window >= 0:
        seen &= (j[None] >= pos[:, None] - window) | (j[None] < sinks)
    z = torch.einsum("ngd,jd->ngj", q.double(), torch.where(seen.any(0)[:, None], keys, 0.0)) * scale
    reach = torch.einsum("ngd,jd->ngj", q.double().abs(), torch.where(seen.any(0)[:, None], keys.abs(), 0.0)) * scale
    z = z.masked_fill(~seen[:, None], -math.inf)
    reach = reach.masked_fill(~seen[:, None], 0.0)
    return z, seen, reach.amax(-1) if length else z.new_zeros(z.shape[:2])


def attn(q, cache, page_table, seqlens, window=-1, cu_seqlens=None, scale=None, sinks=0):
    """out and lse in 64 bits, ``spread`` (sum of the softmax weights times |v|), ``reach``, and ``total`` (sum of |v|
    over all keys that some row of the sequence sees)."""
    heads, hk = q.shape[-2], cache[0].shape[1]
    g = heads // hk
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    spread, total = torch.zeros_like(out), torch.zeros_like(out)
    shape = (*q.shape[:-2], heads)
    lse = torch.full(shape, -math.inf, dtype=torch.float64, device=q.device)
    reach = torch.zeros(shape, dtype=torch.float64, device=q.device)
    for b, length in enumerate(seqlens.tolist()):
        x, o, sp, to = (_rows(t, b, cu_seqlens) for t in (q, out, spread, total))
        ls, re = (_rows(t, b, cu_seqlens) for t in (lse, reach))
        if x.shape[0] == 0 or length <= 0:
            continue
        for h in range(hk):
            mine = slice(h * g, (h + 1) * g)
            z, seen, r = _scores(x[:, mine], cache, page_table, b, h, length, window, sinks, scale)
            values, _ = gather(cache, 1, page_table, b, h, torch.arange(length, device=q.device))
            values = torch.where(seen.any(0)[:, None], values, 0.0)
            norm = torch.logsumexp(z, -1)
            p = torch.where(seen[:, None], torch.exp(z - torch.where(norm.isfinite(), norm, 0.0)[..., None]), 0.0)
            o[:, mine] = p @ values
            sp[:, mine], to[:, mine] = p @ values.abs(), values.abs().sum(0)
            ls[:, mine], re[:, mine] = norm, r
    # (the calls' lse is [batch, heads, seq], of a pack [heads, tokens])
    return out, lse.transpose(-1, -2), spread, reach.transpose(-1, -2), total


def weights(q, cache, page_table, seqlens, lse, running, window=-1, cu_seqlens=None, scale=None, sinks=0):
    """The running sums after the call, in 64 bits, and how far 32-bit scores may put them off: sum of the
    added weights times ``reach``."""
    heads, hk = q.shape[-2], cache[0].shape[1]
    g = heads // hk
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out = running.double().clone()
    off = torch.zeros_like(out)
    rows_lse = lse.transpose(-1, -2).double()
    for b, length in enumerate(seqlens.tolist()):
        x, ls = _rows(q, b, cu_seqlens), _rows(rows_lse, b, cu_seqlens)
        if x.shape[0] == 0 or length <= 0:
            continue
        for h in range(hk):
            mine = slice(h * g, (h + 1) * g)
            z, seen, r = _scores(x[:, mine], cache, page_table, b, h, length, window, sinks, scale)
            p = torch.exp(z - ls[:, mine, None])
            p = torch.where(seen[:, None] & (ls[:, mine, None] != -math.inf), p, 0.0)
            n = min(length, out.shape[-1])
            out[b, h, :n] += p.sum((0, 1))[:n]
            off[b, h, :n] += (p * r[..., None]).sum((0, 1))[:n]
    return out, off


def evict(cache, running, page_table, seqlens, new_page_table, budget, sinks=0, recent=0):
    out = tuple(t.clone() for t in cache)
    codes = bytes_of(out)
    pages, heads, size, dim = cache[0].shape
    batch, width = page_table.shape[0], running.shape[-1]
    kept = torch.full((batch, heads, budget), -1, dtype=torch.int32)
    new_weights = torch.zeros(running.shape, dtype=torch.float32)
    target = new_page_table.tolist()
    count = torch.zeros(batch, dtype=torch.int32)
    for b, (n, row) in enumerate(zip(seqlens.tolist(), page_table.tolist())):
        n = max(0, min(n, len(row) * size))
        there = [j for j in range(n) if 0 <= row[j // size] < pages]  # (tokens without a page are not kept)
        count[b] = min(len(there), budget)
        for h in range(heads):
            w = running[b, h].tolist() + [0.0] * max(0, n - width)
            if len(there) <= budget:
                keep = there
            else:
                must = [j for j in there if j < sinks or j >= n - recent]
                rest = sorted((j for j in there if sinks <= j < n - recent),
                              key=lambda j: (math.isnan(w[j]), -w[j] if not math.isnan(w[j]) else 0.0, j))
                keep = sorted(must + rest[:budget - len(must)])
            tokens = torch.tensor(keep, dtype=torch.long, device=page_table.device)
            kept[b, h, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
            for r, j in enumerate(keep):
                if r < width:
                    new_weights[b, h, r] = w[j]
            for which in (0, 1):
                x, _ = gather(cache, which, page_table, b, h, tokens)
                for i in range(0, len(keep), size):
                    part = x[i:i + size]
                    page = target[b][i // size]
                    if not 0 <= page < pages:
                        continue
                    fine = part[part.isfinite()].abs()
                    byte = scale_byte(fine.max().item() if fine.numel() else 0.0)
                    mine = _page_rows(codes, which, page, h)
                    mine[:part.shape[0]] = encode(part * 2.0 ** (127 - byte))
                    _put_page_rows(codes, which, page, h, mine)
                    codes[2 + which][page, h] = byte
    return out, count, new_weights, kept
