"""The 8-bit paged cache's calls against a 64-bit restatement: append and evict byte for byte, attention and
key weights within bounds that count roundings (below).

``HALF[t]`` is half a step of the type relative to the value.  An output of attention is off by at most
  HALF * |out|            its own rounding
  HALF * spread           the softmax weights' rounding to the type of the product with V (spread = sum p |v|)
  2 * score * spread      32-bit scores: a relative error of `score` in every weight and in their sum
  2^-39 * total           fp16 only: weights below 2^-28 of the largest are multiples of 2^-38 of it (total = sum |v|;
                          the type's normal range ends at 2^-14, and weights are taken 2^14 times as large)
  2^-17 * spread          exp2, running sums and their rescaling, a few units of 2^-24 for each of up to 64 tiles
with score = dim * 2^-24 * reach (a dot product of dim terms summed in 32 bits; reach = scale * sum |q| |k|) plus
2^-21 * reach (the argument of exp2).  lse: score + 2^-20 * (1 + |lse|).  A key's weight: twice score, and 2^-17."""
import math
import random

import pytest
import torch

from oracle import kv_cache_oracle as O

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
NAN_CODE = 0x7F


def make(lens, heads_kv, dim, size, seed, spare=3, max_pages=None, wild=True):
    """A pool with random codes and scales everywhere (what no sequence holds is NaN), pages in no order."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // size) for n in lens]
    total = sum(need) + spare
    codes = torch.randint(0, 256, (2, total, heads_kv, size, dim), generator=g, dtype=torch.uint8)
    codes[(codes & 0x7F) >= 0x78] &= 0x87  # (magnitudes below 1: sums of the size of projected activations)
    scales = torch.randint(122, 130, (2, total, heads_kv), generator=g, dtype=torch.uint8)
    order = torch.randperm(total, generator=g).tolist()
    width = max(max(need, default=0), max_pages or 0)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order[at]
            held = min(size, lens[b] - i * size)
            if wild:
                codes[:, order[at], :, held:] = NAN_CODE
            at += 1
    if wild:
        for page in order[at:]:
            codes[:, page] = NAN_CODE
    k = codes[0].contiguous()
    v = codes[1].view(total, heads_kv, size // 16, 16, dim).transpose(-1, -2).contiguous()
    cache = [t.cuda() for t in (k, v, scales[0].contiguous(), scales[1].contiguous())]
    from ring_swa import KVCache

    cache = KVCache(*(t.view(torch.float8_e4m3fn) for t in cache[:2]), *(t.view(torch.float8_e8m0fnu) for t in cache[2:]))
    return cache, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), order[at:]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def randn(g, dtype, *shape):
    return torch.randn(*shape, generator=g).to(dtype).cuda()


def score_error(reach, dim):
    return reach * (dim * 2.0 ** -24 + 2.0 ** -21)


def check_attn(q, cache, table, lens, out, lse, window=-1, cu=None, scale=None, sinks=0):
    want, want_lse, spread, reach, total = O.attn(q, cache, table, lens, window, cu, scale, sinks)
    rows = slice(None) if cu is None else slice(0, int(cu[-1]))
    out, want, spread = out[rows], want[rows], spread[rows]
    err = score_error(reach, q.shape[-1])
    per_row = err.transpose(-1, -2)[rows][..., None]
    bound = HALF[q.dtype] * (want.abs() + spread) + (2 * per_row + 2.0 ** -17) * spread + 2.0 ** -24
    if q.dtype == torch.float16:
        bound = bound + 2.0 ** -39 * total[rows]
    off = (out.double() - want).abs()
    assert torch.isfinite(out.float()).all()
    assert bool((off <= bound).all()), f"out off by up to {(off / bound).max().item():.2f} of its bound"
    if lse is not None:
        pick = (lambda t: t) if cu is None else (lambda t: t[:, rows])
        lse, want_lse, err = pick(lse), pick(want_lse), pick(err)
        empty = want_lse == -math.inf
        assert bool((lse[empty] == -math.inf).all()) and bool((out.transpose(-2, -3)[empty] == 0).all()
                                                               if cu is None else
                                                               (out.transpose(0, 1)[empty] == 0).all())
        off = (lse.double() - want_lse).abs()[~empty]
        assert bool((off <= (err + 2.0 ** -20 * (1 + want_lse.abs()))[~empty]).all()), f"lse off by {off.max()}"


# ---- append -------------------------------------------------------------------------------------
APPEND = [
    # lens before, new rows (a list: packed), kv heads, dim, page, dtype
    ([0], 1, 8, 128, 64, "bf16"),
    ([5, 63, 64, 127], 1, 2, 128, 64, "bf16"),
    ([0, 1, 15, 16, 17], 1, 3, 64, 16, "fp16"),
    ([0, 7], 100, 2, 128, 32, "bf16"),
    ([250, 3], 300, 1, 64, 256, "fp16"),
    ([10, 0, 200, 77], [5, 0, 1, 130], 4, 128, 64, "bf16"),
    ([0, 0, 128], [33, 1, 128], 2, 64, 128, "fp16"),
    ([i % 37 for i in range(70)], [i % 5 for i in range(70)], 1, 64, 16, "bf16"),
]


@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append_writes_the_restatements_bytes(case):
    from ring_swa import kv_cache_append

    held, new, hk, dim, size, dtype = APPEND[case]
    dtype = DTYPES[dtype]
    packed = isinstance(new, list)
    count = new if packed else [new] * len(held)
    cache, table, _, _ = make([h + n for h, n in zip(held, count)], hk, dim, size, case, wild=False)
    lens = ints(held)
    g = torch.Generator().manual_seed(100 + case)
    cu = None
    if packed:
        cu = ints([sum(new[:i]) for i in range(len(new) + 1)])
        shape = (sum(new) + 3, hk, dim)  # (rows behind the last sequence: not taken)
    else:
        shape = (len(held), new, hk, dim)
    # amplitudes from far below to far above what the pages hold: scales stay and grow
    k, v = (randn(g, torch.float32, *shape) * torch.exp2(torch.randint(-12, 9, (*shape[:-1], 1), generator=g).float()).cuda()
            for _ in range(2))
    k, v = k.to(dtype), v.to(dtype)
    want = O.append(cache, k, v, table, lens, cu)
    kv_cache_append(cache, k, v, table, lens, cu)
    assert O.same_bytes(cache, want)
    assert lens.tolist() == held
    kv_cache_append(cache, k, v, table, lens, cu)  # the same again changes nothing
    assert O.same_bytes(cache, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("held", [0, 9])
def test_append_of_extreme_values(dtype, held):
    """Infinities, NaN, zeros alone, the type's largest and smallest values, and every rounding of the type's
    values around the codes."""
    from ring_swa import kv_cache_append

    dtype = DTYPES[dtype]
    info = torch.finfo(dtype)
    rows = [torch.zeros(128), torch.full((128,), info.max), torch.full((128,), info.tiny), torch.full((128,), -info.max),
            torch.full((128,), math.nan), torch.full((128,), math.inf),
            torch.cat([torch.full((64,), -math.inf), torch.linspace(-3, 3, 64)]),
            448 + torch.arange(128) / 8.0, torch.arange(128) * 3.5 + 0.25, 2.0 ** -10 * torch.arange(128)]
    for j, row in enumerate(rows):
        cache, table, lens, _ = make([held + 1], 1, 128, 64, 7, wild=False)
        lens -= 1
        x = row.to(dtype).cuda().view(1, 1, 1, 128)
        want = O.append(cache, x, x, table, lens)
        kv_cache_append(cache, x, x, table, lens)
        assert O.same_bytes(cache, want), f"row {j}"


def test_append_token_by_token_equals_the_restatement():
    from ring_swa import KVCache, kv_cache_append

    g = torch.Generator().manual_seed(3)
    cache = KVCache.empty(6, 2, 64, 32, device="cuda")
    table = ints([[4, 1, 3], [0, 5, 2]])
    lens = ints([0, 30])
    want = tuple(t.clone() for t in cache)
    for step in range(60):
        k, v = (randn(g, torch.bfloat16, 2, 1, 2, 64) * 1.15 ** step for _ in range(2))
        want = O.append(want, k, v, table, lens)
        kv_cache_append(cache, k, v, table, lens)
        lens += 1
    assert O.same_bytes(cache, want)


def test_append_drops_what_has_no_page():
    from ring_swa import kv_cache_append

    g = torch.Generator().manual_seed(4)
    cache, table, _, _ = make([64] * 4, 2, 64, 16, 9, wild=False)
    table[0, 1] = -1               # a page that is not there
    table[1, 0] = cache.k.shape[0]  # one beyond the pool
    table[2, 2] = 2 ** 31 - 1
    lens = ints([0, 0, 60, 10 ** 9])  # the third runs over its row of the table, the fourth is beyond it
    k, v = (randn(g, torch.bfloat16, 4, 40, 2, 64) for _ in range(2))
    want = O.append(cache, k, v, table, lens)
    kv_cache_append(cache, k, v, table, lens)
    assert O.same_bytes(cache, want)
    # lengths below zero count as none
    kv_cache_append(cache, k, v, table, ints([-5, -1, -2 ** 31, -3]))
    assert O.same_bytes(cache, O.append(want, k, v, table, ints([0, 0, 0, 0])))


# ---- attention ----------------------------------------------------------------------------------
ATTN = [
    # lens (with the new rows), new rows (a list: packed), q heads, kv heads, dim, page, window, sinks, dtype
    ([1], 1, 4, 4, 128, 64, -1, 0, "bf16"),
    ([0, 1, 2, 63, 64, 65, 300], 1, 8, 2, 128, 64, -1, 0, "bf16"),
    ([0, 1, 2, 63, 64, 65, 300], 1, 8, 2, 64, 16, 50, 4, "fp16"),
    ([5000], 1, 32, 8, 128, 64, -1, 0, "bf16"),
    ([4097, 3], 1, 28, 4, 64, 16, 1000, 4, "fp16"),
    ([700, 1300], 1, 32, 1, 128, 32, 0, 0, "bf16"),       # a window of the token alone, 32 heads on one
    ([700, 1300], 1, 48, 1, 64, 256, 100, 70, "bf16"),    # sinks over more than a tile
    ([900, 40, 7], 5, 8, 2, 128, 128, 128, 1, "bf16"),
    ([900, 3, 0], 5, 32, 8, 128, 32, -1, 0, "fp16"),      # rows ahead of the sequence's start see nothing
    ([1000, 555], 17, 12, 12, 64, 64, 90, 100, "bf16"),
    ([777], 200, 8, 2, 128, 64, -1, 0, "bf16"),
    ([777, 200], 200, 4, 4, 64, 16, 150, 4, "fp16"),
    ([1500, 130], 129, 6, 2, 128, 32, 300, 130, "bf16"),
    ([300, 0, 64, 1000, 5], [1, 0, 64, 3, 5], 8, 2, 128, 64, -1, 0, "bf16"),
    ([300, 9, 640, 1000, 5], [1, 0, 600, 3, 5], 8, 2, 64, 32, 200, 4, "fp16"),
    ([2, 3], [4, 5], 8, 2, 128, 64, -1, 0, "bf16"),       # more rows than tokens
    ([(i * 37) % 500 for i in range(150)], 1, 4, 2, 64, 16, -1, 0, "bf16"),
    ([64 + (i * 29) % 300 for i in range(65)], [i % 4 for i in range(65)], 4, 2, 64, 16, 33, 2, "bf16"),
]


@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention(case):
    from ring_swa import kv_cache_attn

    lens, new, hq, hk, dim, size, window, sinks, dtype = ATTN[case]
    cache, table, seqlens, _ = make(lens, hk, dim, size, case, max_pages=max(-(-n // size) for n in lens) + case % 3)
    g = torch.Generator().manual_seed(200 + case)
    cu = None
    if isinstance(new, list):
        cu = ints([sum(new[:i]) for i in range(len(new) + 1)])
        q = randn(g, DTYPES[dtype], sum(new), hq, dim)
    else:
        q = randn(g, DTYPES[dtype], len(lens), new, hq, dim)
    out, lse = kv_cache_attn(q, cache, table, seqlens, window, cu, num_sink_tokens=sinks, return_lse=True)
    check_attn(q, cache, table, seqlens, out, lse, window, cu, None, sinks)
    alone = kv_cache_attn(q, cache, table, seqlens, window, cu, num_sink_tokens=sinks)
    assert torch.equal(alone, out)


@pytest.mark.parametrize("new,heads", [(1, (8, 2)), (40, (4, 4))])
def test_attention_over_a_long_cache(new, heads):
    """Keys shared by many blocks: partial results and their join; with a scale of the caller's."""
    from ring_swa import kv_cache_attn

    lens = [70001, 129, 1500]
    cache, table, seqlens, _ = make(lens, heads[1], 64, 64, 31)
    g = torch.Generator().manual_seed(5)
    q = randn(g, torch.bfloat16, 3, new, heads[0], 64)
    out, lse = kv_cache_attn(q, cache, table, seqlens, softmax_scale=0.2, return_lse=True)
    check_attn(q, cache, table, seqlens, out, lse, scale=0.2)


def test_attention_with_pages_missing():
    """Pages that a window has left behind, and others: their keys are seen by nobody, whatever their number."""
    from ring_swa import kv_cache_attn

    for size in (16, 64, 256):
        cache, table, seqlens, _ = make([1000, 900, 60], 2, 128, size, 40 + size)
        table[0, :2] = -1
        table[1, 1] = cache.k.shape[0] + 5
        table[1, table.shape[1] - 1] = -2 ** 31
        table[2] = -1  # nothing at all
        q = randn(torch.Generator().manual_seed(6), torch.bfloat16, 3, 2, 8, 128)
        out, lse = kv_cache_attn(q, cache, table, seqlens, return_lse=True)
        check_attn(q, cache, table, seqlens, out, lse)
        assert bool((lse[2] == -math.inf).all())


def test_lengths_beyond_the_table_are_cut():
    from ring_swa import kv_cache_attn

    cache, table, seqlens, _ = make([128, 64], 2, 64, 64, 44)
    q = randn(torch.Generator().manual_seed(7), torch.bfloat16, 2, 3, 4, 64)
    want = kv_cache_attn(q, cache, table[:, :1], ints([64, 64]))
    assert torch.equal(kv_cache_attn(q, cache, table[:, :1], ints([10 ** 9, 64])), want)
    out, lse = kv_cache_attn(q, cache, table, ints([-4, -2 ** 31]), return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_attention_masks_infinities_and_nan_of_single_tokens():
    """A single token's query is not touched by NaN codes outside its window, in whole and in cut tiles."""
    from ring_swa import kv_cache_attn

    cache, table, seqlens, _ = make([500], 1, 64, 16, 45)
    k, v = (t.view(torch.uint8) for t in cache[:2])
    window, sinks = 100, 5
    for j in list(range(sinks, 500 - 1 - window)):
        page, place = int(table[0, j // 16]), j % 16
        k[page, 0, place] = NAN_CODE
        v[page, 0, place // 16, :, place % 16] = NAN_CODE
    q = randn(torch.Generator().manual_seed(8), torch.float16, 1, 1, 4, 64)
    out, lse = kv_cache_attn(q, cache, table, seqlens, window, num_sink_tokens=sinks, return_lse=True)
    check_attn(q, cache, table, seqlens, out, lse, window, None, None, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_values_next_to_the_types_largest(dtype):
    """Rounding to e4m3 lifts 65000 to 65536 = 2^16, past fp16's range (and 3.3e38 to 2^128): a key's scores and the
    product with V must not overflow where the results do not."""
    from ring_swa import KVCache, kv_cache_append, kv_cache_attn

    dtype = DTYPES[dtype]
    cache = KVCache.empty(2, 1, 64, 64, device="cuda")
    table, lens = ints([[1]]), ints([0])
    k = torch.full((1, 8, 1, 64), torch.finfo(dtype).max, dtype=dtype, device="cuda")
    v = k * 0.25
    v[0, 3] = torch.finfo(dtype).max
    kv_cache_append(cache, k, v, table, lens)
    q = torch.zeros(1, 1, 2, 64, dtype=dtype, device="cuda")
    q[..., 0], q[..., 1] = torch.finfo(dtype).tiny, -torch.finfo(dtype).tiny
    out, lse = kv_cache_attn(q, cache, table, ints([8]), return_lse=True)
    check_attn(q, cache, table, ints([8]), out, lse)
    assert out.float().abs().max() > 0.2 * torch.finfo(dtype).max


def test_strided_queries_rows_and_caches():
    """q as a slice of a fused projection, k and v too, the caches of two layers in one tensor, a table that is a
    slice of a wider one: as their dense copies."""
    from ring_swa import KVCache, kv_cache_append, kv_cache_attn, kv_cache_weights

    g = torch.Generator().manual_seed(9)
    b, s, hq, hk, d, size, pages = 3, 4, 8, 2, 128, 32, 40
    fused = randn(g, torch.bfloat16, b, s, hq + 2 * hk, d)
    q, k, v = fused.split([hq, hk, hk], dim=2)
    pool = torch.randint(0, 0x78, (pages, 2, 2, hk, size * d), generator=g, dtype=torch.uint8).cuda()
    scales = torch.full((2, hk, 2, pages), 124, dtype=torch.uint8, device="cuda")
    for layer in (0, 1):
        ks, vs = (scales[layer].permute(1, 2, 0)[i].view(torch.float8_e8m0fnu) for i in (0, 1))
        cache = KVCache(pool[:, layer, 0].view(torch.float8_e4m3fn).view(pages, hk, size, d),
                        pool[:, layer, 1].view(torch.float8_e4m3fn).view(pages, hk, size // 16, d, 16), ks, vs)
        dense = KVCache(*(t.contiguous() for t in cache))
        before = pool[:, 1 - layer].clone()
        wide = torch.randperm(pages, generator=g)[:36].view(3, 12).to(torch.int32).cuda()
        table, held = wide[:, 2:9], ints([100, 0, 31])
        for c, tensors in ((cache, (k, v)), (dense, (k.contiguous(), v.contiguous()))):
            kv_cache_append(c, *tensors, table, held)
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(cache, dense))
        assert torch.equal(pool[:, 1 - layer], before)
        lens = held + s
        out, lse = kv_cache_attn(q, cache, table, lens, 60, num_sink_tokens=3, return_lse=True)
        out2, lse2 = kv_cache_attn(q.contiguous(), dense, table.contiguous(), lens, 60, num_sink_tokens=3,
                                   return_lse=True)
        assert torch.equal(out, out2) and torch.equal(lse, lse2)
        check_attn(q, cache, table, lens, out, lse, 60, None, None, 3)
        w, w2 = torch.zeros(b, 2 * hk, 250, device="cuda")[:, ::2, :200], torch.zeros(b, hk, 200, device="cuda")
        kv_cache_weights(q, cache, table, lens, lse, w, 60, num_sink_tokens=3)
        kv_cache_weights(q.contiguous(), dense, table, lens, lse, w2, 60, num_sink_tokens=3)
        assert torch.equal(w, w2)


def test_pools_beyond_4_gib():
    """Pages whose offsets pass 32 bits, at the pool's both ends."""
    from ring_swa import KVCache, kv_cache_append, kv_cache_attn, kv_cache_evict, kv_cache_weights

    pages = (5 << 30) // (8 * 64 * 128)
    cache = KVCache.empty(pages, 8, 128, device="cuda")
    table = ints([[pages - 1, 0, pages - 2], [1, pages - 3, 2]])
    g = torch.Generator().manual_seed(10)
    k, v = (randn(g, torch.bfloat16, 2, 150, 8, 128) for _ in range(2))
    kv_cache_append(cache, k, v, table, ints([0, 0]))
    lens = ints([150, 150])
    # the same in a small pool
    small = KVCache.empty(6, 8, 128, device="cuda")
    kv_cache_append(small, k, v, ints([[0, 1, 2], [3, 4, 5]]), ints([0, 0]))
    q = randn(g, torch.bfloat16, 2, 2, 32, 128)
    out, lse = kv_cache_attn(q, cache, table, lens, return_lse=True)
    want, want_lse = kv_cache_attn(q, small, ints([[0, 1, 2], [3, 4, 5]]), lens, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    w = torch.zeros(2, 8, 192, device="cuda")
    kv_cache_weights(q, cache, table, lens, lse, w)
    want_w = torch.zeros_like(w)
    kv_cache_weights(q, small, ints([[0, 1, 2], [3, 4, 5]]), lens, lse, want_w)
    assert torch.equal(w, want_w)
    new = ints([[pages - 5, 7], [8, pages - 7]])
    n, _, kept = kv_cache_evict(cache, w, table, lens, new, 100, num_sink_tokens=1, num_recent=7)
    assert n.tolist() == [100, 100]
    x, _ = O.gather(cache, 0, new, 1, 3, torch.arange(100, device="cuda"))
    y, _ = O.gather(cache, 0, table, 1, 3, kept[1, 3].long())
    assert torch.allclose(x, y, atol=2.0 ** -8, rtol=2.0 ** -4)  # (codes may be rounded anew)


# ---- weights ------------------------------------------------------------------------------------
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_weights(case):
    from ring_swa import kv_cache_attn, kv_cache_weights

    lens, new, hq, hk, dim, size, window, sinks, dtype = ATTN[case]
    cache, table, seqlens, _ = make(lens, hk, dim, size, case)
    g = torch.Generator().manual_seed(300 + case)
    cu = None
    if isinstance(new, list):
        cu = ints([sum(new[:i]) for i in range(len(new) + 1)])
        q = randn(g, DTYPES[dtype], sum(new), hq, dim)
    else:
        q = randn(g, DTYPES[dtype], len(lens), new, hq, dim)
    _, lse = kv_cache_attn(q, cache, table, seqlens, window, cu, num_sink_tokens=sinks, return_lse=True)
    width = max(1, max(lens) - 7 * (case % 2))
    running = torch.rand(len(lens), hk, width, generator=g).cuda()
    want, off = O.weights(q, cache, table, seqlens, lse, running, window, cu, None, sinks)
    got = running.clone()
    kv_cache_weights(q, cache, table, seqlens, lse, got, window, cu, num_sink_tokens=sinks)
    bound = 2 * score_error(off, dim) + 2.0 ** -17 * (want - running.double()) + 2.0 ** -23 * want + 2.0 ** -40
    diff = (got.double() - want).abs()
    assert bool((diff <= bound).all()), f"off by up to {(diff / bound).max().item():.2f} of the bound"
    # what a row adds over all keys is 1
    if cu is None and width >= max(lens) and min(lens) >= new:
        assert torch.allclose((got - running).double().sum((1, 2)), torch.full((len(lens),), 1.0 * new * hq).double().cuda(),
                              rtol=2.0 ** -12)
    again = running.clone()
    kv_cache_weights(q, cache, table, seqlens, lse, again, window, cu, num_sink_tokens=sinks)
    assert torch.equal(got, again)


# ---- eviction -----------------------------------------------------------------------------------
EVICT = [
    # lens, budget, sinks, recent, kv heads, dim, page, weights
    ([200, 100, 50, 0], 100, 4, 20, 2, 64, 16, "tail"),
    ([1000, 300], 64, 0, 0, 2, 128, 64, "tail"),
    ([1000, 301], 300, 10, 290, 1, 128, 32, "tail"),      # sinks and recent tokens fill the budget
    ([500, 77], 130, 1, 60, 3, 64, 256, "equal"),
    ([500, 77, 128], 100, 4, 30, 2, 128, 128, "zeros"),
    ([700], 130, 2, 5, 2, 64, 64, "wild"),                # NaN, infinities, both zeros, negative ones
    ([3000, 2049, 1], 2048, 4, 512, 1, 64, 64, "few"),    # many equal ones around the least that stays
    ([40, 17], 1, 0, 0, 2, 64, 16, "tail"),
    ([300, 5], 90, 1, 1, 2, 64, 16, "short"),             # weights for fewer tokens than there are
]


@pytest.mark.parametrize("case", range(len(EVICT)))
def test_evict(case):
    from ring_swa import kv_cache_evict

    lens, budget, sinks, recent, hk, dim, size, kind = EVICT[case]
    per = -(-budget // size)
    cache, table, seqlens, free = make(lens, hk, dim, size, 60 + case, spare=per * len(lens) + 1, wild=False)
    new_table = ints(free[:per * len(lens)]).view(len(lens), per)
    if case == 1:
        new_table[1, 0] = -1  # a new page that is not there: its tokens are lost, nothing else
        table[0, 3] = -1      # ... and an old one: its tokens become zeros
    g = torch.Generator().manual_seed(400 + case)
    width = max(lens) if kind != "short" else 100
    w = torch.exp(2 * torch.randn(len(lens), hk, width, generator=g))
    if kind == "equal":
        w = torch.full_like(w, 0.25)
    elif kind == "zeros":
        w = w * (torch.rand(w.shape, generator=g) < 0.2)
    elif kind == "wild":
        pick = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, -1.0, 1.0, 2.0 ** -149, -2.0 ** -149, 3.0])
        w = pick[torch.randint(0, 10, w.shape, generator=g)]
    elif kind == "few":
        w = torch.randint(0, 3, w.shape, generator=g).float()
    w = w.cuda()
    want, want_n, want_w, want_kept = O.evict(cache, w, table, seqlens, new_table, budget, sinks, recent)
    before = w.clone()
    n, new_w, kept = kv_cache_evict(cache, w, table, seqlens, new_table, budget, num_sink_tokens=sinks, num_recent=recent)
    assert torch.equal(n.cpu(), want_n) and torch.equal(kept.cpu(), want_kept)
    assert torch.equal(new_w.cpu().nan_to_num(nan=77.0), want_w.nan_to_num(nan=77.0))
    assert torch.equal(w.nan_to_num(nan=77.0), before.nan_to_num(nan=77.0)) and seqlens.tolist() == lens
    assert O.same_bytes(cache, want)


def test_evict_of_sequences_that_share_pages():
    from ring_swa import kv_cache_evict

    cache, table, seqlens, free = make([200], 2, 64, 16, 80, spare=20, wild=False)
    table, seqlens = table.repeat(2, 1), ints([200, 180])
    new_table = ints(free[:14]).view(2, 7)
    w = torch.rand(2, 2, 200, generator=torch.Generator().manual_seed(1)).cuda()
    want, _, _, want_kept = O.evict(cache, w, table, seqlens, new_table, 100, 1, 10)
    _, _, kept = kv_cache_evict(cache, w, table, seqlens, new_table, 100, num_sink_tokens=1, num_recent=10)
    assert torch.equal(kept.cpu(), want_kept) and O.same_bytes(cache, want)


# ---- together -----------------------------------------------------------------------------------
def test_prompt_then_tokens_then_eviction():
    """As a server runs them: prompts through the streaming-LLM attention, into the cache, drafts and single tokens
    with running sums, eviction, and on.  Every step against the restatement, which is fed the same cache."""
    from ring_swa import (KVCache, kv_cache_append, kv_cache_attn, kv_cache_evict, kv_cache_weights,
                          ring_streaming_llm_attn_varlen)

    g = torch.Generator().manual_seed(11)
    hq, hk, d, size, window, sinks = 8, 2, 128, 32, 120, 4
    prompts = [150, 33, 260]
    cu = ints([0, 150, 183, 443])
    cache = KVCache.empty(60, hk, d, size, device="cuda")
    order = torch.randperm(60, generator=g).to(torch.int32).cuda()
    table = order[:30].view(3, 10)
    q = randn(g, torch.bfloat16, 443, hq, d)
    k, v = (randn(g, torch.bfloat16, 443, hk, d) for _ in range(2))
    held = ints([0, 0, 0])
    kv_cache_append(cache, k, v, table, held, cu)
    held = held + ints(prompts)
    # the cache continues the 16-bit prompt: its outputs differ by the codes' rounding alone
    full = ring_streaming_llm_attn_varlen(q, k, v, window, cu, num_sink_tokens=sinks)
    cached, lse = kv_cache_attn(q, cache, table, held, window, cu, num_sink_tokens=sinks, return_lse=True)
    check_attn(q, cache, table, held, cached, lse, window, cu, None, sinks)
    assert ((full - cached).float().norm() / full.float().norm()).item() < 0.06
    weights = torch.zeros(3, hk, 10 * size, device="cuda")
    running = weights.double()
    for step in range(7):
        n = (1, 3, 1, 2, 1, 1, 1)[step]
        q, k, v = (randn(g, torch.bfloat16, 3, n, h, d) for h in (hq, hk, hk))
        want = O.append(cache, k, v, table, held)
        kv_cache_append(cache, k, v, table, held)
        assert O.same_bytes(cache, want)
        held = held + n
        out, lse = kv_cache_attn(q, cache, table, held, window, num_sink_tokens=sinks, return_lse=True)
        check_attn(q, cache, table, held, out, lse, window, None, None, sinks)
        running, off = O.weights(q, cache, table, held, lse, weights, window, None, None, sinks)
        kv_cache_weights(q, cache, table, held, lse, weights, window, num_sink_tokens=sinks)
        assert bool(((weights.double() - running).abs() <= 2 * score_error(off, d) + 2.0 ** -16 * running + 2.0 ** -40).all())
        if step == 4:
            new_table = order[30:60].view(3, 10)
            want, want_n, want_w, want_kept = O.evict(cache, weights, table, held, new_table, 96, sinks, 40)
            held, weights, kept = kv_cache_evict(cache, weights, table, held, new_table, 96, num_sink_tokens=sinks,
                                                 num_recent=40)
            assert O.same_bytes(cache, want) and torch.equal(kept.cpu(), want_kept)
            assert torch.equal(held.cpu(), want_n) and torch.equal(weights.cpu(), want_w)
            table = new_table


def test_partial_results_of_cache_and_new_keys_merge():
    """The lse is what the merge operator takes: cache before the chunk and the chunk's own 16-bit keys apart."""
    from ring_swa import kv_cache_attn
    from ring_swa.ops import attn_fwd, merge_attn_out

    cache, table, seqlens, _ = make([300, 210], 2, 128, 64, 90)
    g = torch.Generator().manual_seed(12)
    n = 50
    q, k, v = (randn(g, torch.bfloat16, 2, n, h, 128) for h in (8, 2, 2))
    own, own_lse = attn_fwd(q, k, v, None, (-1, 0), True)
    # every row of the chunk sees all that the cache holds: a pack of single rows, each the last of its sequence
    flat = q.reshape(2 * n, 1, 8, 128)
    out, lse = kv_cache_attn(flat, cache, table.repeat_interleave(n, 0), seqlens.repeat_interleave(n), return_lse=True)
    out = out.view(2, n, 8, 128)
    lse = lse.view(2, n, 8).transpose(1, 2).contiguous()
    merge_attn_out(own, own_lse, out, lse)
    for b in range(2):
        for h in range(2):
            j = torch.arange(int(seqlens[b]), device="cuda")
            keys = torch.cat([O.gather(cache, 0, table, b, h, j)[0], k[b, :, h].double()])
            values = torch.cat([O.gather(cache, 1, table, b, h, j)[0], v[b, :, h].double()])
            z = torch.einsum("sgd,jd->gsj", q[b, :, 4 * h:4 * h + 4].double(), keys) * 128 ** -0.5
            at = torch.arange(keys.shape[0], device="cuda")
            z = z.masked_fill(at[None, :] > len(j) + torch.arange(n, device="cuda")[:, None], -math.inf)
            want = (torch.softmax(z, -1) @ values).transpose(0, 1)
            spread = (torch.softmax(z, -1) @ values.abs()).transpose(0, 1)
            # three roundings of out (two partial results, the merge), the weights' rounding, and scores
            bound = 2.0 ** -8 * (4 * spread + want.abs()) + 2.0 ** -10
            assert bool(((own[b, :, 4 * h:4 * h + 4].double() - want).abs() <= bound).all())


# ---- graphs, streams ------------------------------------------------------------------------------
def _step(cache, table, q, k, v, held, lens, weights, new_table):
    from ring_swa import kv_cache_append, kv_cache_attn, kv_cache_evict, kv_cache_weights

    kv_cache_append(cache, k, v, table, held)
    out, lse = kv_cache_attn(q, cache, table, lens, return_lse=True)
    kv_cache_weights(q, cache, table, lens, lse, weights)
    return out, lse, *kv_cache_evict(cache, weights, table, lens, new_table, 700, num_sink_tokens=2, num_recent=30)


def test_a_captured_step_replays():
    """One graph of all four calls, replayed on changed inputs and lengths with eager work in between; two graphs that
    share a memory pool."""
    cache, table, lens, free = make([3000, 900, 1], 2, 64, 32, 95, spare=3 * 22 + 1, max_pages=100, wild=False)
    new_table = ints(free[:66]).view(3, 22)
    held = lens - 1
    g = torch.Generator().manual_seed(13)
    q = randn(g, torch.bfloat16, 3, 1, 8, 64)
    k, v = (randn(g, torch.bfloat16, 3, 1, 2, 64) for _ in range(2))
    weights = torch.rand(3, 2, 3200, generator=g).cuda()
    args = (cache, table, q, k, v, held, lens, weights, new_table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(*args)
    with torch.cuda.graph(other, pool=graph.pool()):
        got2 = _step(*args)
    for trial in range(4):
        q.copy_(randn(g, torch.bfloat16, *q.shape))
        k.copy_(randn(g, torch.bfloat16, *k.shape))
        new = ints([(3000, 900, 1), (1500, 32, 64), (2999, 1, 33), (90, 800, 2)][trial])
        lens.copy_(new)
        held.copy_(new - 1)
        start = torch.rand(3, 2, 3200, generator=g).cuda()
        state = tuple(t.clone() for t in cache)
        for which, (run, outs) in enumerate(((graph, got), (other, got2))):
            weights.copy_(start)
            for t, s in zip(cache, state):
                t.copy_(s)
            run.replay()
            torch.cuda.synchronize()
            replayed = [t.clone() for t in (*outs, weights, *(t.view(torch.uint8) for t in cache))]
            weights.copy_(start)
            for t, s in zip(cache, state):
                t.copy_(s)
            eager = [*_step(*args), weights, *(t.view(torch.uint8) for t in cache)]
            torch.cuda.synchronize()
            for x, y in zip(replayed, eager):
                assert torch.equal(x, y), f"trial {trial}, graph {which}"


def test_calls_on_two_streams_at_once():
    from ring_swa import kv_cache_attn

    cache, table, lens, _ = make([20000, 300, 9000], 2, 64, 64, 96)
    g = torch.Generator().manual_seed(14)
    qs = [randn(g, torch.bfloat16, 3, 1, 8, 64) for _ in range(8)]
    want = [kv_cache_attn(q, cache, table, lens) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(kv_cache_attn(q, cache, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_rows_behind_the_last_sequence_are_left():
    """Through the C ABI, into buffers that hold something; and cu_seqlens that overlap or leave the tensor."""
    from ring_swa import _lib
    from ring_swa.ops import kv_cache as K

    cache, table, lens, _ = make([500, 700], 2, 64, 16, 97)
    q = randn(torch.Generator().manual_seed(15), torch.bfloat16, 90, 8, 64)
    L = _lib.lib()

    def call(cu):
        p, dev = K._cache_params(cache, table, lens, q, cu)
        K._query_params(p, q, 2, None, -1, 0, True)
        out = torch.full_like(q, 7.0)
        lse = torch.full((8, 90), 7.0, device="cuda")
        p.out, p.out_stride, p.lse, p.lse_stride = out.data_ptr(), (0, 512, 64), lse.data_ptr(), (0, 90, 1)
        ws = torch.empty(int(L.rswa_cache_attn_workspace_bytes(p)), dtype=torch.uint8, device="cuda")
        p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
        _lib.launch(dev, L.rswa_cache_attn, p)
        torch.cuda.synchronize()
        return out, lse

    cu = ints([0, 3, 70])
    out, lse = call(cu)
    check_attn(q, cache, table, lens, out, lse, cu=cu)
    assert bool((out[70:] == 7).all()) and bool((lse[:, 70:] == 7).all())
    for wild in ([0, 90, 0], [-5, 50, 10 ** 9], [80, 20, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31, 5]):
        call(ints(wild))  # (rows of no sequence, or of two: any values, nothing outside the buffers)


def test_random_calls():
    from ring_swa import kv_cache_attn

    rng = random.Random(5)
    for trial in range(25):
        hk = rng.choice([1, 2, 4])
        hq = hk * rng.choice([1, 2, 3, 7, 8, 20])
        dim, size = rng.choice([64, 128]), rng.choice([16, 32, 64, 128, 256])
        batch = rng.choice([1, 2, 5])
        new = rng.choice([1, 1, 2, 6, 30, 70])
        lens = [rng.choice([0, 1, rng.randrange(1, 200), rng.randrange(1, 3000)]) for _ in range(batch)]
        window = rng.choice([-1, 0, rng.randrange(1, 400)])
        sinks = rng.choice([0, 1, 4, 65])
        dtype = rng.choice([torch.bfloat16, torch.float16])
        cache, table, seqlens, _ = make(lens, hk, dim, size, trial)
        q = randn(torch.Generator().manual_seed(trial), dtype, batch, new, hq, dim)
        if table.shape[1] == 0:
            continue
        out, lse = kv_cache_attn(q, cache, table, seqlens, window, num_sink_tokens=sinks, return_lse=True)
        check_attn(q, cache, table, seqlens, out, lse, window, None, None, sinks)
