"""Values that the type of the queries holds as infinite (written from bf16, read by fp16 queries; or at scales beyond
those that an append writes): they reach the rows that see them, and no others.

Half the value of code c at scale byte e is ``decode(c) * 2**(e - 128)``; it is infinite from 2^16 on in fp16, from
2^128 on in bf16."""
import math

import pytest
import torch

from test_kv_cache_gpu import DTYPES, ints, make, randn
from test_kv_cache_nan_gpu import CALLS, sees

pytestmark = pytest.mark.gpu

LIMIT = {"fp16": 16, "bf16": 128}
# where the least magnitude that is infinite is 0x78, 0x70, 0x58, 8, 4, 2, 1, and where none is
SCALES = [("fp16", e) for e in (135, 136, 137, 140, 150, 151, 152, 153, 200)] + [("bf16", e) for e in (247, 248, 250, 254)]


def infinite(dtype, e):
    """Which of the magnitudes 0 .. 0x7e are infinite."""
    values = torch.arange(0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    return values >= 2.0 ** (LIMIT[dtype] + 128 - e)


def fill(cache, dtype, e, seed):
    """All values at scale byte ``e``, one in fifty infinite and the others far below that; the same without them; which
    are infinite, laid out as the values."""
    g = torch.Generator().manual_seed(seed)
    bad = infinite(dtype, e)
    first = int(bad.int().argmax()) if bad.any() else 0x7F
    codes = torch.randint(0, max(1, first - 16), cache.v.shape, generator=g, dtype=torch.uint8)
    pick = torch.zeros(cache.v.shape, dtype=torch.bool)
    if first < 0x7F:
        pick = torch.rand(cache.v.shape, generator=g) < 0.02
    sign = torch.randint(0, 2, cache.v.shape, generator=g, dtype=torch.uint8) << 7
    wild = torch.randint(first, 0x7F, cache.v.shape, generator=g, dtype=torch.uint8) if first < 0x7F else codes
    cache.v_scale.view(torch.uint8).fill_(e)
    finite = torch.where(pick, 0, codes | sign).cuda()
    return finite, torch.where(pick, wild | sign, codes | sign).cuda(), pick.cuda()


@pytest.mark.parametrize("dtype,e", SCALES)
@pytest.mark.parametrize("case", [2, 3, 4, 5])
def test_infinite_values_are_for_the_rows_that_see_them(case, dtype, e):
    from ring_swa import kv_cache_attn

    lens, new, hq, hk, dim, size, window, sinks, _ = CALLS[case]
    lens = [min(n, 1600) for n in lens]
    cache, table, seqlens, _ = make(lens, hk, dim, size, 920 + case, wild=False)
    q = randn(torch.Generator().manual_seed(930 + case), DTYPES[dtype], len(lens), new, hq, dim)
    finite, codes, where = fill(cache, dtype, e, 7)
    # only the keys that some row does not see have infinite values
    last, table_cpu = torch.zeros(where.shape, dtype=torch.bool), table.tolist()
    for b, length in enumerate(lens):
        for j in range(length):
            if not bool(sees(new, length, window, sinks, j).all()):
                last[table_cpu[b][j // size], :, j % size // 16, :, j % 16] = True
    last = last.cuda()
    codes, where = torch.where(last, codes, finite), where & last
    v = cache.v.view(torch.uint8)
    v.copy_(finite)
    want, want_lse = kv_cache_attn(q, cache, table, seqlens, window, num_sink_tokens=sinks, return_lse=True)
    assert bool(want.isfinite().all())
    v.copy_(codes)
    out, lse = kv_cache_attn(q, cache, table, seqlens, window, num_sink_tokens=sinks, return_lse=True)
    bad = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    for b, length in enumerate(lens):
        j = torch.arange(length, device="cuda")
        page = table[b].long()[j // size]
        seen = torch.stack([sees(new, length, window, sinks, i) for i in range(length)]).T.double().cuda()  # [rows, keys]
        for h in range(hk):
            mine = where[page, h, j % size // 16, :, j % 16].double()  # [keys, dim]
            bad[b, :, h * (hq // hk):(h + 1) * (hq // hk)] = ((seen @ mine) > 0)[:, None]
    assert e in (135, 247) or bool(bad.any()) and not bool(bad.all())
    assert torch.equal(out.isfinite(), ~bad)
    assert torch.equal(out[~bad], want[~bad]) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("new", [4, 300])
def test_what_append_has_written_from_bf16(new):
    """... and its signs: with equal weights a row that sees one infinite value is infinite, with two unlike ones NaN."""
    from ring_swa import KVCache, kv_cache_append, kv_cache_attn

    heads, held = 8, 40
    cache = KVCache.empty(8, heads, 128, 64, device="cuda")
    table, n = ints([[6, 1, 5, 0, 2, 7]]), held + new
    g = torch.Generator().manual_seed(8)
    k, v = (randn(g, torch.bfloat16, 1, n, heads, 128) for _ in range(2))
    v[0, n - 3, :, 5] = 1e6
    v[0, n - 2, 1, 5] = -1e6
    v[0, n - 1, 2, 7] = -math.inf  # (stored as NaN)
    kv_cache_append(cache, k, v, table, ints([0]))
    q = torch.zeros(1, new, 4 * heads, 128, dtype=torch.float16, device="cuda")
    out = kv_cache_attn(q, cache, table, ints([n])).unflatten(2, (heads, 4)).float()
    want = torch.zeros_like(out)
    want[:, new - 3:, :, :, 5] = math.inf
    want[:, new - 2:, 1, :, 5] = math.nan
    want[:, new - 1:, 2, :, 7] = math.nan
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out == math.inf, want == math.inf)
    assert not bool((out == -math.inf).any())
    v[0, n - 3:] = 0
    kv_cache_append(cache, k, v, table, ints([0]))
    fine = kv_cache_attn(q, cache, table, ints([n])).unflatten(2, (heads, 4)).float()
    # ahead of the three tokens nothing of them is seen (their page's scale, which they raise, rounds the others' values)
    before = n - 3 - (n - 3) % 64 - held
    assert torch.equal(out[:, :max(0, before)], fine[:, :max(0, before)])
