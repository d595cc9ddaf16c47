"""NaN in queries and in cached keys and values: it reaches the results that the formula takes it into, and no others.
Bounds of the others as in test_kv_cache_gpu."""
import math

import pytest
import torch

from test_kv_cache_gpu import DTYPES, NAN_CODE, check_attn, ints, make, randn

pytestmark = pytest.mark.gpu

# lens (with the new rows), new rows, q heads, kv heads, dim, page, window, sinks, dtype: one wave's rows of one chunk
# and of several, two tiles of rows, rows of a wave's own
CALLS = [
    ([50, 300], 1, 8, 2, 128, 64, -1, 0, "bf16"),
    ([9000, 300], 1, 8, 2, 64, 16, -1, 0, "fp16"),
    ([700, 301], 5, 8, 2, 128, 32, 130, 3, "bf16"),
    ([9000, 300], 12, 8, 2, 128, 64, -1, 0, "fp16"),
    ([1500, 333], 520, 32, 8, 128, 64, -1, 0, "bf16"),
    ([1500, 333], 520, 32, 8, 64, 16, 100, 70, "fp16"),
]


def call(case):
    lens, new, hq, hk, dim, size, window, sinks, dtype = CALLS[case]
    cache, table, seqlens, _ = make(lens, hk, dim, size, 900 + case)
    q = randn(torch.Generator().manual_seed(910 + case), DTYPES[dtype], len(lens), new, hq, dim)
    return q, cache, table, seqlens, window, sinks


def plant(cache, which, table, b, h, j, dim=slice(None)):
    """NaN as token j of sequence b (in one dimension, or all)."""
    size = cache.k.shape[2]
    page, place = int(table[b, j // size]), j % size
    t = cache[which].view(torch.uint8)
    if which == 0:
        t[page, h, place, dim] = NAN_CODE
    else:
        t[page, h, place // 16, dim, place % 16] = NAN_CODE


def sees(n_rows, length, window, sinks, j):
    """Which of the rows see key j."""
    pos = length - n_rows + torch.arange(n_rows)
    return (j <= pos) & ((window < 0) | (j >= pos - window) | (j < sinks))


@pytest.mark.parametrize("case", range(len(CALLS)))
def test_a_query_of_nan_is_its_own_row_s_alone(case):
    from ring_swa import kv_cache_attn

    q, cache, table, lens, window, sinks = call(case)
    want, want_lse = kv_cache_attn(q, cache, table, lens, window, num_sink_tokens=sinks, return_lse=True)
    bad = torch.zeros(q.shape[:3], dtype=torch.bool, device="cuda")
    bad[0, -1, 1] = bad[1, 0, 0] = bad[1, q.shape[1] // 2, -1] = True
    q[..., 3][bad] = math.nan
    # (a row ahead of the sequence's start sees nothing: 0 and -inf whatever its query is)
    bad &= (lens[:, None] - q.shape[1] + torch.arange(q.shape[1], device="cuda") >= 0)[..., None]
    out, lse = kv_cache_attn(q, cache, table, lens, window, num_sink_tokens=sinks, return_lse=True)
    assert bool(out[bad].isnan().all()) and bool(lse.transpose(1, 2)[bad].isnan().all())
    assert torch.equal(out[~bad], want[~bad]) and torch.equal(lse.transpose(1, 2)[~bad], want_lse.transpose(1, 2)[~bad])


@pytest.mark.parametrize("case", range(len(CALLS)))
def test_a_key_of_nan_is_for_the_rows_that_see_it(case):
    from ring_swa import kv_cache_attn

    q, cache, table, lens, window, sinks = call(case)
    n, group = q.shape[1], q.shape[2] // cache.k.shape[1]
    want, want_lse = kv_cache_attn(q, cache, table, lens, window, num_sink_tokens=sinks, return_lse=True)
    bad = torch.zeros(q.shape[:3], dtype=torch.bool)
    for b, length in enumerate(lens.tolist()):
        for j in (length - 1, length - n // 2 - 1, max(0, length - n - 40)):
            plant(cache, 0, table, b, b, j, dim=5)
            bad[b, :, b * group:(b + 1) * group] |= sees(n, length, window, sinks, j)[:, None]
    out, lse = kv_cache_attn(q, cache, table, lens, window, num_sink_tokens=sinks, return_lse=True)
    bad = bad.cuda()
    assert bool(out[bad].isnan().all()) and bool(lse.transpose(1, 2)[bad].isnan().all())
    assert torch.equal(out[~bad], want[~bad]) and torch.equal(lse.transpose(1, 2)[~bad], want_lse.transpose(1, 2)[~bad])


@pytest.mark.parametrize("case", range(len(CALLS)))
def test_a_query_of_nan_adds_to_the_weights_of_the_keys_that_it_sees(case):
    from ring_swa import kv_cache_attn, kv_cache_weights

    q, cache, table, lens, window, sinks = call(case)
    n, group = q.shape[1], q.shape[2] // cache.k.shape[1]
    longest = int(lens.max())
    bad = torch.zeros(len(lens), cache.k.shape[1], longest + 9, dtype=torch.bool)
    for b, row, head in ((0, n - 1, 1), (1, 0, 0), (1, n // 2, 0)):
        q[b, row, head, 3] = math.nan
        for j in range(int(lens[b])):
            bad[b, head // group, j] |= bool(sees(n, int(lens[b]), window, sinks, j)[row])
    _, lse = kv_cache_attn(q, cache, table, lens, window, num_sink_tokens=sinks, return_lse=True)
    w = torch.zeros(bad.shape, device="cuda")
    kv_cache_weights(q, cache, table, lens, lse, w, window, num_sink_tokens=sinks)
    assert torch.equal(w.isnan().cpu(), bad)


@pytest.mark.parametrize("whole_token", [True, False])
@pytest.mark.parametrize("case", range(len(CALLS)))
def test_a_value_of_nan_is_for_the_rows_that_see_it(case, whole_token):
    """... and, where it is one dimension, for that one alone."""
    from ring_swa import kv_cache_attn

    q, cache, table, lens, window, sinks = call(case)
    n, group, dim = q.shape[1], q.shape[2] // cache.k.shape[1], q.shape[3]
    want, want_lse = kv_cache_attn(q, cache, table, lens, window, num_sink_tokens=sinks, return_lse=True)
    bad = torch.zeros(q.shape, dtype=torch.bool)
    for b, length in enumerate(lens.tolist()):
        for i, j in enumerate((length - 1, length - n // 2 - 1, max(0, length - n - 40), length - n - 150, sinks - 1)):
            if j < 0:
                continue
            dims = slice(None) if whole_token else slice(dim - 1 - 21 * i, dim - 21 * i)
            plant(cache, 1, table, b, b, j, dims)
            mine = torch.zeros(dim, dtype=torch.bool)
            mine[dims] = True
            bad[b, :, b * group:(b + 1) * group] |= sees(n, length, window, sinks, j)[:, None, None] & mine
    out, lse = kv_cache_attn(q, cache, table, lens, window, num_sink_tokens=sinks, return_lse=True)
    assert torch.equal(out.isnan().cpu(), bad)
    bad = bad.cuda()
    assert torch.equal(out[~bad], want[~bad]) and torch.equal(lse, want_lse)
