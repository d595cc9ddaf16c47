"""Page tables without columns.  Attention through the C ABI: no keys at all, so every row of a sequence is 0 and its lse
-inf (the Python function answers such calls by itself).  Eviction: nothing to keep."""
import math

import pytest
import torch

from ring_swa import _lib
from ring_swa.ops import kv_cache as K
from test_kv_cache_gpu import DTYPES, ints, make


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("new,heads,packed", [(1, 4, False), (9, 8, False), (600, 32, False), (40, 8, True), (1100, 32, True)])
def test_a_table_without_columns(new, heads, packed, dtype):
    cache, table, lens, _ = make([40, 7], 2, 128, 16, 1)
    lead = (new,) if packed else (2, new)
    cu = ints([0, new // 2, new - 3]) if packed else None
    q = torch.ones(*lead, heads, 128, dtype=DTYPES[dtype], device="cuda")
    p, dev = K._cache_params(cache, table[:, :0], lens, q, cu)
    assert p.max_pages == 0
    K._query_params(p, q, 2, None, -1, 0, packed)
    out = torch.full_like(q, 7.0)
    lse = torch.full((heads, new) if packed else (2, heads, new), 7.0, device="cuda")
    p.out, p.out_stride = out.data_ptr(), K._strides3(out, packed)
    p.lse, p.lse_stride = lse.data_ptr(), K._strides3(lse, packed)
    assert _lib.lib().rswa_cache_attn_workspace_bytes(p) == 0
    _lib.launch(dev, _lib.lib().rswa_cache_attn, p)
    rows = new - 3 if packed else new
    assert bool((out[..., :rows, :, :] == 0).all()) and bool((lse[..., :rows] == -math.inf).all())
    assert bool((out[..., rows:, :, :] == 7).all()) and bool((lse[..., rows:] == 7).all())


@pytest.mark.gpu
def test_eviction_from_tables_without_columns():
    from ring_swa import kv_cache_evict

    cache, table, lens, _ = make([40, 7], 2, 128, 16, 2)
    before = [t.view(torch.uint8).clone() for t in cache]
    w = torch.rand(2, 2, 50, device="cuda")
    for new in (table[:, :0].clone(), table):
        n, new_w, kept = kv_cache_evict(cache, w, table[:, :0], lens, new, 5, num_sink_tokens=1, num_recent=2)
        assert n.tolist() == [0, 0] and bool((new_w == 0).all()) and bool((kept == -1).all())
    assert all(torch.equal(t.view(torch.uint8), was) for t, was in zip(cache, before))
