"""Reads of the cache into rows of many layouts: what shares no element is filled, what does is refused and left."""
import pytest
import torch

from test_kv_cache_gpu import ints, make
from test_kv_cache_read_rows_cpu import LAYOUTS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name,k,v,meet", LAYOUTS, ids=[x[0].replace(" ", "_") for x in LAYOUTS])
def test_layouts_in_use(name, k, v, meet, native, monkeypatch):
    from ring_swa import _lib, kv_cache_read

    if not native:
        monkeypatch.setattr(_lib, "torch_calls", lambda: None)
    batch, rows, heads, dim = k.shape
    cache, table, _, _ = make([rows + 3] * batch, heads, dim, 32, 17, wild=False)
    first = ints([3] * batch)
    storage = k.untyped_storage()
    one = storage.data_ptr() == v.untyped_storage().data_ptr()
    at = [torch.full((s.nbytes() // 2,), 7.0, dtype=torch.bfloat16, device="cuda")
          for s in ((storage,) if one else (storage, v.untyped_storage()))]
    to = [mine.as_strided(t.shape, t.stride(), t.storage_offset()) for mine, t in zip((at[0], at[-1]), (k, v))]
    want = [torch.empty(k.shape, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    kv_cache_read(cache, *want, table, first)
    versions = [t._version for t in at]
    if meet:
        with pytest.raises(AssertionError, match="overlap"):
            kv_cache_read(cache, *to, table, first)
        assert all(bool((t == 7).all()) for t in at) and [t._version for t in at] == versions
        return
    kv_cache_read(cache, *to, table, first)
    for mine, w in zip(to, want):
        assert torch.equal(mine, w)
    written = [torch.zeros_like(t, dtype=torch.bool) for t in at]
    for mine, t in zip((written[0], written[-1]), (k, v)):
        mine.as_strided(t.shape, t.stride(), t.storage_offset()).fill_(True)
    assert all(bool((t[~w] == 7).all()) for t, w in zip(at, written))  # (nothing else)
