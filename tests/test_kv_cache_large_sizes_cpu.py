"""Sizes that 32 bits do not hold are refused, and not cut to what is left of them; and batches whose lengths, which
every block of attention and weights reads, would take seconds."""
import pytest
import torch

import ring_swa
from ring_swa import KVCache, _lib
from test_kv_cache_cpu import params


@pytest.fixture(autouse=True)
def on_cpu(monkeypatch):
    """The checks ahead of the launch, with tensors that live on the CPU; the launch itself is a failure."""
    monkeypatch.setattr(_lib, "require_device", lambda *t: t[0].device)

    def launch(*_):
        raise ValueError("launched")

    monkeypatch.setattr(_lib, "launch", launch)


def inputs():
    return KVCache.empty(8, 2, 64, 16), torch.zeros(1, 3, dtype=torch.int32), torch.ones(1, dtype=torch.int32)


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 5])
def test_rows(n):
    cache, table, lens = inputs()
    k = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="2.31"):
        ring_swa.kv_cache_append(cache, k.expand(1, n, 2, 64), k.expand(1, n, 2, 64), table, lens)
    cu = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="2.31"):
        ring_swa.kv_cache_append(cache, k[0].expand(n, 2, 64), k[0].expand(n, 2, 64), table, lens, cu)
    with pytest.raises(ValueError, match="launched"):
        ring_swa.kv_cache_append(cache, k, k, table, lens)


@pytest.mark.parametrize("budget", [2 ** 31, 2 ** 32 + 16, 2 ** 70])
def test_budget(budget):
    cache, table, lens = inputs()
    with pytest.raises(AssertionError, match="2.31"):
        ring_swa.kv_cache_evict(cache, torch.zeros(1, 2, 9), table, lens, table + 3, budget)
    with pytest.raises(ValueError, match="launched"):
        ring_swa.kv_cache_evict(cache, torch.zeros(1, 2, 9), table, lens, table + 3, 16)


def test_running_sums():
    cache, table, lens = inputs()
    w = torch.zeros(1, device="meta").as_strided((1, 2, 2 ** 32 + 9), (2 ** 33, 2 ** 33, 1))
    with pytest.raises(AssertionError, match="2.31"):
        ring_swa.ops.kv_cache._weights_params(_lib.CacheParams(batch=1, heads_kv=2), cache.k, w)


@pytest.mark.parametrize("batch,heads_q,heads_kv", [(1 << 17, 32, 8), (1 << 18, 4, 2), (1 << 20, 1, 1), (1 << 15, 128, 128)])
@pytest.mark.parametrize("call", ["attn", "weights"])
def test_batches(call, batch, heads_q, heads_kv):
    L = _lib.lib()
    assert getattr(L, "rswa_cache_" + call)(params({"batch": batch, "heads_q": heads_q, "heads_kv": heads_kv}), None) == -2
    assert "2^36" in L.rswa_last_error().decode()
