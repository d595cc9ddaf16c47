"""A step of the cache's calls compiled and traced: the eager step's bits, on inputs that were not traced."""
import pytest
import torch

import ring_swa
from ring_swa import KVCache
from test_kv_cache_gpu import ints, make, randn

pytestmark = pytest.mark.gpu


def inputs(seed):
    cache, table, lens, free = make([3000, 90, 1], 2, 64, 32, 950 + seed, spare=3 * 22 + 1, max_pages=100, wild=False)
    g = torch.Generator().manual_seed(960 + seed)
    q = randn(g, torch.bfloat16, 3, 1, 8, 64)
    k, v = (randn(g, torch.bfloat16, 3, 1, 2, 64) for _ in range(2))
    return (*cache, table, lens - seed, q, k, v, torch.rand(3, 2, 3200, generator=g).cuda(), ints(free[:66]).view(3, 22))


def step(k_codes, v_codes, k_scale, v_scale, table, held, q, k, v, weights, new_table):
    cache = KVCache(k_codes, v_codes, k_scale, v_scale)
    ring_swa.kv_cache_append(cache, k, v * 1, table, held)
    lens = held + 1
    out, lse = ring_swa.kv_cache_attn(q, cache, table, lens, 900, num_sink_tokens=2, return_lse=True)
    ring_swa.kv_cache_weights(q, cache, table, lens, lse, weights, 900, num_sink_tokens=2)
    return out, lse, *ring_swa.kv_cache_evict(cache, weights, table, lens, new_table, 700, num_sink_tokens=2, num_recent=30)


def check(run):
    for seed in (0, 1):
        mine, want = inputs(seed), inputs(seed)
        got = (*run(*mine), *mine)
        for x, y in zip(got, (*step(*want), *want)):
            assert torch.equal(x.view(torch.uint8) if x.element_size() == 1 else x,
                               y.view(torch.uint8) if y.element_size() == 1 else y)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled(backend):
    torch._dynamo.reset()
    check(torch.compile(step, backend=backend))


def test_traced():
    check(torch.jit.trace(step, inputs(2), check_trace=False))


def test_traced_by_dispatch():
    from torch.fx.experimental.proxy_tensor import make_fx

    check(make_fx(step)(*inputs(2)))
