"""The cache's calls have no derivative: every floating-point input that wants one is refused, in both directions."""
import pytest
import torch
from torch.autograd import forward_ad

import ring_swa
from ring_swa import KVCache, _lib


@pytest.fixture(autouse=True)
def on_cpu(monkeypatch):
    """The checks ahead of the launch, with tensors that live on the CPU; the launch itself does nothing."""
    monkeypatch.setattr(_lib, "require_device", lambda *t: t[0].device)
    monkeypatch.setattr(_lib, "launch", lambda *_: None)


def inputs():
    cache = KVCache.empty(12, 2, 64, 16)
    for t in cache[:2]:
        t.view(torch.uint8).zero_()
    rows = torch.randn(2, 1, 8, 64).bfloat16()
    return dict(cache._asdict(), q=rows[:, :, :4], new_k=rows[:, :, 4:6], new_v=rows[:, :, 6:], lse=torch.rand(2, 4, 1),
                weights=torch.rand(2, 2, 48))


CALLS = {
    "append": (("new_k", "new_v"), lambda c, table, lens, x: ring_swa.kv_cache_append(c, x["new_k"], x["new_v"], table, lens)),
    "attn": (("q",), lambda c, table, lens, x: ring_swa.kv_cache_attn(x["q"], c, table, lens)),
    "weights": (("q", "lse", "weights"),
                lambda c, table, lens, x: ring_swa.kv_cache_weights(x["q"], c, table, lens, x["lse"], x["weights"])),
    "evict": (("weights",), lambda c, table, lens, x: ring_swa.kv_cache_evict(c, x["weights"], table, lens, table + 6, 20)),
}
INPUTS = [(call, name) for call, (names, _) in CALLS.items() for name in names + KVCache._fields]


def run(call, x):
    table, lens = torch.arange(6, dtype=torch.int32).view(2, 3), torch.tensor([9, 30], dtype=torch.int32)
    return CALLS[call][1](KVCache(*(x[f] for f in KVCache._fields)), table, lens, x)


@pytest.mark.parametrize("call,name", INPUTS)
def test_tensors_that_need_a_gradient(call, name):
    x = inputs()
    run(call, x)
    x[name] = x[name].detach().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        run(call, x)
    with torch.no_grad():
        run(call, x)


@pytest.mark.parametrize("call,name", [i for i in INPUTS if i[1] not in KVCache._fields])
def test_tensors_with_a_tangent(call, name):
    x = inputs()
    with forward_ad.dual_level():
        run(call, x)
        x[name] = forward_ad.make_dual(x[name].detach(), torch.ones_like(x[name]))
        with pytest.raises(RuntimeError, match="no forward derivative"):
            run(call, x)


def test_transforms():
    def attn(q):
        return run("attn", dict(inputs(), q=q)).float().sum()

    q = inputs()["q"].detach()
    with pytest.raises(RuntimeError, match="no backward"):
        torch.func.grad(attn)(q)
    with pytest.raises(RuntimeError, match="no forward derivative"):
        torch.func.jvp(attn, (q,), (torch.ones_like(q),))
    with pytest.raises(RuntimeError):
        torch.func.jacrev(attn)(q)
