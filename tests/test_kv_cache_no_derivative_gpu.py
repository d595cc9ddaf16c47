"""Inputs of the cache's calls that want a derivative, on the device, where the native module sees them first."""
import pytest
import torch
from torch.autograd import forward_ad

from ring_swa import KVCache
from test_kv_cache_no_derivative_cpu import CALLS, INPUTS, inputs

pytestmark = pytest.mark.gpu


def run(call, x):
    table = torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3)
    return CALLS[call][1](KVCache(*(x[f] for f in KVCache._fields)), table,
                          torch.tensor([9, 30], dtype=torch.int32, device="cuda"), x)


def on_device():
    return {name: t.cuda() for name, t in inputs().items()}


@pytest.mark.parametrize("call,name", INPUTS)
def test_tensors_that_need_a_gradient(call, name):
    x = on_device()
    run(call, x)
    x[name] = x[name].detach().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        run(call, x)
    with torch.no_grad():
        run(call, x)


@pytest.mark.parametrize("call,name", [i for i in INPUTS if i[1] not in KVCache._fields])
def test_tensors_with_a_tangent(call, name):
    x = on_device()
    with forward_ad.dual_level():
        run(call, x)
        x[name] = forward_ad.make_dual(x[name].detach(), torch.ones_like(x[name]))
        with pytest.raises(RuntimeError, match="no forward derivative"):
            run(call, x)
