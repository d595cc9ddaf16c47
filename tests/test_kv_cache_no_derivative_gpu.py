"""Inputs of the cache's calls that need a gradient, on the device, where the native module sees them first."""
import pytest
import torch

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
