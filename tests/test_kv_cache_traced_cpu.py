"""The cache's calls in compiled and traced programs, without a GPU: a compiled program makes them between its graphs,
and in a traced one each is an operation, whose run makes the launch.  The launch itself is a stub that writes what can
be told apart."""
import ctypes

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import ring_swa
from ring_swa import KVCache, _lib

CALLS = ["append", "attn", "attn_lse", "weights", "evict"]


@pytest.fixture
def launches(monkeypatch):
    """Names of the entry points launched; the stub writes to each call's results and to what it changes in place."""
    names = []

    def launch(_, entry, p):
        names.append(entry.__name__)
        tokens = p.batch * p.seqlen_q * p.heads_q
        if entry.__name__ == "rswa_cache_append":
            ctypes.memset(p.k, 0x38, p.page_size * p.head_dim)
            ctypes.memset(p.v_scale, 0x7F, 1)
        elif entry.__name__ == "rswa_cache_attn":
            ctypes.memmove(p.out, p.q, tokens * p.head_dim * 2)
            if p.lse:
                ctypes.memset(p.lse, 0x40, tokens * 4)
        elif entry.__name__ == "rswa_cache_weights":
            ctypes.memset(p.weights, 0x3F, 4 * p.weights_len)
        else:
            ctypes.memset(p.k_scale, 0x70, 1)
            ctypes.memset(p.new_seqlens, 0, 4 * p.batch)
            ctypes.memset(p.new_weights, 0, 4 * p.batch * p.heads_kv * p.weights_len)
            ctypes.memset(p.kept, 0xFF, 4 * p.batch * p.heads_kv * p.budget)

    monkeypatch.setattr(_lib, "require_device", lambda *t: t[0].device)
    monkeypatch.setattr(_lib, "launch", launch)
    return names


def inputs():
    cache = KVCache.empty(8, 2, 64, 16)
    for t in cache[:2]:
        t.view(torch.uint8).zero_()
    g = torch.Generator().manual_seed(1)
    return (*cache, torch.arange(6, dtype=torch.int32).view(2, 3), torch.tensor([9, 30], dtype=torch.int32),
            torch.randn(2, 1, 4, 64, generator=g).bfloat16(), torch.rand(2, 4, 1, generator=g),
            torch.rand(2, 2, 48, generator=g))


def program(call):
    def run(k, v, k_scale, v_scale, table, lens, q, lse, w):
        cache = KVCache(k, v, k_scale, v_scale)
        if call == "append":
            ring_swa.kv_cache_append(cache, q[:, :, :2], q[:, :, 2:], table, lens)
            return lens + 1
        if call == "attn":
            return ring_swa.kv_cache_attn(q, cache, table, lens, 9, num_sink_tokens=2) + 1
        if call == "attn_lse":
            return ring_swa.kv_cache_attn(q, cache, table, lens, softmax_scale=0.5, return_lse=True)
        if call == "weights":
            ring_swa.kv_cache_weights(q, cache, table, lens, lse, w)
            return w * 2
        return ring_swa.kv_cache_evict(cache, w, table, lens, table + 4, 20, num_sink_tokens=1, num_recent=4)

    return run


def same(got, want):
    got, want = ([x] if torch.is_tensor(x) else list(x) for x in (got, want))
    assert len(got) == len(want)
    for x, y in zip(got, want):
        assert x.dtype == y.dtype and torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


def check(call, run, names):
    """``run`` against the plain program on inputs of its own, results and what is changed in place."""
    mine, want = inputs(), inputs()
    names.clear()
    results = run(*mine)
    assert names == ["rswa_cache_" + call.split("_")[0]]
    same(results, program(call)(*want))
    same(mine, want)


@pytest.mark.parametrize("backend", ["eager", "aot_eager", "inductor"])
@pytest.mark.parametrize("call", CALLS)
def test_compiled(call, backend, launches):
    torch._dynamo.reset()
    run = torch.compile(program(call), backend=backend)
    for _ in range(2):
        check(call, run, launches)


@pytest.mark.parametrize("call", CALLS)
def test_traced(call, launches):
    run = torch.jit.trace(program(call), inputs(), check_trace=False)
    assert "ring_swa::cache_" + call.split("_")[0] in str(run.graph)
    check(call, run, launches)


@pytest.mark.parametrize("mode", ["real", "fake"])
@pytest.mark.parametrize("call", CALLS)
def test_traced_by_dispatch(call, mode, launches):
    run = make_fx(program(call), tracing_mode=mode)(*inputs())
    check(call, run, launches)


def test_a_mode_sees_the_call(launches):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Mode(TorchDispatchMode):
        seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            Mode.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    with Mode():
        program("attn")(*inputs())
    assert "ring_swa.cache_attn.default" in Mode.seen and launches == ["rswa_cache_attn"]


def test_a_program_of_one_graph_is_refused(launches):
    torch._dynamo.reset()
    with pytest.raises(torch._dynamo.exc.Unsupported, match="_uncompiled"):
        torch.compile(program("append"), backend="eager", fullgraph=True)(*inputs())
    assert launches == []


def test_refusals_inside_a_compiled_program(launches):
    torch._dynamo.reset()
    args = list(inputs())
    args[4] = args[4].long()
    with pytest.raises(AssertionError, match="int32"):
        torch.compile(program("attn"), backend="eager")(*args)
    assert launches == []
