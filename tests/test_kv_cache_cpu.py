"""What the cache's calls refuse, and their sizes, without a GPU."""
import ctypes
import math

import pytest
import torch

import ring_swa
from oracle import kv_cache_oracle as O
from ring_swa import KVCache, _lib
from ring_swa.ops import kv_cache as K


def test_struct_layout():
    assert _lib.lib().rswa_sizeof_cache_params() == ctypes.sizeof(_lib.CacheParams)


def test_public_names():
    for name in ("KVCache", "kv_cache_append", "kv_cache_attn", "kv_cache_weights", "kv_cache_evict"):
        assert getattr(ring_swa, name) is getattr(ring_swa.ops, name)
        assert name in ring_swa.__all__ and name in ring_swa.ops.__all__


def args(page=64, heads=2, dim=64, batch=2, width=3):
    cache = KVCache.empty(8, heads, dim, page)
    table = torch.zeros(batch, width, dtype=torch.int32)
    lens = torch.ones(batch, dtype=torch.int32)
    return cache, table, lens, torch.zeros(batch, 1, 4, dim, dtype=torch.bfloat16)


def test_an_empty_cache():
    cache = KVCache.empty(3, 2, 128, 32)
    assert cache.page_size == 32 and cache.k.shape == (3, 2, 32, 128) and cache.v.shape == (3, 2, 2, 128, 16)
    assert cache.k_scale.dtype == torch.float8_e8m0fnu
    with pytest.raises(AssertionError):
        KVCache.empty(3, 2, 128, 48)


def test_cpu_tensors_are_refused():
    cache, table, lens, q = args()
    with pytest.raises(RuntimeError, match="GPU"):
        ring_swa.kv_cache_attn(q, cache, table, lens)
    with pytest.raises(RuntimeError, match="GPU"):
        ring_swa.kv_cache_append(cache, q[:, :, :2], q[:, :, :2], table, lens)
    with pytest.raises(RuntimeError, match="GPU"):
        ring_swa.kv_cache_evict(cache, torch.zeros(2, 2, 9), table, lens, table.clone(), 4)


def test_tensors_that_need_a_gradient_are_refused():
    cache, table, lens, q = args()
    q.requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        ring_swa.kv_cache_attn(q, cache, table, lens)
    with pytest.raises(RuntimeError, match="no backward"):
        ring_swa.kv_cache_append(cache, q[:, :, :2], q[:, :, :2], table, lens)


@pytest.fixture
def on_cpu(monkeypatch):
    """The checks ahead of the launch, with tensors that live on the CPU; the launch itself is a failure."""
    monkeypatch.setattr(_lib, "require_device", lambda *t: t[0].device)

    def launch(*_):
        raise AssertionError("launched")

    monkeypatch.setattr(_lib, "launch", launch)


def refuses(fn, *a, **kw):
    with pytest.raises((AssertionError, NotImplementedError, ValueError)) as e:
        fn(*a, **kw)
    assert "launched" not in str(e.value), "accepted"


def test_shapes_and_types_are_checked(on_cpu):
    cache, table, lens, q = args()
    attn = ring_swa.kv_cache_attn
    refuses(attn, q[0], cache, table, lens)                                   # packed without cu_seqlens
    refuses(attn, q[:1], cache, table, lens)                                  # batch
    refuses(attn, q[:, :, :3], cache, table, lens)                            # heads
    refuses(attn, q[..., :32], cache, table, lens)                            # head_dim
    refuses(attn, q, cache, table.long(), lens)
    refuses(attn, q, cache, table[0], lens)
    refuses(attn, q, cache, table.t().contiguous().t(), lens)
    refuses(attn, q, cache, table, lens.long())
    refuses(attn, q, cache, table, lens[:1])
    refuses(attn, q, cache, table, lens, num_sink_tokens=-1)
    refuses(attn, q.int(), cache, table, lens)
    refuses(attn, q[:, 0], cache, table, lens, -1, torch.zeros(2, dtype=torch.int32))
    refuses(attn, q[:, 0], cache, table, lens, -1, torch.zeros(3, dtype=torch.int64))
    refuses(attn, q, cache._replace(k=cache.k.view(torch.uint8)), table, lens)
    refuses(attn, q, cache._replace(k_scale=cache.k_scale.view(torch.uint8)), table, lens)
    refuses(attn, q, cache._replace(v=cache.v[:, :, :2]), table, lens)
    refuses(attn, q, cache._replace(v_scale=cache.v_scale[:, :1]), table, lens)
    refuses(attn, q, cache._replace(k=cache.k.transpose(2, 3)), table, lens)
    k = q[:, :, :2]
    append = ring_swa.kv_cache_append
    refuses(append, cache, k, k[:, :, :1], table, lens)
    refuses(append, cache, q, q, table, lens)
    refuses(append, cache, k, k.half(), table, lens)
    weights = ring_swa.kv_cache_weights
    lse, w = torch.zeros(2, 4, 1), torch.zeros(2, 2, 9)
    refuses(weights, q, cache, table, lens, lse[:, :3], w)
    refuses(weights, q, cache, table, lens, lse.double(), w)
    refuses(weights, q, cache, table, lens, lse, w[:1])
    refuses(weights, q, cache, table, lens, lse, w.double())
    refuses(weights, q, cache, table, lens, lse, w.transpose(1, 2).contiguous().transpose(1, 2))
    evict = ring_swa.kv_cache_evict
    refuses(evict, cache, w, table, lens, table.clone(), 0)
    refuses(evict, cache, w, table, lens, table.clone(), 4, num_sink_tokens=3, num_recent=2)
    refuses(evict, cache, w, table, lens, table.clone()[:1], 4)
    refuses(evict, cache, w, table, lens, table.clone().long(), 4)
    refuses(evict, cache, w, table, lens, table.clone(), 4, num_recent=-1)


def params(fill):
    cache, table, lens, q = args(dim=128)
    p = _lib.CacheParams(dtype=0, head_dim=128, batch=2, heads_q=4, heads_kv=2, page_size=64, num_pages=8, max_pages=3,
                         seqlen_q=1, softmax_scale=0.1, window_left=-1)
    for name in ("k", "v", "k_scale", "v_scale", "page_table", "seqlens", "q", "out", "new_k", "new_v", "lse", "weights",
                 "new_seqlens", "new_weights", "kept"):
        setattr(p, name, 4096)
    p.new_page_table, p.new_max_pages, p.budget, p.weights_len = 8192, 1, 64, 64
    p.workspace, p.workspace_bytes = 4096, 1 << 40
    for name, value in fill.items():
        if isinstance(value, tuple):
            getattr(p, name)[:] = value
        else:
            setattr(p, name, value)
    return p


def test_running_sums_that_overlap_are_refused(on_cpu):
    cache, table, lens, q = args()
    lse = torch.zeros(q.shape[0], q.shape[2], q.shape[1])
    batch, heads = table.shape[0], cache.k.shape[1]
    room = torch.zeros(10000)
    for strides, fine in (((20 * heads, 20, 1), True), ((20, 20 * batch, 1), True), ((30, 20, 1), False),
                          ((20, 20, 1), False), ((0, 20, 1), False), ((20 * heads, 19, 1), False)):
        w = room.as_strided((batch, heads, 20), strides)
        with pytest.raises(AssertionError, match="launched" if fine else "overlap"):
            ring_swa.kv_cache_weights(q, cache, table, lens, lse, w)


@pytest.mark.parametrize("call", ["append", "attn", "weights", "evict"])
@pytest.mark.parametrize("fill,status", [
    ({"dtype": 2}, -2), ({"head_dim": 96}, -2), ({"page_size": 48}, -2), ({"page_size": 8}, -2), ({"page_size": 512}, -2),
    ({"heads_kv": 0}, -1), ({"batch": -1}, -1), ({"heads_q": 5}, -1), ({"max_pages": 1 << 22}, -2), ({"k": None}, -1),
    ({"v_scale": None}, -1), ({"seqlens": None}, -1), ({"page_table": None}, -1), ({"k": 4100}, -2),
    ({"v_stride": (8, 16)}, -2), ({"num_pages": 0}, -1)])
def test_every_call_refuses(call, fill, status):
    L = _lib.lib()
    assert getattr(L, "rswa_cache_" + call)(params(fill), None) == status
    assert L.rswa_last_error().decode().startswith("cache_" + call)


@pytest.mark.parametrize("call,fill,status", [
    ("attn", {"softmax_scale": 0.0}, -1), ("attn", {"softmax_scale": math.inf}, -1),
    ("attn", {"softmax_scale": math.nan}, -1), ("attn", {"num_sink": -1}, -1), ("attn", {"q": None}, -1),
    ("attn", {"q": 4104}, -2), ("attn", {"q_stride": (4, 8, 8)}, -2), ("attn", {"out": None}, -1),
    ("attn", {"out_stride": (8, 8, 4)}, -2), ("attn", {"workspace": None, "max_pages": 1000}, -1),
    ("attn", {"workspace_bytes": 16, "max_pages": 1000}, -1), ("attn", {"workspace": 4104, "max_pages": 1000}, -1),
    ("attn", {"seqlen_q": 1 << 28}, -2),
    ("append", {"new_k": None}, -1), ("append", {"new_v": 4104}, -2), ("append", {"new_k_stride": (8, 4, 8)}, -2),
    ("weights", {"lse": None}, -1), ("weights", {"weights": None}, -1), ("weights", {"weights_len": -1}, -1),
    ("evict", {"budget": 0}, -1), ("evict", {"num_sink": 60, "num_recent": 5}, -1), ("evict", {"num_recent": -1}, -1),
    ("evict", {"kept": None}, -1), ("evict", {"new_page_table": 4096}, -1), ("evict", {"new_max_pages": 0}, -1),
    ("evict", {"budget": 65}, -1), ("evict", {"new_weights": None}, -1)])
def test_single_calls_refuse(call, fill, status):
    assert getattr(_lib.lib(), "rswa_cache_" + call)(params(fill), None) == status


def test_nothing_to_do_is_no_error():
    """Calls without rows or sequences launch nothing, whatever else is missing."""
    L = _lib.lib()
    for call in ("append", "attn", "weights"):
        assert getattr(L, "rswa_cache_" + call)(params({"seqlen_q": 0, "q": None, "new_k": None}), None) == 0
    for call in ("append", "attn", "weights", "evict"):
        assert getattr(L, "rswa_cache_" + call)(params({"batch": 0}), None) == 0


def test_running_sums_of_no_tokens_need_no_memory():
    assert _lib.lib().rswa_cache_weights(params({"weights_len": 0, "weights": None}), None) == 0


def test_workspace_is_bounded_and_grows_with_what_is_shared():
    L = _lib.lib()
    size = lambda **kw: int(L.rswa_cache_attn_workspace_bytes(params(kw)))  # noqa: E731
    assert size(max_pages=4) == 0                       # one chunk holds all a sequence can have
    assert 0 < size(max_pages=64) <= size(max_pages=4096)
    assert size(max_pages=1 << 20, seqlen_q=1 << 16) < 1 << 28


def test_the_restatement_rounds_as_the_type_does():
    """Codes of the restatement against the definition of e4m3: nearest value, ties to the even code."""
    codes = torch.arange(0x7F, dtype=torch.uint8)
    values = O.decode(codes)
    assert values[1].item() == 2.0 ** -9 and values[-1].item() == 448.0 and values[8].item() == 2.0 ** -6
    middle = (values[1:] + values[:-1]) / 2
    even = codes[:-1] + codes[:-1] % 2
    assert torch.equal(O.encode(middle), even) and torch.equal(O.encode(values), codes)
    assert torch.equal(O.encode(middle * (1 + 1e-6)), codes[1:]) and torch.equal(O.encode(middle * (1 - 1e-6)), codes[:-1])
    assert O.scale_byte(0.0) == 7 and O.scale_byte(448.0) == 127 and O.scale_byte(448.1) == 128
    assert O.scale_byte(3.4e38) == 247
