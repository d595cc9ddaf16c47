"""Attention of many rows over the 8-bit paged cache (blocks whose waves have rows of their own), the key weights of
as many rows, and the Python route of the cache's calls beside the native one.  Bounds as in test_kv_cache_gpu."""
import math

import pytest
import torch

from oracle import kv_cache_oracle as O
from test_kv_cache_gpu import DTYPES, check_attn, ints, make, randn, score_error

pytestmark = pytest.mark.gpu

# 32768 (row, q head) pairs or more, above 64 rows per kv head: lens, new rows (a list: packed), q heads, kv heads, dim,
# page, window, sinks, dtype
MANY = [
    ([1500, 300, 777, 300], 300, 32, 8, 128, 64, -1, 0, "bf16"),
    ([1500, 300, 777, 2], 300, 32, 8, 64, 16, 100, 4, "fp16"),     # 300 rows of 2 tokens
    ([2111], 1100, 32, 32, 128, 32, 500, 70, "fp16"),              # as many kv heads as q heads, sinks over two tiles
    ([900, 0, 1025, 64, 3], [700, 0, 250, 64, 40], 32, 4, 128, 256, -1, 0, "bf16"),
    ([900, 0, 1025, 64, 3], [700, 0, 250, 64, 1], 48, 2, 64, 128, 333, 1, "bf16"),
    ([66000], 1030, 32, 8, 64, 64, -1, 0, "bf16"),                 # row tiles of several chunks
    ([5000], 1100, 33, 1, 128, 16, 0, 0, "bf16"),                  # a window of the token alone, group of 33
]


def call(case, seed=0):
    lens, new, hq, hk, dim, size, window, sinks, dtype = MANY[case]
    cache, table, seqlens, _ = make(lens, hk, dim, size, 500 + case, max_pages=-(-max(lens) // size) + case % 2)
    g = torch.Generator().manual_seed(600 + case + seed)
    cu = None
    if isinstance(new, list):
        cu = ints([sum(new[:i]) for i in range(len(new) + 1)])
        q = randn(g, DTYPES[dtype], sum(new), hq, dim)
    else:
        q = randn(g, DTYPES[dtype], len(lens), new, hq, dim)
    return q, cache, table, seqlens, window, cu, sinks


@pytest.mark.parametrize("case", range(len(MANY)))
def test_many_rows(case):
    from ring_swa import kv_cache_attn

    q, cache, table, seqlens, window, cu, sinks = call(case)
    out, lse = kv_cache_attn(q, cache, table, seqlens, window, cu, num_sink_tokens=sinks, return_lse=True)
    check_attn(q, cache, table, seqlens, out, lse, window, cu, None, sinks)
    assert torch.equal(kv_cache_attn(q, cache, table, seqlens, window, cu, num_sink_tokens=sinks), out)


@pytest.mark.parametrize("size", [16, 128])
def test_many_rows_with_pages_missing(size):
    from ring_swa import kv_cache_attn

    cache, table, seqlens, _ = make([1000, 900], 8, 128, size, 700 + size)
    table[0, :1] = -1
    table[0, 3] = cache.k.shape[0]
    table[1, 1] = -7
    q = randn(torch.Generator().manual_seed(20), torch.bfloat16, 2, 520, 32, 128)
    out, lse = kv_cache_attn(q, cache, table, seqlens, return_lse=True)
    check_attn(q, cache, table, seqlens, out, lse)


@pytest.mark.parametrize("case", range(len(MANY)))
def test_weights_of_many_rows(case):
    from ring_swa import kv_cache_attn, kv_cache_weights

    q, cache, table, seqlens, window, cu, sinks = call(case, 50)
    _, lse = kv_cache_attn(q, cache, table, seqlens, window, cu, num_sink_tokens=sinks, return_lse=True)
    running = torch.rand(len(seqlens), cache.k.shape[1], int(seqlens.max()), generator=torch.Generator().manual_seed(1)).cuda()
    want, off = O.weights(q, cache, table, seqlens, lse, running, window, cu, None, sinks)
    got = running.clone()
    kv_cache_weights(q, cache, table, seqlens, lse, got, window, cu, num_sink_tokens=sinks)
    # (a sum of up to 48 x 1100 terms in 32 bits, lane by lane and then 16 lanes: 2^-24 for each of some 2^8 additions)
    bound = 2 * score_error(off, q.shape[-1]) + 2.0 ** -16 * (want - running.double()) + 2.0 ** -23 * want + 2.0 ** -40
    diff = (got.double() - want).abs()
    assert bool((diff <= bound).all()), f"off by up to {(diff / bound).max().item():.2f} of the bound"


def test_cu_seqlens_that_overlap_or_leave_the_tensor():
    """Any results, but nothing read or written that is not the call's: pages of no sequence stay as they are, and the
    sums behind a sequence's tokens."""
    import ring_swa

    cache, table, lens, free = make([500, 700], 8, 64, 16, 815, spare=5, max_pages=120)
    q = randn(torch.Generator().manual_seed(36), torch.bfloat16, 1100, 32, 64)
    k, v = (randn(torch.Generator().manual_seed(37 + i), torch.bfloat16, 1100, 8, 64) for i in range(2))
    kept = [t.view(torch.uint8)[free].clone() for t in cache]
    for wild in ([0, 1100, 0], [-5, 600, 10 ** 9], [800, 200, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31, 5]):
        cu = ints(wild)
        out, lse = ring_swa.kv_cache_attn(q, cache, table, lens, -1, cu, return_lse=True)
        assert out.shape == q.shape and lse.shape == (32, 1100)
        w = torch.zeros(2, 8, 900, device="cuda")
        ring_swa.kv_cache_weights(q, cache, table, lens, lse, w, -1, cu)
        assert bool((w[0, :, 500:] == 0).all()) and bool((w[1, :, 700:] == 0).all())
        ring_swa.kv_cache_append(cache, k, v, table, lens, cu)
        for t, was in zip(cache, kept):
            assert torch.equal(t.view(torch.uint8)[free], was)


def test_packs_that_begin_behind_the_first_row():
    """Rows ahead of cu_seqlens[0] are no sequence's: neither written to the cache nor answered."""
    import ring_swa

    for cu_list in ([40, 43, 90], [200, 200, 263], [17, 80, 80]):
        cache, table, lens, _ = make([500, 70], 2, 64, 16, 816, max_pages=40, wild=False)
        g = torch.Generator().manual_seed(39)
        k, v = (randn(g, torch.bfloat16, 300, 2, 64) for _ in range(2))
        q = randn(g, torch.bfloat16, 300, 8, 64)
        cu = ints(cu_list)
        held = lens - cu.diff()
        want = O.append(cache, k, v, table, held, cu)
        ring_swa.kv_cache_append(cache, k, v, table, held, cu)
        assert O.same_bytes(cache, want)
        out, lse = ring_swa.kv_cache_attn(q, cache, table, lens, -1, cu, return_lse=True)
        at = cu_list[0]
        w = torch.zeros(2, 2, 500, device="cuda")
        ring_swa.kv_cache_weights(q, cache, table, lens, lse, w, -1, cu)
        moved = ints([x - at for x in cu_list])  # the same pack from its first row on
        out2, lse2 = ring_swa.kv_cache_attn(q[at:], cache, table, lens, -1, moved, return_lse=True)
        w2 = torch.zeros(2, 2, 500, device="cuda")
        ring_swa.kv_cache_weights(q[at:], cache, table, lens, lse2, w2, -1, moved)
        n = cu_list[-1] - at
        assert torch.equal(out[at:cu_list[-1]], out2[:n]) and torch.equal(lse[:, at:cu_list[-1]], lse2[:, :n])
        assert torch.equal(w, w2)


def test_the_python_route_gives_the_native_one_s_bits(monkeypatch):
    """Every call through the native module, which must take it, and again without the module."""
    import ring_swa
    from ring_swa import _lib

    def run():
        g = torch.Generator().manual_seed(30)
        results = []
        for packed in (False, True):
            cache, table, held, free = make([300, 70, 1], 2, 64, 32, 800, spare=20, max_pages=16, wild=False)
            new = [3, 0, 5] if packed else [4] * 3
            cu = ints([0, 3, 3, 8]) if packed else None
            lead = (8,) if packed else (3, 4)
            q, k, v = (randn(g, torch.float16, *lead, h, 64) for h in (4, 2, 2))
            ring_swa.kv_cache_append(cache, k, v, table, held, cu)
            lens = held + ints(new)
            out = ring_swa.kv_cache_attn(q, cache, table, lens, 50, cu, 0.3, num_sink_tokens=2)
            out2, lse = ring_swa.kv_cache_attn(q, cache, table, lens, -1, cu, return_lse=True)
            w = torch.zeros(3, 2, 400, device="cuda")
            ring_swa.kv_cache_weights(q, cache, table, lens, lse, w, -1, cu)
            n, w2, kept = ring_swa.kv_cache_evict(cache, w, table, lens, ints(free[:12]).view(3, 4), 100,
                                                  num_sink_tokens=1, num_recent=10)
            results += [out, out2, lse, w, n, w2, kept, *(t.view(torch.uint8) for t in cache)]
        return results

    assert _lib.torch_calls() is not None

    def launch(*_):
        raise AssertionError("the native module did not take a call")

    with monkeypatch.context() as m:
        m.setattr(_lib, "launch", launch)
        native = run()
    monkeypatch.setattr(_lib, "_torch_calls", False)
    for x, y in zip(native, run()):
        assert torch.equal(x, y)


def test_running_sums_that_share_memory_are_refused():
    import ring_swa

    cache, table, lens, _ = make([40, 40], 2, 64, 16, 810)
    q = randn(torch.Generator().manual_seed(31), torch.bfloat16, 2, 1, 4, 64)
    _, lse = ring_swa.kv_cache_attn(q, cache, table, lens, return_lse=True)
    w = torch.zeros(1, 2, 40, device="cuda").expand(2, 2, 40)
    with pytest.raises(AssertionError, match="overlap"):
        ring_swa.kv_cache_weights(q, cache, table, lens, lse, w)


def test_running_sums_whose_strides_interleave():
    """Rows of one tensor in either order; as far apart in one direction as in the other they would meet."""
    import ring_swa

    cache, table, lens, _ = make([40, 40], 2, 64, 16, 813)
    q = randn(torch.Generator().manual_seed(34), torch.bfloat16, 2, 1, 4, 64)
    _, lse = ring_swa.kv_cache_attn(q, cache, table, lens, return_lse=True)
    want = torch.zeros(2, 2, 40, device="cuda")
    ring_swa.kv_cache_weights(q, cache, table, lens, lse, want)
    w = torch.zeros(2, 2, 40, device="cuda").transpose(0, 1)
    ring_swa.kv_cache_weights(q, cache, table, lens, lse, w)
    assert torch.equal(w, want)
    with pytest.raises(AssertionError, match="overlap"):
        ring_swa.kv_cache_weights(q, cache, table, lens, lse, torch.zeros(120, device="cuda").as_strided((2, 2, 40), (40, 40, 1)))


def test_running_sums_of_no_tokens():
    """Nothing to add to, and every weight 0 for the eviction: the earliest stay."""
    import ring_swa

    cache, table, lens, _ = make([40, 9], 2, 64, 16, 814)
    q = randn(torch.Generator().manual_seed(35), torch.bfloat16, 2, 1, 4, 64)
    _, lse = ring_swa.kv_cache_attn(q, cache, table, lens, return_lse=True)
    w = torch.zeros(2, 2, 0, device="cuda")
    ring_swa.kv_cache_weights(q, cache, table, lens, lse, w)
    n, w, kept = ring_swa.kv_cache_evict(cache, w, table, lens, ints([[-1], [-1]]), 10, num_recent=2)
    assert n.tolist() == [10, 9] and w.shape == (2, 2, 0)
    assert kept[0, 1].tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 38, 39] and kept[1, 0].tolist() == list(range(9)) + [-1]


def test_calls_under_no_grad_and_with_a_gradient():
    import ring_swa

    cache, table, lens, _ = make([40], 2, 64, 16, 811)
    q = randn(torch.Generator().manual_seed(32), torch.bfloat16, 1, 1, 4, 64)
    want = ring_swa.kv_cache_attn(q, cache, table, lens)
    q.requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        ring_swa.kv_cache_attn(q, cache, table, lens)
    with torch.no_grad():
        assert torch.equal(ring_swa.kv_cache_attn(q, cache, table, lens), want)
    with torch.inference_mode():
        assert torch.equal(ring_swa.kv_cache_attn(q, cache, table, lens), want)


def test_empty_calls():
    import ring_swa

    cache, table, lens, _ = make([40, 7], 2, 64, 16, 812)
    q = torch.empty(2, 0, 4, 64, dtype=torch.bfloat16, device="cuda")
    out, lse = ring_swa.kv_cache_attn(q, cache, table, lens, return_lse=True)
    assert out.shape == q.shape and lse.shape == (2, 4, 0)
    kv = torch.empty(2, 0, 2, 64, dtype=torch.bfloat16, device="cuda")
    ring_swa.kv_cache_append(cache, kv, kv, table, lens)
    none = table[:0]
    out = ring_swa.kv_cache_attn(torch.empty(0, 1, 4, 64, dtype=torch.bfloat16, device="cuda"), cache, none, lens[:0])
    assert out.shape == (0, 1, 4, 64)
    n, w, kept = ring_swa.kv_cache_evict(cache, torch.empty(0, 2, 9, device="cuda"), none, lens[:0], none.clone(), 5)
    assert n.shape == (0,) and w.shape == (0, 2, 9) and kept.shape == (0, 2, 5)
    # a table without columns: no keys at all
    q = randn(torch.Generator().manual_seed(33), torch.bfloat16, 2, 1, 4, 64)
    out, lse = ring_swa.kv_cache_attn(q, cache, table[:, :0], lens, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("kind", ["tail", "equal", "few", "zeros"])
def test_evict_from_long_sequences(kind):
    """Beyond 8192 tokens a table row (larger blocks), 32768 tokens (weights read again in each step), and more weights
    of one digit than the list holds."""
    from ring_swa import kv_cache_evict

    lens, budget, size = [40000, 9001, 33000, 70], 1000, 128
    per = -(-budget // size)
    cache, table, seqlens, free = make(lens, 1, 64, size, 900, spare=per * 4, wild=False)
    new_table = ints(free).view(4, per)
    g = torch.Generator().manual_seed(40)
    w = torch.exp(2 * torch.randn(4, 1, 40000, generator=g))
    if kind == "equal":
        w = torch.full_like(w, 3.5)
    elif kind == "few":
        w = torch.randint(0, 30, w.shape, generator=g).float()
    elif kind == "zeros":
        w = w * (torch.rand(w.shape, generator=g) < 0.01)
    w = w.cuda()
    want, want_n, want_w, want_kept = O.evict(cache, w, table, seqlens, new_table, budget, 4, 64)
    n, new_w, kept = kv_cache_evict(cache, w, table, seqlens, new_table, budget, num_sink_tokens=4, num_recent=64)
    assert torch.equal(n.cpu(), want_n) and torch.equal(kept.cpu(), want_kept) and torch.equal(new_w.cpu(), want_w)
    assert O.same_bytes(cache, want)
