"""Rows that a read of the cache writes may not share an element, with one another or with the other tensor's: told from
sizes, strides and addresses, and refused ahead of the launch."""
import random

import numpy as np
import pytest
import torch

from ring_swa import _lib
from test_drafts_cpu import inputs, on_cpu, params, refuses  # noqa: F401  (on_cpu is a fixture)

BASE = 1 << 20


def asked(counts, k_strides, v_strides, apart, dim, packed):
    """`apart`: elements from k to v."""
    p = _lib.CacheParams(head_dim=dim, heads_kv=counts[2], new_k=BASE, new_v=BASE + 2 * apart)
    if packed:
        p.batch, p.total_q, p.cu_seqlens_q = 3, counts[1], 4096
    else:
        p.batch, p.seqlen_q = counts[:2]
    p.new_k_stride[:], p.new_v_stride[:] = k_strides, v_strides
    return bool(_lib.lib().rswa_cache_read_rows_meet(p))


def places(counts, strides, dim, at=0):
    a, b, c = (np.arange(n)[:, None] * s for n, s in zip(counts, strides))
    return (at + a[:, None, None] + b[None, :, None] + c[None, None] + np.arange(dim)).ravel()


def really(counts, k_strides, v_strides, apart, dim):
    both = np.concatenate((places(counts, k_strides, dim), places(counts, v_strides, dim, apart)))
    return len(np.unique(both)) < len(both)


@pytest.mark.parametrize("packed", [False, True])
def test_random_layouts(packed):
    rng = random.Random(packed)
    told = {True: 0, False: 0}
    for _ in range(6000):
        counts = [1 if packed else rng.randint(1, 4), rng.randint(1, 6), rng.randint(1, 4)]
        dim = rng.choice((1, 2, 4, 8))

        def strides():
            if rng.random() < 0.4:
                return [rng.randrange(0, 200) for _ in range(3)]
            # dimensions inside one another, in any order, with room between them or, now and then, too little
            order, st, step = rng.sample(range(3), 3), [0] * 3, dim
            for d in order:
                step += rng.choice((0, 0, 0, 1, dim, 3 * dim, -1))
                st[d] = max(step, 0)
                step = st[d] * counts[d]
            return st

        ks = strides()
        vs = ks if rng.random() < 0.5 else strides()
        span = sum((n - 1) * s for n, s in zip(counts, ks)) + dim
        apart = rng.choice((rng.randint(-span, span), span, dim, -dim, rng.choice(ks)))
        want = really(counts, ks, vs, apart, dim)
        told[want] += 1
        assert asked(counts, ks, vs, apart, dim, packed) == want, (counts, ks, vs, apart, dim)
    assert min(told.values()) > 1000


def layouts():
    """Tensors that programs have: (k, v, whether they meet)."""
    b, s, h, d = 3, 40, 4, 64
    kv = torch.empty(b, s, 2, h, d, dtype=torch.bfloat16)
    yield "between rows", kv[:, :, 0], kv[:, :, 1], False
    kv = torch.empty(b, s, h, 2, d, dtype=torch.bfloat16)
    yield "between heads", kv[..., 0, :], kv[..., 1, :], False
    kv = torch.empty(b, s, h, 3 * d, dtype=torch.bfloat16)
    yield "parts of rows", kv[..., d:2 * d], kv[..., 2 * d:], False
    yield "overlapping parts of rows", kv[..., d:2 * d], kv[..., d + 8:2 * d + 8], True
    kv = torch.empty(2, b, s, h, d, dtype=torch.bfloat16)
    yield "one after the other", kv[0], kv[1], False
    yield "one tensor", kv[0], kv[0], True
    yield "the same from the second row on", kv[0, :, 1:], kv[0, :, :-1], True
    kv = torch.empty(b, 2, s * h * d, dtype=torch.bfloat16)
    yield "two orders of a sequence's rows", kv[:, 0].view(b, s, h, d), kv[:, 1].view(b, h, s, d).transpose(1, 2), False
    yield "two orders of the same", kv[:, 0].view(b, s, h, d), kv[:, 0].view(b, h, s, d).transpose(1, 2), True
    t = torch.empty(b, h, s, d, dtype=torch.bfloat16).transpose(1, 2)
    yield "heads first", t, torch.empty_like(t), False
    t = torch.empty(s, b, h, d, dtype=torch.bfloat16).transpose(0, 1)
    yield "rows first, every second", t[:, ::2], t[:, 1::2], False
    t = torch.empty(b, s + 9, h, d, dtype=torch.bfloat16)
    other = torch.empty(b, s, h, d, dtype=torch.bfloat16)
    yield "windows of a row each", t.as_strided((b, s, h, d), (9 * h * d, h * d, d, 1)), other, True
    yield "rows of less than heads * dim", t.as_strided((1, s, h, d), (0, (h - 1) * d, d, 1)), other[:1], True
    yield "rows that begin inside one another", other[:1], t.as_strided((1, s, h, d), (0, h * d, 8, 1)), True
    yield "one sequence for all", t[:1, :s].expand(b, s, h, d), other, True
    yield "one row for all", other, t[:, :1].expand(b, s, h, d), True
    yield "one head for all", t[:, :s, :1].expand(b, s, h, d), other, True
    yield "a stride of one element", t[:1, :1].as_strided((1, 1, h, d), (0, 0, d, 1)), other[:1, :1], False


LAYOUTS = list(layouts())


@pytest.mark.parametrize("name,k,v,meet", LAYOUTS, ids=[x[0].replace(" ", "_") for x in LAYOUTS])
def test_layouts_in_use(name, k, v, meet, on_cpu):
    table = torch.arange(k.shape[0], dtype=torch.int32)[:, None].contiguous()
    changed = dict(cache=type(inputs()["cache"]).empty(8, k.shape[2], 64, 64), k=k, v=v, table=table,
                   lens=torch.zeros(k.shape[0], dtype=torch.int32))
    refuses("cache_read", not meet, **changed)
    if k.shape[0] == 1:  # packed
        changed.update(k=k[0], v=v[0])
        refuses("cache_read", not meet, {"cu_seqlens": torch.tensor([0, 1], dtype=torch.int32)}, **changed)


def test_the_library_refuses():
    """(its callers from C)"""
    L = _lib.lib()
    p = params("cache_read", {"new_k_stride": (3 * 256, 256, 128), "new_v_stride": (3 * 256, 256, 128)})  # one tensor
    assert L.rswa_cache_read(p, None) == -1 and b"overlap" in L.rswa_last_error()
    p = params("cache_read", {"new_k_stride": (3 * 256, 256, 128), "new_v_stride": (3 * 256, 256, 128),
                              "new_v": 4096 + 2 * 6 * 256 - 16})
    assert L.rswa_cache_read(p, None) == -1 and b"overlap" in L.rswa_last_error()


def test_strides_and_counts_of_any_size():
    most = (1 << 63) - 1
    assert not asked((2, 2, 2), (most - 7, 1 << 40, 64), (most - 7, 1 << 40, 64), 1 << 50, 64, False)
    assert asked((2, 2, 2), (-(1 << 63), 1 << 40, 64), (0, 64, 128), 1 << 50, 64, False)  # (heads of v on its rows)
    assert asked((1 << 30, 1 << 30, 1 << 16), (0, 0, 0), (0, 0, 0), 1 << 50, 128, False)
    assert not asked((0, 5, 5), (0, 0, 0), (0, 0, 0), 0, 128, False)
    assert asked((4, 1 << 28, 8), (1 << 38, 1024, 128), (1 << 38, 1024, 128), 1 << 37, 128, False)  # (row 2^27 of k)
    assert not asked((4, 1 << 28, 8), (1 << 39, 1024, 128), (1 << 39, 1024, 128), 1 << 38, 128, False)
    # negative strides, which a caller from C may have: the last row first
    assert not asked((2, 3, 2), (600, -200, 100), (600, -200, 100), 2000, 100, False)
    assert asked((2, 3, 2), (600, -200, 100), (600, -200, 100), -100, 100, False)
