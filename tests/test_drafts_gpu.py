"""Drafted tokens over the 8-bit paged cache against 64-bit restatements: trees, accepted drafts and what is read back
value for value, verification choice for choice, attention within the bounds of test_kv_cache_gpu (nodes are keys whose
values are exact, and whose weights are rounded like the others': the count of roundings is the same; but in fp16 the
nodes' weights are halved for the product with V, so that the smallest are multiples of 2^-37 of the largest where cached
keys' are of 2^-38: off by 2^-38 at most, and 2^-38 * total in the place of 2^-39)."""
import math
import random

import pytest
import torch

from oracle import drafts_oracle as R
from oracle import kv_cache_oracle as O
from test_kv_cache_gpu import DTYPES, HALF, check_attn, ints, make, randn, score_error

pytestmark = pytest.mark.gpu


def some_parents(rng, n, width, holes=0.0):
    """A tree of n nodes; ``holes``: the share of nodes with a parent that is none."""
    parents = []
    for i in range(n):
        p = rng.randrange(max(0, i - width), i) if i else -1
        if i and rng.random() < holes:
            p = rng.choice([-2, i, i + 1, n + 5, -7, 2 ** 31 - 1, -2 ** 31, -1])
        parents.append(p)
    return parents


def tree_tensors(parents, packed):
    """``parents``: lists.  The DraftTree of the restatement."""
    from ring_swa import DraftTree

    most = max(1, max(map(len, parents)))
    parts = [R.tree(p, most) for p in parents]
    rows = [[x for part in parts for x in part[i]] for i in range(3)]
    shape = (len(rows[0]),) if packed else (len(parents), len(parents[0]))
    words = (most + 63) // 64
    return DraftTree(ints(rows[0]).view(shape), ints(rows[1]).view(shape),
                     torch.tensor(rows[2], dtype=torch.int64).view(*shape, words).cuda())


# ---- the tree -----------------------------------------------------------------------------------
@pytest.mark.parametrize("n,width,holes", [(1, 1, 0), (2, 1, 0), (63, 5, 0.1), (64, 64, 0.05), (65, 1, 0), (200, 8, 0.02),
                                           (513, 200, 0.01), (1000, 1, 0), (1024, 1, 0), (1024, 3, 0.002)])
def test_tree(n, width, holes):
    from ring_swa import draft_tree

    rng = random.Random(n + width)
    parents = [some_parents(rng, n, width, holes if b else 0) for b in range(3)] + [[-2] * n]
    got = draft_tree(ints(parents))
    want = tree_tensors(parents, False)
    for g, w in zip(got, want):
        assert g.dtype == w.dtype and torch.equal(g, w)
    # one tree for all, and rows apart
    shared = draft_tree(ints(parents[1:2]).expand(5, n))
    room = torch.full((4, n + 3), 9, dtype=torch.int32, device="cuda")
    room[:, 1:n + 1] = ints(parents)
    apart = draft_tree(room[:, 1:n + 1])
    for g, a, w in zip(shared, apart, want):
        assert all(torch.equal(g[b], w[1]) for b in range(5)) and torch.equal(a, w)


def test_tree_of_packs():
    from ring_swa import draft_tree

    rng = random.Random(5)
    sizes = [0, 5, 1, 300, 0, 64, 7, 0]
    parents = [some_parents(rng, n, 4, 0.05) for n in sizes]
    cu = ints([3 + sum(sizes[:i]) for i in range(len(sizes) + 1)])  # (three rows ahead are nobody's, two behind)
    flat = ints([7, 7, 7] + sum(parents, []) + [7, 7])
    for most in (300, 299, 70, 64, 1):
        got = draft_tree(flat, cu, max_nodes=most)
        assert got.ancestors.shape == (len(flat), (most + 63) // 64)
        for b, p in enumerate(parents):
            want = R.tree(p, most)
            at = slice(int(cu[b]), int(cu[b + 1]))
            assert got.parents[at].tolist() == want[0] and got.depths[at].tolist() == want[1]
            assert got.ancestors[at].tolist() == want[2]
    assert draft_tree(flat[:0], ints([0, 0]), max_nodes=4).depths.shape == (0,)
    assert draft_tree(flat.view(1, -1)[:0]).parents.shape == (0, len(flat))


def test_rows_that_are_no_sequences_are_left():
    """(The rows a pack's tree does not write, through the C ABI, where the results are the caller's.)"""
    from ring_swa import _lib

    flat, cu = ints([-1, -1, 0, -1, -1]), ints([1, 3])
    made = [torch.full(s, 77, dtype=t, device="cuda") for s, t in (((5,), torch.int32), ((5,), torch.int32), ((5, 1), torch.int64))]
    p = _lib.TreeParams(batch=1, max_nodes=8, total=5, cu_seqlens=cu.data_ptr(), parents=flat.data_ptr(),
                        tree_parents=made[0].data_ptr(), depths=made[1].data_ptr(), ancestors=made[2].data_ptr())
    _lib.launch(flat.device, _lib.lib().rswa_draft_tree, p)
    assert [t.flatten().tolist() for t in made] == [[77, -1, 0, 77, 77], [77, 0, 1, 77, 77], [77, 1, 3, 77, 77]]


# ---- attention ----------------------------------------------------------------------------------
TREES = [
    # cached tokens, nodes (a list: packed), width of the trees, q heads, kv heads, dim, page, window, sinks, dtype
    ([0], 1, 1, 4, 4, 128, 64, -1, 0, "bf16"),
    ([0, 1, 63, 64, 65, 300], 5, 3, 8, 2, 128, 64, -1, 0, "bf16"),
    ([0, 1, 63, 64, 65, 300], 16, 1, 8, 2, 64, 16, 5, 4, "fp16"),        # a window shorter than the chain, sinks among the nodes
    ([4001], 32, 16, 32, 8, 128, 64, -1, 0, "bf16"),                      # split over blocks, and joined
    ([2500, 3], 64, 8, 28, 4, 64, 16, 1000, 4, "fp16"),
    ([700, 0, 90], 65, 4, 12, 12, 128, 32, -1, 0, "fp16"),                # a second tile of nodes, of one
    ([130, 1000], 200, 1, 4, 1, 64, 128, 70, 2, "bf16"),                  # chains over four tiles under a window
    ([40, 9], 130, 60, 6, 2, 128, 16, 0, 0, "bf16"),                      # a window of the token alone
    ([900, 0, 33, 2049, 5], [7, 1, 0, 90, 64], 6, 16, 4, 128, 256, -1, 0, "bf16"),
    ([900, 0, 33, 2049, 5], [7, 1, 0, 90, 64], 6, 28, 4, 64, 16, 40, 10, "fp16"),
    ([3] * 70, [i % 4 for i in range(70)], 2, 8, 8, 64, 16, -1, 0, "bf16"),
    ([500 + 97 * i for i in range(16)], 64, 12, 32, 8, 128, 64, -1, 0, "bf16"),  # waves with rows of their own
    ([77 * i for i in range(12)], 100, 9, 32, 4, 64, 32, 300, 3, "fp16"),
    ([1500, 0, 31, 800, 64, 9], [300, 2, 0, 130, 64, 257], 20, 48, 2, 128, 64, 100, 70, "bf16"),
    ([9000], 1024, 1, 32, 8, 128, 64, -1, 0, "fp16"),                     # the largest tree, a chain
    # 32 rows a wave, over row tiles of several chunks
    ([4000 + 100 * i for i in range(12)], 100, 9, 32, 4, 128, 32, 3000, 3, "fp16"),
    ([7000, 0, 31, 6800, 64, 6000], [300, 2, 0, 330, 64, 257], 20, 48, 2, 128, 64, -1, 0, "bf16"),
    ([9000, 12000, 700, 0], 130, 30, 16, 1, 64, 16, 8000, 2, "bf16"),
    # 16 rows a wave
    ([11 * i for i in range(64)], 12, 5, 32, 8, 128, 64, -1, 0, "bf16"),
    ([(37 * i) % 900 for i in range(128)], 10, 4, 16, 4, 64, 32, 100, 3, "fp16"),
    ([(61 * i) % 900 for i in range(70)], [(7 * i) % 25 for i in range(70)], 4, 32, 8, 128, 16, 9, 2, "fp16"),
    ([9000, 12000, 700, 0], 130, 30, 32, 2, 64, 16, 8000, 2, "bf16"),     # 32 rows a wave again, of head_dim 64
]


def tree_case(case, seed=0, wild=True, holes=0.03):
    lens, nodes, width, hq, hk, dim, size, window, sinks, dtype = TREES[case]
    rng = random.Random(7000 + case + seed)
    packed = isinstance(nodes, list)
    sizes = nodes if packed else [nodes] * len(lens)
    parents = [some_parents(rng, n, width, holes if n > 4 else 0) for n in sizes]
    cache, table, seqlens, _ = make(lens, hk, dim, size, 800 + case + seed, max_pages=max(1, -(-max(lens) // size) + case % 2))
    g = torch.Generator().manual_seed(900 + case + seed)
    lead = (sum(sizes) + 2,) if packed else (len(lens), nodes)  # (rows behind the last sequence)
    q = randn(g, DTYPES[dtype], *lead, hq, dim)
    k, v = (randn(g, DTYPES[dtype], *lead, hk, dim) for _ in range(2))
    cu = ints([sum(sizes[:i]) for i in range(len(sizes) + 1)]) if packed else None
    tree = tree_tensors(parents, packed)
    if packed:
        tree = type(tree)(*(torch.cat((t, t.new_full((2, *t.shape[1:]), -1))) for t in tree))
    if wild:  # what is not there may hold anything
        for b, at in enumerate(R.slices(cu, len(lens))):
            for i, line in enumerate(R.lines(parents[b])):
                if line is None:
                    for t in (q, k, v):
                        t[at][i] = math.nan if i % 2 else math.inf
    return (q, k, v, tree, cache, table, seqlens, window, cu, sinks), parents


def check_tree(args, parents, out, lse, scale=None):
    q, k, v, _, cache, table, seqlens, window, cu, sinks = args
    want, want_lse, spread, reach, total = R.tree_attn(q, k, v, parents, cache, table, seqlens, window, cu, scale, sinks)
    rows = slice(None) if cu is None else slice(0, int(cu[-1]))
    out, want, spread, total = out[rows], want[rows], spread[rows], total[rows]
    err = score_error(reach, q.shape[-1])
    per_row = err.transpose(-1, -2)[rows][..., None]
    bound = HALF[q.dtype] * (want.abs() + spread) + (2 * per_row + 2.0 ** -17) * spread + 2.0 ** -24
    if q.dtype == torch.float16:
        bound = bound + 2.0 ** -38 * total
    off = (out.double() - want).abs()
    assert torch.isfinite(out.float()).all()
    assert bool((off <= bound).all()), f"out off by up to {(off / bound).max().item():.2f} of its bound"
    if lse is not None:
        pick = (lambda t: t) if cu is None else (lambda t: t[:, rows])
        lse, want_lse, err = pick(lse), pick(want_lse), pick(err)
        empty = want_lse == -math.inf
        assert bool((lse[empty] == -math.inf).all())
        assert bool((out.transpose(-2, -3)[empty] == 0).all())
        off = (lse.double() - want_lse).abs()[~empty]
        assert bool((off <= (err + 2.0 ** -20 * (1 + want_lse.abs()))[~empty]).all()), f"lse off by {off.max()}"


def attend(args, **more):
    from ring_swa import kv_cache_tree_attn

    q, k, v, tree, cache, table, seqlens, window, cu, sinks = args
    return kv_cache_tree_attn(q, k, v, tree, cache, table, seqlens, window, cu, num_sink_tokens=sinks, **more)


@pytest.mark.parametrize("case", range(len(TREES)))
def test_tree_attention(case):
    args, parents = tree_case(case)
    out, lse = attend(args, return_lse=True)
    check_tree(args, parents, out, lse)
    rows = args[0].shape[-3] if args[8] is None else int(args[8][-1])  # (those behind are not written)
    assert torch.equal(out[..., :rows, :, :], attend(args)[..., :rows, :, :]), "without the lse"
    again = attend(args, return_lse=True)
    assert torch.equal(out[..., :rows, :, :], again[0][..., :rows, :, :]) and torch.equal(lse[..., :rows], again[1][..., :rows])


def test_a_scale_of_ones_own():
    args, parents = tree_case(1)
    out, lse = attend(args, softmax_scale=0.3, return_lse=True)
    check_tree(args, parents, out, lse, 0.3)


@pytest.mark.parametrize("window", [-1, 40])
def test_a_chain_whose_values_the_cache_holds_exactly(window):
    """Nodes that are e4m3 values, and a chain: ``kv_cache_attn`` after an append has the same result to approach."""
    from ring_swa import kv_cache_append, kv_cache_attn

    held, n, hk, dim = [3000, 50, 0, 64], 5, 2, 128
    cache, table, _, _ = make([h + n for h in held], hk, dim, 32, 21, wild=False)
    g = torch.Generator().manual_seed(3)
    q = randn(g, torch.bfloat16, 4, n, 8, dim)
    # (multiples of 1/4 up to 2 are codes at any scale between 2^-7, which holds them, and 2^3; a page's scale is 2^-5 to 2^2)
    k, v = ((torch.randint(-8, 9, (4, n, hk, dim), generator=g) / 4).bfloat16().cuda() for _ in range(2))
    chain = [list(range(-1, n - 1))] * 4
    args = (q, k, v, tree_tensors(chain, False), cache, table, ints(held), window, None, 3)
    out, lse = attend(args, return_lse=True)
    check_tree(args, chain, out, lse)
    kv_cache_append(cache, k, v, table, ints(held))
    lens = ints(held) + n
    check_attn(q, cache, table, lens, out, lse, window, sinks=3)
    check_attn(q, cache, table, lens, *kv_cache_attn(q, cache, table, lens, window, num_sink_tokens=3, return_lse=True), window, sinks=3)


@pytest.mark.parametrize("case", [1, 4, 11, 13, 15, 17, 19, 20])
def test_what_is_not_finite_reaches_the_descendants_alone(case):
    args, parents = tree_case(case, wild=False)
    q, k, v, tree, cache, table, lens, window, cu, sinks = args
    clean = attend(args)
    bad = v.clone()
    marks = {}
    for b, at in enumerate(R.slices(cu, len(lens))):
        n = len(parents[b])
        for i, value in ((0, None), (n // 3, math.inf), (n // 2, -math.inf), (n - 1, math.nan)):
            if value is not None and 0 < i < n:
                bad[at][i, :, 3::7] = value
                marks.setdefault(b, {})[i] = value
    out = attend((q, k, bad, *args[3:]))
    for b, at in enumerate(R.slices(cu, len(lens))):
        length = int(lens[b])
        see = R.seen(parents[b], length, window, sinks, torch.ones(length, dtype=torch.bool))[:, length:]
        for r in range(len(parents[b])):
            hit = [v for i, v in marks.get(b, {}).items() if see[r, i]]
            mine, was = out[at][r].float(), clean[at][r].float()
            assert torch.equal(mine[:, 0], was[:, 0]), "dimensions without such values"
            if not hit:
                assert torch.equal(mine, was), (b, r)
            elif any(math.isnan(x) for x in hit) or {math.inf, -math.inf} <= set(hit):
                assert bool(mine[:, 3::7].isnan().all()), (b, r)
            else:  # (a weight too small for its type times infinity is NaN)
                there = mine[:, 3::7]
                assert bool(((there == hit[0]) | there.isnan()).all()), (b, r)


@pytest.mark.parametrize("case", [12, 15, 19, 21])
def test_cached_values_that_are_not_finite(case):
    """NaN codes in the window of some nodes and not of others."""
    args, parents = tree_case(case, wild=False, holes=0)
    q, k, v, tree, cache, table, lens, window, cu, sinks = args
    clean = attend(args)
    size = cache[0].shape[2]
    codes = cache[1].view(torch.uint8)
    hit = {}
    for b, n in enumerate(lens.tolist()):
        j = n - window + 1  # (the root and its children see it, deeper nodes do not)
        if j >= sinks:
            codes[int(table[b, j // size]), :, (j % size) // 16, 5, j % 16] = 0x7F
            hit[b] = j
    out = attend(args)
    assert hit
    for b in range(len(lens)):
        depth = tree.depths[b]
        sees = (depth <= 1) if b in hit else torch.zeros_like(depth, dtype=torch.bool)
        for r in range(out.shape[1]):
            if bool(sees[r]):
                assert bool(out[b, r, :, 5].isnan().all())
                assert torch.equal(out[b, r, :, :5], clean[b, r, :, :5])
            else:
                assert torch.equal(out[b, r], clean[b, r])


def test_pages_missing_lengths_beyond_and_tables_without_columns():
    args, parents = tree_case(5)
    q, k, v, tree, cache, table, lens, window, cu, sinks = args
    table = table.clone()
    table[0, 3], table[0, 5], table[2, 1] = -1, cache[0].shape[0], 2 ** 31 - 1
    cut = (q, k, v, tree, cache, table, lens, window, cu, sinks)
    out, lse = attend(cut, return_lse=True)
    check_tree(cut, parents, out, lse)
    # (the pages of `make` hold NaN behind the last token, which a longer length rightly sees: pages without)
    clean, places, _, _ = make([200] * 3, k.shape[2], q.shape[-1], 32, 5, wild=False)
    long = (q, k, v, tree, clean, places, ints([2 ** 30, -5, 10 ** 6]), window, cu, sinks)
    out, lse = attend(long, return_lse=True)
    check_tree(long, parents, out, lse)
    none = cut[:5] + (table[:, :0],) + cut[6:]
    out, lse = attend(none, return_lse=True)
    check_tree(none, parents, out, lse)


def test_strided_rows_trees_and_caches():
    args, parents = tree_case(4, wild=False)
    q, k, v, tree, cache, table, lens, window, cu, sinks = args
    want = attend(args, return_lse=True)
    b, n, hq, d = q.shape
    qkv = torch.zeros(b, n, hq + 2 * k.shape[2] + 1, d, dtype=q.dtype, device="cuda")
    qs, ks, vs = qkv[:, :, :hq], qkv[:, :, hq:hq + k.shape[2]], qkv[:, :, hq + k.shape[2]:-1]
    qs.copy_(q), ks.copy_(k), vs.copy_(v)
    apart = [torch.stack((t, t), 1)[:, 0] for t in tree]
    assert apart[2].stride(0) == 2 * tree[2].stride(0)
    got = attend((qs, ks, vs, type(tree)(*apart), *args[4:]), return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = type(tree)(*(t[:1].expand(b, *t.shape[1:]) for t in tree))
    got = attend((q, k, v, one, *args[4:]), return_lse=True)
    check_tree((q, k, v, one, *args[4:]), [parents[0]] * b, *got)


def test_rows_behind_the_last_sequence_are_left(monkeypatch):
    args, _ = tree_case(8)
    from ring_swa.ops import drafts

    made = []

    def results(q, packed, return_lse):
        made[:] = [torch.full_like(q, 7.0), torch.full((q.shape[1], q.shape[0]), 7.0, device="cuda")]
        return tuple(made)

    monkeypatch.setattr(drafts, "_results", results)
    monkeypatch.setattr(drafts, "_calls", lambda *_: None)
    out, lse = attend(args, return_lse=True)
    rows = int(args[8][-1])
    assert bool((out[rows:] == 7).all()) and bool((lse[:, rows:] == 7).all()) and not bool((out[:rows] == 7).all())


# ---- verification -------------------------------------------------------------------------------
def probabilities(g, rows, vocab, dtype, sharp=2.0):
    common = torch.randn(rows, vocab, generator=g) * sharp
    return [torch.softmax(common + torch.randn(rows, vocab, generator=g) * 0.7, -1).to(dtype) for _ in range(2)]


def drawn(rng, parents, q):
    """Tokens of the nodes: drawn from their parents' row of q."""
    q = q.double().cumsum(-1)
    return [int(torch.searchsorted(q[p], rng.random() * q[p][-1])) if p >= 0 else 0 for p in parents]


VERIFY = [
    # nodes (a list: packed), width, vocab, dtype, draft, type of tokens
    ([1], 1, 1, "fp32", True, torch.int32),
    ([6] * 5, 1, 1000, "fp32", True, torch.int64),
    ([32] * 7, 10, 5003, "fp32", True, torch.int32),
    ([32] * 7, 10, 5003, "bf16", True, torch.int32),
    ([40] * 4, 39, 4097, "fp16", True, torch.int64),
    ([9, 1, 0, 70, 3, 64], 30, 8191, "fp32", True, torch.int32),
    ([9, 1, 0, 70, 3, 64], 30, 300, "bf16", False, torch.int64),
    ([25] * 9, 24, 40, "fp32", False, torch.int32),
    ([130] * 3, 129, 50, "fp32", False, torch.int32),
    ([130] * 3, 129, 20, "fp32", True, torch.int32),
    ([12] * 3, 4, 150001, "fp32", True, torch.int32),
]


@pytest.mark.parametrize("case", range(len(VERIFY)))
def test_verification(case):
    from ring_swa import verify_drafts

    sizes, width, vocab, dtype, sampled, kind = VERIFY[case]
    packed = len(set(sizes)) > 1
    dtype = {"fp32": torch.float32, **DTYPES}[dtype]
    rng = random.Random(case)
    g = torch.Generator().manual_seed(case)
    taken = 0
    for trial in range(6):
        parents = [some_parents(rng, n, width, 0.02) for n in sizes]
        parents = [[-1] + p[1:] if p else p for p in parents]
        total = sum(sizes)
        p, q = probabilities(g, total, vocab, dtype)
        tokens, base = [], 0
        for own in parents:
            there = [x if R.lines(own)[i] is not None else -2 for i, x in enumerate(own)]
            tokens.append(drawn(rng, there, q[base:base + len(own)]))
            base += len(own)
        flat = torch.tensor(sum(tokens, []), dtype=kind)
        u = torch.rand(total, generator=g)
        tree = tree_tensors(parents, packed)
        cu = ints([sum(sizes[:i]) for i in range(len(sizes) + 1)]) if packed else None
        shape = (total,) if packed else (len(sizes), sizes[0])
        path, accepted, token = verify_drafts(tree, flat.view(shape).cuda(), p.view(*shape, vocab).cuda(),
                                              q.view(*shape, vocab).cuda() if sampled else None, u.view(shape).cuda(), cu)
        assert path.dtype == accepted.dtype == torch.int32 and token.dtype == kind
        base = 0
        for b, own in enumerate(parents):
            rows = slice(base, base + len(own))
            base += len(own)
            there = R.tree(own, max(1, len(own)))[0]
            want, following = R.verify(there, flat[rows].tolist(), p[rows], q[rows] if sampled else None,
                                       u[rows].tolist())
            assert int(accepted[b]) == len(want), (trial, b)
            assert path[b].tolist() == want + [-1] * (path.shape[1] - len(want)), (trial, b)
            assert int(token[b]) == following, (trial, b)
            taken += max(0, len(want) - 1)
    assert taken > 0 or vocab == 1 or not sampled  # (tokens drawn from the draft, not its likeliest: few are taken without it)


def verified(parents, tokens, target, draft, uniforms, kind=torch.int32):
    """One sequence; (nodes, next token)."""
    from ring_swa import verify_drafts

    n = len(parents)
    path, accepted, token = verify_drafts(
        tree_tensors([parents], False), torch.tensor([tokens], dtype=kind).cuda(), target[None].cuda(),
        None if draft is None else draft[None].cuda(), torch.tensor([uniforms], dtype=torch.float32).cuda())
    assert path.shape == (1, n)
    return path[0, :int(accepted)].tolist(), int(token)


def test_verification_at_the_edges():
    eye = torch.eye(6)
    half = torch.tensor([0.5, 0.5, 0, 0, 0, 0])
    # greedy: one-hot targets take the one token, whatever the draft gave it
    p = torch.stack((eye[3], eye[4], eye[5]))
    q = torch.full((3, 6), 1 / 6)
    assert verified([-1, 0, 1], [0, 3, 4], p, q, [0.999, 0.99, 0.99]) == ([0, 1, 2], 5)
    assert verified([-1, 0, 1], [0, 2, 4], p, q, [0.0, 0.0, 0.0]) == ([0], 3)
    assert verified([-1, 0, 0], [0, 2, 3], p, q, [0.5, 0.0, 0.9]) == ([0, 2], 5)
    assert verified([-1, 0, 0], [0, 2, 3], p, None, [0.5, 0.0, 0.9]) == ([0, 2], 5)
    # the same distribution in both: always taken
    assert verified([-1, 0, 1], [0, 0, 1], torch.stack((half, half, eye[2])), torch.stack((half, half, half)),
                    [0.1, 1 - 2.0 ** -24, 1 - 2.0 ** -24]) == ([0, 1, 2], 2)
    # a token that the draft gave no probability, and the target some
    assert verified([-1, 0], [0, 1], torch.stack((half, eye[0])), torch.stack((eye[0], eye[0])), [0.3, 0.99]) == ([0, 1], 0)
    # ties: the border itself belongs to the next token
    assert verified([-1], [0], half[None], None, [0.5]) == ([0], 1)
    assert verified([-1], [0], half[None], None, [0.5 - 2.0 ** -25]) == ([0], 0)
    # tokens out of the vocabulary, twice the same one
    assert verified([-1, 0, 0, 0], [0, 6, -1, 0], torch.stack([half] * 4), None, [0.2, 0.0, 0.0, 0.4]) == ([0, 3], 0)
    assert verified([-1, 0, 0, 0], [0, 2 ** 40, -2 ** 40, 0], torch.stack([half] * 4), None, [0.2, 0.0, 0.0, 0.4], torch.int64) == ([0, 3], 0)
    assert verified([-1, 0, 0, 0], [0, 0, 0, 1], torch.stack([half] * 4), None, [0.7, 0.6, 0.0, 0.99]) == ([0, 3], 1)
    # nothing is left of the target after its tokens were tried: drawn from itself
    tiny = torch.tensor([0.5, 0.25, 0, 0, 0, 0])
    assert verified([-1, 0, 0], [0, 0, 1], torch.stack([tiny] * 3), None, [0.9, 0.9, 0.99]) == ([0], 1)
    q = torch.stack([torch.tensor([0.9, 0.9, 0, 0, 0, 0])] * 2)
    assert verified([-1, 0], [0, 0], torch.stack((tiny, tiny)), q, [0.1, 0.99]) == ([0], 0)
    # no probabilities at all, and such as are none
    none = torch.zeros(2, 6)
    assert verified([-1, 0], [0, 0], none, none, [0.5, 0.0]) == ([0], -1)
    odd = torch.tensor([[math.nan, -1.0, 0.25, -math.inf, 0.75, math.nan]] * 2)
    assert verified([-1, 0], [0, 0], odd, None, [0.1, 0.0]) == ([0], 2)
    assert verified([-1, 0], [0, 4], odd, odd, [0.9, 0.9]) == ([0, 1], 4)
    # a uniform of one or more, or NaN
    assert verified([-1], [0], half[None], None, [1.0]) == ([0], 1)
    assert verified([-1], [0], half[None], None, [math.nan]) == ([0], 1)
    # the root is not there
    assert verified([-2, 0], [0, 0], torch.stack((half, half)), None, [0.1, 0.1]) == ([], -1)
    # a second tree of the sequence: not the root's
    assert verified([-1, -1, 1, 0], [0, 0, 0, 1], torch.stack([half] * 4), None, [0.1, 0.0, 0.0, 0.3]) == ([0, 3], 0)


def test_sequences_without_nodes():
    from ring_swa import DraftTree, verify_drafts

    tree = DraftTree(ints([]), ints([]), torch.zeros(0, 2, dtype=torch.int64, device="cuda"))
    none = torch.zeros(0, 9, device="cuda")
    path, accepted, token = verify_drafts(tree, ints([]), none, none, torch.zeros(0, device="cuda"), ints([0, 0, 0]))
    assert path.shape == (2, 128) and bool((path == -1).all()) and accepted.tolist() == [0, 0] and token.tolist() == [-1, -1]
    dense = DraftTree(ints([[], []]), ints([[], []]), torch.zeros(2, 0, 1, dtype=torch.int64, device="cuda"))
    path, accepted, token = verify_drafts(dense, ints([[], []]), none.view(2, 0, 9), None, torch.zeros(2, 0, device="cuda"))
    assert path.shape == (2, 0) and accepted.tolist() == [0, 0] and token.tolist() == [-1, -1]


def test_strided_probabilities():
    from ring_swa import verify_drafts

    g = torch.Generator().manual_seed(8)
    rng = random.Random(8)
    parents = [some_parents(rng, 20, 9) for _ in range(3)]
    p, q = (t.view(3, 20, 777).cuda() for t in probabilities(g, 60, 777, torch.bfloat16))
    tokens = torch.stack([torch.tensor(drawn(rng, own, q[b].cpu())) for b, own in enumerate(parents)]).cuda()
    u = torch.rand(3, 20, generator=g).cuda()
    tree = tree_tensors(parents, False)
    want = verify_drafts(tree, tokens, p, q, u)
    room = torch.zeros(3, 21, 2, 779, dtype=torch.bfloat16, device="cuda")
    room[:, 1:, 0, 1:778], room[:, 1:, 1, 2:779] = p, q
    wide = torch.zeros(3, 40, dtype=tokens.dtype, device="cuda")
    wide[:, 20:] = tokens
    got = verify_drafts(tree, wide[:, 20:], room[:, 1:, 0, 1:778], room[:, 1:, 1, 2:779], torch.cat((u, u), 1)[:, :20])
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("sampled", [True, False])
def test_tokens_are_distributed_as_the_targets(sampled):
    """Of 60000 sequences with the same distributions the first chosen token's share is the target's, within five standard
    deviations of a count (a chance of 1e-6 for each of the 7 tokens, and the numbers are always the same)."""
    from ring_swa import verify_drafts

    n, vocab = 60000, 7
    g = torch.Generator().manual_seed(4)
    p = torch.softmax(torch.randn(vocab, generator=g) * 1.2, -1)
    q = torch.softmax(torch.randn(vocab, generator=g) * 1.2, -1)
    parents = [-1, 0, 0, 0]
    if sampled:
        tokens = torch.multinomial(q.expand(4 * n, vocab), 1, generator=g).view(n, 4).int()
    else:
        tokens = q.topk(4).indices.int().expand(n, 4)
    tree = tree_tensors([parents], False)
    tree = type(tree)(*(t.expand(n, *t.shape[1:]) for t in tree))
    rows = lambda t: t.cuda().expand(n, 4, vocab)
    path, accepted, token = verify_drafts(tree, tokens.cuda(), rows(p), rows(q) if sampled else None, torch.rand(n, 4, generator=g).cuda())
    first = torch.where(accepted > 1, tokens.cuda().gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], token)
    share = first.long().bincount(minlength=vocab).double().cpu() / n
    assert bool(((share - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()), (share, p)
    taken = float((accepted > 1).double().mean())
    if sampled:
        assert 0.5 < taken < 1
    else:  # (its three drafts' own probabilities)
        want = float(p[tokens[0, 1:].long()].sum())
        assert abs(taken - want) <= 5 * (want * (1 - want) / n) ** 0.5


# ---- the accepted drafts into the cache ---------------------------------------------------------
ACCEPT = [
    # lens before, nodes (a list: packed), path (its most), kv heads, dim, page, dtype
    ([0], 1, 1, 8, 128, 64, "bf16"),
    ([5, 63, 64, 127], 9, 4, 2, 128, 64, "bf16"),
    ([0, 1, 15, 16, 17], 20, 20, 3, 64, 16, "fp16"),        # more rows than a wave holds, over three pages
    ([250, 3], 300, 290, 1, 64, 256, "fp16"),
    ([10, 0, 200, 77], [5, 0, 1, 130], 70, 4, 128, 64, "bf16"),
    ([i % 37 for i in range(70)], [i % 5 for i in range(70)], 6, 1, 64, 16, "bf16"),
]


@pytest.mark.parametrize("case", range(len(ACCEPT)))
def test_accept_is_an_append_of_the_named_rows(case):
    from ring_swa import kv_cache_accept

    held, nodes, most, hk, dim, size, dtype = ACCEPT[case]
    dtype = DTYPES[dtype]
    packed = isinstance(nodes, list)
    sizes = nodes if packed else [nodes] * len(held)
    cache, table, _, _ = make([h + most for h in held], hk, dim, size, 40 + case, wild=False)
    lens = ints(held)
    g = torch.Generator().manual_seed(70 + case)
    rng = random.Random(case)
    lead = (sum(sizes) + 3,) if packed else (len(held), nodes)
    k, v = (randn(g, torch.float32, *lead, hk, dim) * torch.exp2(torch.randint(-12, 9, (*lead, hk, 1), generator=g).float()).cuda()
            for _ in range(2))
    k, v = k.to(dtype), v.to(dtype)
    cu = ints([sum(sizes[:i]) for i in range(len(sizes) + 1)]) if packed else None
    path = []
    for n in sizes:
        count = rng.randint(0, min(n, most))
        row = [rng.randrange(n) for _ in range(count)]  # (any rows in any order)
        end = rng.choice([-1, n, 2 ** 31 - 1, -2 ** 31])  # (behind an entry that is none nothing is looked at)
        path.append((row + [end] + [0] * most)[:most])
    room = torch.zeros(len(held), most + 2, dtype=torch.int32, device="cuda")
    room[:, 1:most + 1] = ints(path)
    path = room[:, 1:most + 1]
    want = R.accept(cache, k, v, path, table, lens, cu)
    kv_cache_accept(cache, k, v, path, table, lens, cu)
    assert O.same_bytes(cache, want)
    assert lens.tolist() == held
    kv_cache_accept(cache, k, v, path, table, lens, cu)  # the same again changes nothing
    assert O.same_bytes(cache, want)


def test_accept_drops_what_has_no_page():
    from ring_swa import kv_cache_accept

    g = torch.Generator().manual_seed(4)
    cache, table, _, _ = make([64] * 4, 2, 64, 16, 9, wild=False)
    table[0, 1], table[1, 0], table[2, 2] = -1, cache.k.shape[0], 2 ** 31 - 1
    lens = ints([10, 0, 60, 2 ** 31 - 1])  # the third runs over its row of the table, the fourth is beyond it
    k, v = (randn(g, torch.bfloat16, 4, 40, 2, 64) for _ in range(2))
    path = torch.arange(40, dtype=torch.int32, device="cuda").expand(4, 40)
    want = R.accept(cache, k, v, path, table, lens)
    kv_cache_accept(cache, k, v, path, table, lens)
    assert O.same_bytes(cache, want)
    kv_cache_accept(cache, k, v, path, table, ints([-5, -1, -2 ** 31, -3]))
    assert O.same_bytes(cache, R.accept(want, k, v, path, table, ints([0, 0, 0, 0])))
    before = [t.view(torch.uint8).clone() for t in cache]
    kv_cache_accept(cache, k, v, path[:, :0], table, lens)
    kv_cache_accept(cache, k[:, :0], v[:, :0], path, table, lens)
    kv_cache_accept(cache, k, v, path, table[:, :0], lens)
    assert all(torch.equal(t.view(torch.uint8), was) for t, was in zip(cache, before))


def test_accept_of_extreme_values():
    from ring_swa import kv_cache_accept

    for dtype in (torch.bfloat16, torch.float16):
        info = torch.finfo(dtype)
        rows = torch.stack([torch.zeros(128), torch.full((128,), info.max), torch.full((128,), info.tiny),
                            torch.full((128,), math.nan), torch.full((128,), -math.inf),
                            torch.cat([torch.full((64,), math.inf), torch.linspace(-3, 3, 64)]), 448 + torch.arange(128) / 8.0])
        x = rows.to(dtype).cuda().view(1, -1, 1, 128)
        for path in ([0], [1], [2], [3, 4], [5], [6, 0], [2, 5, 1, 3]):
            cache, table, lens, _ = make([9 + len(path)], 1, 128, 64, 7, wild=False)
            lens -= len(path)
            want = R.accept(cache, x, x, ints([path]), table, lens)
            kv_cache_accept(cache, x, x, ints([path]), table, lens)
            assert O.same_bytes(cache, want), path


# ---- cached tokens back -------------------------------------------------------------------------
READ = [
    # lens, rows read (a list: packed), from the end?, kv heads, dim, page, dtype
    ([1], 1, True, 1, 64, 16, "bf16"),
    ([100, 64, 63], 50, True, 8, 128, 64, "bf16"),
    ([300, 17, 16], 16, False, 3, 64, 16, "fp16"),
    ([700, 1000], 700, True, 2, 128, 256, "fp16"),
    ([900, 31, 5, 64], [500, 31, 0, 7], True, 4, 128, 32, "bf16"),
    ([33] * 70, [i % 30 for i in range(70)], True, 1, 64, 128, "bf16"),
]


@pytest.mark.parametrize("case", range(len(READ)))
def test_read_is_what_the_codes_say(case):
    from ring_swa import kv_cache_read

    lens, rows, from_end, hk, dim, size, dtype = READ[case]
    packed = isinstance(rows, list)
    counts = rows if packed else [rows] * len(lens)
    cache, table, _, _ = make(lens, hk, dim, size, 60 + case)
    first = ints([n - r if from_end else 0 for n, r in zip(lens, counts)])
    lead = (sum(counts) + 3,) if packed else (len(lens), rows)
    # (rows of a tensor that holds more than them)
    both = torch.full((*lead, 2 * hk + 1, dim), 7.0, dtype=DTYPES[dtype], device="cuda")
    k, v = both[..., :hk, :], both[..., hk:2 * hk, :]
    cu = ints([sum(counts[:i]) for i in range(len(counts) + 1)]) if packed else None
    kv_cache_read(cache, k, v, table, first, cu)
    assert bool((both[..., -1, :] == 7).all())
    if packed:
        assert bool((both[sum(counts):] == 7).all())
    got = R.read(cache, table, first, counts)
    for b, at in enumerate(R.slices(cu, len(lens))):
        for mine, want in zip((k[at], v[at]), got[b]):
            assert torch.equal(mine, want.to(DTYPES[dtype]))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_read_of_every_code_at_every_scale(dtype):
    """All 256 codes at the scales of the type's ends and between: rounded once, infinite beyond the largest, NaN codes NaN."""
    from ring_swa import KVCache, kv_cache_read

    dtype = DTYPES[dtype]
    scales = [0, 1, 7, 8, 60, 100, 103, 104, 105, 110, 118, 127, 130, 134, 135, 136, 140, 200, 240, 246, 247, 248, 254]
    pages = len(scales)
    codes = torch.arange(256, dtype=torch.uint8).repeat(pages, 1, 4, 1).view(pages, 1, 16, 64)  # 16 tokens of 64
    cache = KVCache.empty(pages, 1, 64, 16, device="cuda")
    cache.k.view(torch.uint8).copy_(codes)
    cache.v.view(torch.uint8).copy_(codes.view(pages, 1, 1, 16, 64).transpose(-1, -2))
    for t in cache[2:]:
        t.view(torch.uint8).copy_(torch.tensor(scales, dtype=torch.uint8)[:, None])
    k, v = (torch.empty(1, 16 * pages, 1, 64, dtype=dtype, device="cuda") for _ in range(2))
    kv_cache_read(cache, k, v, ints([list(range(pages))]), ints([0]))
    want = (O.decode(codes).view(pages, 16, 64) * torch.pow(2.0, torch.tensor(scales).double() - 127)[:, None, None]).to(dtype)
    for x in (k, v):
        x = x.cpu().view(pages, 16, 64)
        same = (x == want) | (x.isnan() & want.isnan())
        assert bool(same.all()), [scales[i] for i in (~same).flatten(1).any(1).nonzero().flatten().tolist()]


def test_read_where_there_is_nothing():
    from ring_swa import kv_cache_read

    cache, table, _, _ = make([64] * 4, 2, 64, 16, 9, wild=False)
    table[0, 1], table[1, 0], table[2, 2] = -1, cache.k.shape[0], 2 ** 31 - 1
    first = ints([0, -7, 50, 2 ** 31 - 1])
    k, v = (torch.full((4, 40, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kv_cache_read(cache, k, v, table, first)
    for b, got in enumerate(R.read(cache, table, first, [40] * 4)):
        assert torch.equal(k[b], got[0].bfloat16()) and torch.equal(v[b], got[1].bfloat16())
    assert bool((k[3] == 0).all())
    k.fill_(7.0), v.fill_(7.0)
    kv_cache_read(cache, k, v, table[:, :0], first)
    assert bool((k == 0).all()) and bool((v == 0).all())
    kv_cache_read(cache, k[:, :0], v[:, :0], table, first)


def test_what_was_appended_comes_back_within_half_a_step():
    """A code is off by half a step of e4m3 at most (2^-4 of the value, or half of the least step at the page's scale, 2^-10
    of its power of two); reading adds nothing: code values are exact in bf16 and, at these sizes, in fp16."""
    from ring_swa import KVCache, kv_cache_append, kv_cache_read

    g = torch.Generator().manual_seed(2)
    for dtype in (torch.bfloat16, torch.float16):
        cache = KVCache.empty(12, 3, 128, 32, device="cuda")
        table = torch.randperm(12, generator=g).int().view(2, 6).cuda()
        k, v = (randn(g, dtype, 2, 150, 3, 128) for _ in range(2))
        kv_cache_append(cache, k, v, table, ints([0, 30]))
        a, b = torch.empty_like(k), torch.empty_like(v)
        kv_cache_read(cache, a, b, table, ints([0, 30]))
        for x, y in ((k, a), (v, b)):
            step = x.abs().amax().double() / 224 * 2.0 ** -10  # (a scale is below max / 224)
            assert bool(((x.double() - y.double()).abs() <= x.double().abs() * 2.0 ** -4 + step).all())


# ---- together -----------------------------------------------------------------------------------
def step(cache, table, held, parents, q, k, v, tokens, target, draft, uniforms):
    """One layer's share of a step with drafts, as a server makes it."""
    from ring_swa import draft_tree, kv_cache_accept, kv_cache_read, kv_cache_tree_attn, verify_drafts

    tree = draft_tree(parents)
    out, lse = kv_cache_tree_attn(q, k, v, tree, cache, table, held, 900, num_sink_tokens=2, return_lse=True)
    path, accepted, token = verify_drafts(tree, tokens, target, draft, uniforms)
    kv_cache_accept(cache, k, v, path, table, held)
    held += accepted
    back = [torch.empty_like(k) for _ in range(2)]
    kv_cache_read(cache, *back, table, held - accepted)
    return (*tree, out, lse, path, accepted, token, *back)


def step_inputs(seed, lens=(3000, 90, 1), nodes=20):
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    cache, table, _, _ = make([n + nodes for n in lens], 2, 64, 32, 300, max_pages=100, wild=False)
    parents = [some_parents(rng, nodes, 6) for _ in lens]
    q = randn(g, torch.bfloat16, len(lens), nodes, 8, 64)
    k, v = (randn(g, torch.bfloat16, len(lens), nodes, 2, 64) for _ in range(2))
    p, d = (t.view(len(lens), nodes, 2000) for t in probabilities(g, len(lens) * nodes, 2000, torch.float32))
    tokens = torch.tensor([drawn(rng, own, d[b]) for b, own in enumerate(parents)])
    return [cache, table, ints(lens), ints(parents), q, k, v, tokens.cuda(), p.cuda(), d.cuda(),
            torch.rand(len(lens), nodes, generator=g).cuda()]


def as_bytes(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def test_a_step_of_drafts():
    """Several steps: each part against its restatement, the cache and the lengths carried on."""
    cache, table, held, *_ = step_inputs(0)
    for seed in range(4):
        _, _, _, parents, q, k, v, tokens, p, d, u = step_inputs(seed)
        before, was = type(cache)(*(t.clone() for t in cache)), held.clone()
        got = step(cache, table, held, parents, q, k, v, tokens, p, d, u)
        _, depths, _, out, lse, path, accepted, token, back_k, back_v = got
        lists = parents.tolist()
        check_tree((q, k, v, None, before, table, was, 900, None, 2), lists, out, lse)
        for b, own in enumerate(lists):
            want = R.verify(own, tokens[b].tolist(), p[b].cpu(), d[b].cpu(), u[b].tolist())
            assert path[b, :int(accepted[b])].tolist() == want[0] and int(token[b]) == want[1]
            assert depths[b, want[0]].tolist() == list(range(len(want[0])))
        assert O.same_bytes(cache, R.accept(before, k, v, path, table, was))
        assert torch.equal(held, was + accepted)
        for b in range(len(lists)):
            n = int(accepted[b])
            for x, y in ((k, back_k), (v, back_v)):
                x, y = x[b, path[b, :n].long()].double(), y[b, :n].double()
                assert bool(((x - y).abs() <= x.abs() * 2.0 ** -4 + 2.0 ** -6).all())


def test_a_captured_step_replays():
    args = step_inputs(1)
    cache, table, held = args[:3]
    start = [t.clone() for t in cache], held.clone()

    def reset():
        for t, s in zip(cache, start[0]):
            t.copy_(s)
        held.copy_(start[1])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*args)
    with torch.cuda.graph(other, pool=graph.pool()):
        got2 = step(*args)
    for trial in range(4):
        for mine, new in zip(args[3:], step_inputs(10 + trial)[3:]):
            mine.copy_(new)
        start[1].copy_(ints([(3000, 90, 1), (1500, 32, 64), (2999, 1, 0), (90, 60, 2)][trial]))
        for run, outs in ((graph, got), (other, got2)):
            reset()
            run.replay()
            torch.cuda.synchronize()
            replayed = [as_bytes(t).clone() for t in (*outs, *cache, held)]
            reset()
            eager = [as_bytes(t) for t in (*step(*args), *cache, held)]
            torch.cuda.synchronize()
            for i, (x, y) in enumerate(zip(replayed, eager)):
                assert torch.equal(x, y), (trial, i)


def test_steps_on_two_streams_at_once():
    want = []
    for seed in (2, 3):
        args = step_inputs(seed)
        want.append([as_bytes(t).clone() for t in (*step(*args), *args[0])])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        both = [step_inputs(seed) for seed in (2, 3)]
        torch.cuda.synchronize()
        outs = []
        for stream, args in zip(streams, both):
            with torch.cuda.stream(stream):
                outs.append(step(*args))
        torch.cuda.synchronize()
        for got, args, w in zip(outs, both, want):
            for x, y in zip((*got, *args[0]), w):
                assert torch.equal(as_bytes(x), y)


def test_the_python_route_beside_the_native_one(monkeypatch):
    from ring_swa.ops import drafts, kv_cache

    for lens in ((3000, 90, 1), (5,)):
        args = step_inputs(6, lens)
        want = [as_bytes(t).clone() for t in (*step(*args), *args[0], args[2])]
        with monkeypatch.context() as m:
            for mod in (drafts, kv_cache):
                m.setattr(mod, "_calls", lambda *_: None)
            args = step_inputs(6, lens)
            got = [as_bytes(t) for t in (*step(*args), *args[0], args[2])]
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_the_native_route_takes_the_calls(monkeypatch):
    """(None of these may fall through to Python.)"""
    from ring_swa.ops import drafts, kv_cache

    def fell(*_):
        raise AssertionError("not taken")

    for mod, names in ((drafts, ("_tree", "_tree_attn", "_verify", "_accept")), (kv_cache, ("_read",))):
        for name in names:
            monkeypatch.setattr(mod, name, fell)
    step(*step_inputs(6))
    from ring_swa import draft_tree, kv_cache_accept, verify_drafts

    args, _ = tree_case(8)
    attend(args)
    draft_tree(args[3].parents, args[8], max_nodes=90)
    kv_cache_accept(args[4], args[1], args[2], ints([[0, -1]] * 5), args[5], args[6], args[8])
    p = torch.rand(args[0].shape[0], 50, device="cuda")
    verify_drafts(args[3], args[3].parents.clamp(min=0), p, None, torch.rand(len(p), device="cuda"), args[8])


def test_prefixes_read_back_go_to_the_attention_functions():
    """A cached sequence's end attended by the training kernels, over what is read back, and by the cache's: within the sum
    of the two's roundings (outputs and weights, of values below 4)."""
    from ring_swa import kv_cache_attn, kv_cache_read, ring_sliding_window_attn_varlen

    lens = [500, 64, 1, 333]
    cache, table, seqlens, _ = make(lens, 2, 128, 64, 31)
    cu = ints([sum(lens[:i]) for i in range(len(lens) + 1)])
    g = torch.Generator().manual_seed(5)
    q = randn(g, torch.bfloat16, sum(lens), 8, 128)
    k, v = (torch.empty(sum(lens), 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kv_cache_read(cache, k, v, table, torch.zeros_like(seqlens), cu)
    want, _, spread, _, _ = O.attn(q, cache, table, seqlens, 100, cu)
    for out in (kv_cache_attn(q, cache, table, seqlens, 100, cu), ring_sliding_window_attn_varlen(q, k, v, 100, cu)):
        # (the training kernels also round the weights at a stale maximum, up to 2^8 of it: the same relative step)
        assert bool(((out.double() - want).abs() <= 2 * HALF[torch.bfloat16] * (want.abs() + spread) + 2.0 ** -12 * spread + 2.0 ** -24).all())


def test_compiled_and_traced_steps():
    def run(k_codes, v_codes, k_scale, v_scale, *rest):
        from ring_swa import KVCache

        return step(KVCache(k_codes, v_codes, k_scale, v_scale), *rest)

    from torch.fx.experimental.proxy_tensor import make_fx

    def flat(seed):
        cache, *rest = step_inputs(seed)
        return (*cache, *rest)

    torch._dynamo.reset()
    for made in (torch.compile(run, backend="eager"), torch.jit.trace(run, flat(5), check_trace=False), make_fx(run)(*flat(5))):
        for seed in (6, 7):
            mine, want = flat(seed), flat(seed)
            got = (*made(*mine), *mine)
            for x, y in zip(got, (*run(*want), *want)):
                assert torch.equal(as_bytes(x), as_bytes(y))


def test_derivatives_are_refused():
    from ring_swa import DraftTree, kv_cache_accept, kv_cache_read, kv_cache_tree_attn, verify_drafts

    cache, table, held, parents, q, k, v, tokens, p, d, u = step_inputs(6)
    from ring_swa import draft_tree

    tree = draft_tree(parents)
    path = torch.zeros_like(parents)
    calls = [lambda t: kv_cache_tree_attn(t, k, v, tree, cache, table, held), lambda t: kv_cache_tree_attn(q, t, v, tree, cache, table, held),
             lambda t: kv_cache_tree_attn(q, k, t, tree, cache, table, held)]
    for call, t in zip(calls, (q, k, v)):
        with pytest.raises(RuntimeError, match="no backward"):
            call(t.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no backward"):
        verify_drafts(tree, tokens, p.clone().requires_grad_(), d, u)
    with pytest.raises(RuntimeError, match="no backward"):
        verify_drafts(tree, tokens, p, d.clone().requires_grad_(), u)
    with pytest.raises(RuntimeError, match="no backward"):
        kv_cache_accept(cache, k.clone().requires_grad_(), v, path, table, held)
    with pytest.raises(RuntimeError, match="no backward"):
        kv_cache_read(cache, k.clone().requires_grad_(), v, table, held)
    assert isinstance(tree, DraftTree)


def test_pools_beyond_4_gib():
    """Pages whose offsets pass 32 bits, at the pool's both ends: what a small pool gives."""
    from ring_swa import KVCache, kv_cache_accept, kv_cache_append, kv_cache_read

    pages = (5 << 30) // (8 * 64 * 128)
    pools = (KVCache.empty(pages, 8, 128, device="cuda"), ints([[pages - 1, 0, pages - 2], [1, pages - 3, 2]])), \
        (KVCache.empty(6, 8, 128, device="cuda"), ints([[0, 1, 2], [3, 4, 5]]))
    parents = [some_parents(random.Random(b), 40, 7) for b in range(2)]
    tree = tree_tensors(parents, False)
    path = ints([[0, 5, 30, -1], [0, 1, 2, 39]])
    results = []
    for cache, table in pools:
        g = torch.Generator().manual_seed(10)
        kv_cache_append(cache, *(randn(g, torch.bfloat16, 2, 126, 8, 128) for _ in range(2)), table, ints([0, 0]))
        q, (k, v) = randn(g, torch.bfloat16, 2, 40, 32, 128), (randn(g, torch.bfloat16, 2, 40, 8, 128) for _ in range(2))
        out, lse = attend((q, k, v, tree, cache, table, ints([126, 126]), -1, None, 0), return_lse=True)
        kv_cache_accept(cache, k, v, path, table, ints([126, 126]))
        back = [torch.empty(2, 129, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        kv_cache_read(cache, *back, table, ints([0, 0]))
        results.append((out, lse, *back))
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_a_tree_with_room_for_more_nodes():
    from ring_swa import draft_tree, verify_drafts

    args, parents = tree_case(3)
    q, k, v, tree, cache, table, lens, window, cu, sinks = args
    wide = draft_tree(tree.parents, max_nodes=1000)
    assert wide.ancestors.shape == (1, 32, 16) and bool((wide.ancestors[..., 1:] == 0).all())
    assert torch.equal(wide.ancestors[..., :1], tree.ancestors)
    for x, y in zip(attend(args, return_lse=True), attend((q, k, v, wide, *args[4:]), return_lse=True)):
        assert (x - y).abs().max() <= 2.0 ** -7 * x.abs().max()  # (cut elsewhere: other sums, within a rounding of each)
    p = torch.rand(1, 32, 900, device="cuda")
    tokens, u = torch.randint(0, 900, (1, 32), device="cuda"), torch.rand(1, 32, device="cuda")
    for x, y in zip(verify_drafts(tree, tokens, p, p, u), verify_drafts(wide, tokens, p, p, u)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("native", [True, False])
def test_a_graph_that_has_saved_the_rows_notices_a_read(native, monkeypatch):
    from ring_swa import kv_cache_read, ring_sliding_window_attn
    from ring_swa.ops import kv_cache

    if not native:
        monkeypatch.setattr(kv_cache, "_calls", lambda *_: None)
    cache, table, lens, _ = make([100], 2, 64, 32, 77)
    k, v = (torch.empty(1, 100, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    first = torch.zeros_like(lens)
    kv_cache_read(cache, k, v, table, first)
    q = torch.randn(1, 100, 4, 64, device="cuda").bfloat16().requires_grad_()
    ring_sliding_window_attn(q, k, v, 50).float().sum().backward()
    out = ring_sliding_window_attn(q, k, v, 50)
    kv_cache_read(cache, k, v, table, first)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.float().sum().backward()
    with torch.inference_mode():
        k, v = (torch.empty(1, 100, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        kv_cache_read(cache, k, v, table, first)
    kv_cache_read(cache, k, v, table, first)


@pytest.mark.parametrize("nodes,vocab", [(8, 70000), (9, 65536), (9, 65535), (24, 65537), (24, 131072),
                                         (24, 32768), (24, 32769), (24, 16385), (24, 16384), (9, 8191)])
def test_verification_over_large_vocabularies(nodes, vocab):
    """(Passes of several launches from 65536 tokens and 9 nodes on; rows held in registers up to 32768.)  All siblings of the root, most of them rejected."""
    from ring_swa import verify_drafts

    g = torch.Generator().manual_seed(nodes + vocab)
    batch = 6
    parents = [[-1] + [0] * (nodes - 3) + [1, 2]] * batch
    tree = tree_tensors(parents, False)
    p, q = (t.view(batch, nodes, vocab).cuda() for t in probabilities(g, batch * nodes, vocab, torch.float32, 1.0))
    # drafts that the target likes less than the draft does, which are all rejected, and of the last sequences what it draws
    tokens = (q / p).topk(nodes, -1).indices[:, 0].contiguous()
    for b in range(3, batch):
        tokens[b] = torch.tensor(drawn(random.Random(b + vocab), parents[b], q[b].cpu()))
    u = torch.rand(batch, nodes, generator=g)
    u[0] = 0.9999
    path, accepted, token = verify_drafts(tree, tokens, p, q, u.cuda())
    counts = set()
    for b in range(batch):
        want = R.verify(parents[b], tokens[b].tolist(), p[b].cpu(), q[b].cpu(), u[b].tolist())
        assert path[b, :int(accepted[b])].tolist() == want[0] and int(token[b]) == want[1], b
        counts.add(want[0][1] if len(want[0]) > 1 else 0)
    assert 0 in counts and len(counts) > 1  # (some with all rejected, some not)


# ---- packs that begin behind the first row (cu_seqlens[0] > 0) -----------------------------------
AHEAD = 37  # rows that are no sequence's, ahead of the first


def behind(t, fill):
    return torch.cat((t.new_full((AHEAD, *t.shape[1:]), fill), t))


@pytest.mark.parametrize("case", [8, 9, 10, 13, 16, 20])
def test_attention_of_packs_from_a_later_row(case):
    from ring_swa import DraftTree, draft_tree

    args, parents = tree_case(case)
    q, k, v, tree, cache, table, lens, window, cu, sinks = args
    later = DraftTree(behind(tree[0], 0), behind(tree[1], 5), behind(tree[2], -1))
    out, lse = attend((*(behind(t, math.nan) for t in (q, k, v)), later, cache, table, lens, window, cu + AHEAD, sinks),
                      return_lse=True)
    check_tree(args, parents, out[AHEAD:], lse[:, AHEAD:])
    most = max(map(len, parents))
    made = draft_tree(behind(ints([x for p in parents for x in p] + [-2, -2]), -1), cu + AHEAD, max_nodes=most)
    for mine, want in zip(made, tree):
        assert torch.equal(mine[AHEAD:-2], want[:-2])


@pytest.mark.parametrize("sampled", [True, False])
def test_the_other_calls_of_packs_from_a_later_row(sampled):
    from ring_swa import DraftTree, kv_cache_accept, kv_cache_read, verify_drafts

    sizes, vocab = [9, 1, 0, 70, 3, 64], 3001
    rng = random.Random(5)
    g = torch.Generator().manual_seed(5)
    parents = [some_parents(rng, n, 20, 0.02) for n in sizes]
    tree = tree_tensors(parents, True)
    p, q = (t.cuda() for t in probabilities(g, sum(sizes), vocab, torch.float32, 1.0))
    base = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    tokens = ints([x for b, own in enumerate(parents) for x in drawn(
        rng, [i if -1 <= i < n else -2 for n, i in enumerate(own)], q[base[b]:base[b + 1]].cpu())])
    u, cu = torch.rand(sum(sizes), generator=g).cuda(), ints(base)
    want = verify_drafts(tree, tokens, p, q if sampled else None, u, cu)
    later = DraftTree(behind(tree[0], -1), behind(tree[1], 0), behind(tree[2], 1))
    got = verify_drafts(later, behind(tokens, 0), behind(p, math.nan), behind(q, math.nan) if sampled else None,
                        behind(u, 0.0), cu + AHEAD)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert int(want[1].max()) > 1 or not sampled  # (tokens drawn from the draft: few are taken without it)

    held = [10, 0, 200, 77, 63, 64]
    k, v = (randn(g, torch.bfloat16, sum(sizes), 3, 64) for _ in range(2))
    made = [make([h + 70 for h in held], 3, 64, 32, 44, wild=False) for _ in range(2)]
    for (cache, table, _, _), ahead in zip(made, (0, AHEAD)):
        kv_cache_accept(cache, behind(k, math.nan)[AHEAD - ahead:], behind(v, math.inf)[AHEAD - ahead:], want[0], table,
                        ints(held), cu + ahead)
    assert O.same_bytes(made[0][0], made[1][0])
    cache, table, _, _ = made[0]
    rows = [torch.full((sum(sizes) + ahead, 3, 64), 7.0, dtype=torch.bfloat16, device="cuda") for ahead in (0, 0, AHEAD, AHEAD)]
    kv_cache_read(cache, *rows[:2], table, ints(held), cu)
    kv_cache_read(cache, *rows[2:], table, ints(held), cu + AHEAD)
    for mine, other in zip(rows[:2], rows[2:]):
        assert torch.equal(mine, other[AHEAD:]) and bool((other[:AHEAD] == 7).all())


@pytest.mark.parametrize("shape", [([0, 70, 500], 40, 4, 2), ([900, 64], 130, 8, 1), ([3000] * 8, 64, 16, 4)])
def test_bits_of_any_kind_say_who_sees_whom(shape, monkeypatch):
    """Ancestor bits that are no tree's (descendants, no node itself, nobody, nodes behind the last) and depths that are none's."""
    from ring_swa import DraftTree

    held, nodes, hq, hk = shape
    g = torch.Generator().manual_seed(nodes)
    words = (nodes + 63) // 64
    bits = torch.rand(len(held), nodes, 64 * words, generator=g) < 0.3
    bits[:, 3] = False
    depths = torch.randint(0, nodes, (len(held), nodes), generator=g, dtype=torch.int32)
    depths[:, 5] = -1
    weights = torch.ones(64, dtype=torch.int64) << torch.arange(64)
    packed = (bits.view(len(held), nodes, words, 64).long() * weights).sum(-1)
    cache, table, seqlens, _ = make(held, hk, 64, 32, 9, max_pages=max(held) // 32 + 1)
    q = randn(g, torch.bfloat16, len(held), nodes, hq, 64)
    k, v = (randn(g, torch.bfloat16, len(held), nodes, hk, 64) for _ in range(2))
    tree = DraftTree(depths.cuda(), depths.cuda(), packed.cuda())

    def seen(b, length, window, sinks, there):
        see = torch.cat((there.expand(nodes, length), bits[b, :, :nodes]), 1).clone()
        see[depths[b] < 0] = False
        return see

    monkeypatch.setattr(R, "seen", seen)
    args = (q, k, v, tree, cache, table, seqlens, -1, None, 0)
    out, lse = attend(args, return_lse=True)
    check_tree(args, list(range(len(held))), out, lse)


@pytest.mark.parametrize("sampled", [True, False])
def test_probabilities_beyond_2_to_31_elements(sampled):
    """The last sequences of a batch: what they give alone."""
    from ring_swa import DraftTree, verify_drafts

    batch, nodes, vocab = 34, 32, 1 << 21
    assert (batch - 2) * nodes * vocab >= 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(3)
    parents = [[-1] + [max(0, i - 3) for i in range(1, nodes)]] * batch
    tree = tree_tensors(parents, False)
    p = torch.zeros(batch, nodes, vocab, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros_like(p) if sampled else None
    for t in (p, q) if sampled else (p,):
        t[-2:] = torch.softmax(3 * torch.randn(2, nodes, vocab, generator=g, device="cuda"), -1).bfloat16()
    tokens = torch.randint(0, vocab, (batch, nodes), generator=g, device="cuda")
    tokens[-1, 1::2] = p[-1, 0].argmax()
    u = torch.rand(batch, nodes, generator=g, device="cuda")
    u[-1, 1:] = 0
    got = verify_drafts(tree, tokens, p, q, u)
    alone = verify_drafts(DraftTree(*(t[-2:] for t in tree)), tokens[-2:], p[-2:].clone(), q[-2:].clone() if sampled else None, u[-2:])
    assert all(torch.equal(a[-2:], b) for a, b in zip(got, alone))
    assert int(alone[1].max()) > 1 and int(alone[2].min()) >= 0
    assert got[1][:-2].tolist() == [1] * (batch - 2) and got[2][:-2].tolist() == [-1] * (batch - 2)  # (nothing in their rows)
