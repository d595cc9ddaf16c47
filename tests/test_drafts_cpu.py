"""The calls on drafted tokens without a GPU: layouts, names, refusals, compiled and traced programs, and the restatements
that the GPU's results are held to."""
import ctypes
import math
import random

import pytest
import torch

import ring_swa
from oracle import drafts_oracle as R
from oracle import kv_cache_oracle as O
from ring_swa import DraftTree, KVCache, _lib

NAMES = ["DraftTree", "draft_tree", "kv_cache_tree_attn", "verify_drafts", "kv_cache_accept", "kv_cache_read"]


def test_struct_layouts():
    L = _lib.lib()
    assert L.rswa_sizeof_tree_params() == ctypes.sizeof(_lib.TreeParams)
    assert L.rswa_sizeof_draft_params() == ctypes.sizeof(_lib.DraftParams)
    assert L.rswa_sizeof_verify_params() == ctypes.sizeof(_lib.VerifyParams)


def test_public_names():
    from ring_swa import ops

    for name in NAMES:
        assert name in ring_swa.__all__ and name in ops.__all__ and getattr(ring_swa, name) is getattr(ops, name)


def inputs(batch=2, nodes=3, vocab=11):
    cache = KVCache.empty(8, 2, 64, 16)
    for t in cache[:2]:
        t.view(torch.uint8).zero_()
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(batch, nodes, 8, 64, generator=g).bfloat16()
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32).expand(batch, nodes).contiguous()
    tree = DraftTree(parents, parents + 1, torch.tensor([1, 3, 5]).expand(batch, nodes).unsqueeze(-1).contiguous())
    return dict(cache=cache, q=rows[:, :, :4], k=rows[:, :, 4:6], v=rows[:, :, 6:], parents=parents, tree=tree,
                table=torch.arange(6, dtype=torch.int32).view(2, 3), lens=torch.tensor([9, 30], dtype=torch.int32),
                tokens=torch.randint(0, vocab, (batch, nodes), generator=g),
                target=torch.rand(batch, nodes, vocab, generator=g), draft=torch.rand(batch, nodes, vocab, generator=g),
                uniforms=torch.rand(batch, nodes, generator=g), path=torch.tensor([[0, 1], [0, -1]], dtype=torch.int32),
                cu=torch.tensor([0, 2, 3], dtype=torch.int32))


CALLS = {
    "draft_tree": lambda x, **kw: ring_swa.draft_tree(x["parents"], **kw),
    "cache_tree_attn": lambda x, **kw: ring_swa.kv_cache_tree_attn(x["q"], x["k"], x["v"], x["tree"], x["cache"], x["table"],
                                                                   x["lens"], **kw),
    "verify_drafts": lambda x, **kw: ring_swa.verify_drafts(x["tree"], x["tokens"], x["target"], x["draft"], x["uniforms"], **kw),
    "cache_accept": lambda x, **kw: ring_swa.kv_cache_accept(x["cache"], x["k"], x["v"], x["path"], x["table"], x["lens"], **kw),
    "cache_read": lambda x, **kw: ring_swa.kv_cache_read(x["cache"], x["k"], x["v"], x["table"], x["lens"], **kw),
}


@pytest.mark.parametrize("call", CALLS)
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="GPU"):
        CALLS[call](inputs())


@pytest.fixture
def on_cpu(monkeypatch):
    """The checks ahead of the launch, with tensors that live on the CPU; the launch itself is a failure."""
    monkeypatch.setattr(_lib, "require_device", lambda *t: t[0].device)

    def launch(*_):
        raise AssertionError("launched")

    monkeypatch.setattr(_lib, "launch", launch)


def refuses(call, _fine=False, _kw={}, **changed):
    with pytest.raises((AssertionError, NotImplementedError, ValueError)) as e:
        CALLS[call](dict(inputs(), **changed), **_kw)
    assert ("launched" in str(e.value)) == _fine, e.value


def packed(x):
    """The inputs' first sequence as a pack of two."""
    return {n: (DraftTree(*(t[0] for t in x[n])) if n == "tree" else x[n][0])
            for n in ("q", "k", "v", "parents", "tree", "tokens", "target", "draft", "uniforms")}


def test_shapes_and_types_are_checked(on_cpu):
    x = inputs()
    cu = dict(cu_seqlens=x["cu"])
    for call in CALLS:
        refuses(call, True)
        refuses(call, True, {**cu, "max_nodes": 2} if call == "draft_tree" else cu, **packed(x))
        refuses(call, **packed(x))                                     # packed without cu_seqlens
        refuses(call, False, {**cu, "max_nodes": 2} if call == "draft_tree" else cu)
        refuses(call, False, {"cu_seqlens": x["cu"].long(), **({"max_nodes": 2} if call == "draft_tree" else {})}, **packed(x))
    refuses("draft_tree", False, cu, **packed(x))                      # no max_nodes
    refuses("draft_tree", False, {"max_nodes": 2})
    refuses("draft_tree", False, {"max_nodes": 1025})
    refuses("draft_tree", False, {"max_nodes": 0})
    refuses("draft_tree", parents=x["parents"].long())
    refuses("draft_tree", parents=x["parents"].t().contiguous().t())
    refuses("draft_tree", parents=torch.zeros(1, 1025, dtype=torch.int32))

    t = x["tree"]
    for call, names in (("cache_tree_attn", "qkv"), ("cache_accept", "kv"), ("cache_read", "kv")):
        for n in names:
            refuses(call, **{n: x[n].half()})
            refuses(call, **{n: x[n].float()})
            refuses(call, **{n: x[n][..., :32]})
            refuses(call, **{n: x[n][:1]})
            refuses(call, **{n: x[n][:, :2]})
            refuses(call, **{n: torch.cat((x[n], x[n][:, :, :1]), 2)})
            refuses(call, **{n: torch.stack((x[n], x[n]), -1)[..., 0]})
        refuses(call, table=x["table"].long())
        refuses(call, lens=x["lens"].long())
        refuses(call, cache=x["cache"]._replace(k=x["cache"].k.view(torch.uint8)))
    refuses("cache_tree_attn", tree=t._replace(depths=t.depths.long()))
    refuses("cache_tree_attn", tree=t._replace(depths=t.depths[:, :2]))
    refuses("cache_tree_attn", tree=t._replace(ancestors=t.ancestors.int()))
    refuses("cache_tree_attn", tree=t._replace(ancestors=t.ancestors[..., 0]))
    refuses("cache_tree_attn", tree=t._replace(ancestors=t.ancestors[:, :2]))
    refuses("cache_tree_attn", tree=t._replace(ancestors=torch.zeros(2, 3, 17, dtype=torch.int64)))
    refuses("cache_tree_attn", tree=t._replace(ancestors=torch.zeros(2, 3, 0, dtype=torch.int64)))
    refuses("cache_tree_attn", tree=t._replace(ancestors=torch.zeros(2, 3, 2, dtype=torch.int64)[..., :1]))
    refuses("cache_tree_attn", False, {"num_sink_tokens": -1})
    refuses("cache_accept", path=x["path"].long())
    refuses("cache_accept", path=x["path"][:1])
    refuses("cache_accept", path=x["path"][0])
    refuses("cache_accept", path=x["path"].t().contiguous().t())
    refuses("cache_read", k=x["k"][:, :1].expand(2, 3, 2, 64))         # rows that are one another's
    refuses("cache_read", v=x["v"][:, :, :1].expand(2, 3, 2, 64))

    refuses("verify_drafts", True, draft=None)
    refuses("verify_drafts", True, tokens=x["tokens"].int())
    refuses("verify_drafts", True, target=x["target"].half(), draft=x["draft"].half())
    refuses("verify_drafts", target=x["target"].half())
    refuses("verify_drafts", draft=x["draft"].half())
    refuses("verify_drafts", draft=x["draft"][..., :10])
    refuses("verify_drafts", target=x["target"].double(), draft=x["draft"].double())
    refuses("verify_drafts", target=x["target"].transpose(1, 2).contiguous().transpose(1, 2))
    refuses("verify_drafts", target=x["target"][..., :0], draft=x["draft"][..., :0])
    refuses("verify_drafts", tokens=x["tokens"].float())
    refuses("verify_drafts", tokens=x["tokens"][:, :2])
    refuses("verify_drafts", uniforms=x["uniforms"].double())
    refuses("verify_drafts", uniforms=x["uniforms"].t().contiguous().t())
    refuses("verify_drafts", tree=t._replace(parents=t.parents.long()))
    refuses("verify_drafts", tree=t._replace(ancestors=torch.zeros(2, 3, 17, dtype=torch.int64)))


DERIVED = [("cache_tree_attn", n) for n in "qkv"] + [("verify_drafts", n) for n in ("target", "draft", "uniforms")] + [
    (call, n) for call in ("cache_accept", "cache_read") for n in "kv"]


@pytest.mark.parametrize("call,name", DERIVED)
def test_derivatives_are_refused(call, name, monkeypatch):
    from torch.autograd import forward_ad

    monkeypatch.setattr(_lib, "require_device", lambda *t: t[0].device)
    monkeypatch.setattr(_lib, "launch", lambda *_: None)
    x = inputs()
    x[name] = x[name].detach().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        CALLS[call](x)
    with torch.no_grad():
        CALLS[call](x)
    with forward_ad.dual_level():
        x[name] = forward_ad.make_dual(x[name].detach(), torch.ones_like(x[name]))
        with pytest.raises(RuntimeError, match="no forward derivative"):
            CALLS[call](x)


# ---- the library's own refusals -----------------------------------------------------------------
def filled(p, fill):
    for name, value in fill.items():
        at = p
        while "." in name:
            head, name = name.split(".", 1)
            at = getattr(at, head)
        if isinstance(value, tuple):
            getattr(at, name)[:] = value
        else:
            setattr(at, name, value)
    return p


def params(call, fill):
    """A call's parameters that nothing is wrong with, but for ``fill`` (no launch is made without a refusal: sizes of 0)."""
    if call == "draft_tree":
        p = _lib.TreeParams(batch=2, nodes=3, max_nodes=3, parents=4096, tree_parents=4096, depths=4096, ancestors=4096)
        return filled(p, fill)
    if call == "verify_drafts":
        p = _lib.VerifyParams(dtype=2, token_bytes=4, batch=2, nodes=3, max_nodes=64, vocab=100, path_len=3)
        for name in ("parents", "tokens", "uniforms", "target", "draft", "path", "accepted", "next_token", "workspace"):
            setattr(p, name, 4096)
        p.workspace_bytes = 1 << 40
        return filled(p, fill)
    c = _lib.CacheParams(dtype=0, head_dim=128, batch=2, heads_q=4, heads_kv=2, page_size=64, num_pages=8, max_pages=3,
                         seqlen_q=3, softmax_scale=0.1, window_left=-1)
    for name in ("k", "v", "k_scale", "v_scale", "page_table", "seqlens", "q", "out", "new_k", "new_v"):
        setattr(c, name, 4096)
    c.workspace, c.workspace_bytes = 4096, 1 << 40
    if call == "cache_read":
        return filled(c, {n.replace("cache.", ""): v for n, v in fill.items()})
    p = _lib.DraftParams(cache=c, depths=4096, ancestors=4096, words=1, path=4096, path_len=2)
    return filled(p, fill)


CACHED = ["cache_tree_attn", "cache_accept", "cache_read"]


@pytest.mark.parametrize("call,fill,status", [
    *[(c, {"cache." + n: v}, s) for c in CACHED for n, v, s in (
        ("dtype", 2, -2), ("head_dim", 96, -2), ("page_size", 48, -2), ("heads_kv", 0, -1), ("batch", -1, -1),
        ("max_pages", 1 << 22, -2), ("k", None, -1), ("v_scale", None, -1), ("seqlens", None, -1), ("page_table", None, -1),
        ("k", 4100, -2), ("v_stride", (8, 16), -2), ("num_pages", 0, -1), ("new_k", None, -1), ("new_v", 4104, -2),
        ("new_k_stride", (0, 4, 8), -2), ("new_v_stride", (8, 8, 1), -2))],
    *[("cache_tree_attn", f, s) for f, s in (
        ({"cache.heads_q": 5}, -1), ({"cache.q": None}, -1), ({"cache.out": None}, -1), ({"cache.out": 4104}, -2),
        ({"cache.q_stride": (8, 8, 4)}, -2), ({"cache.softmax_scale": 0.0}, -1), ({"cache.softmax_scale": math.inf}, -1),
        ({"cache.num_sink": -1}, -1), ({"words": 0}, -2), ({"words": 17}, -2), ({"cache.seqlen_q": 65}, -1),
        ({"depths": None}, -1), ({"ancestors": None}, -1), ({"cache.max_pages": 4000, "cache.workspace": None}, -1),
        ({"cache.max_pages": 4000, "cache.workspace_bytes": 100}, -1), ({"cache.batch": 1 << 20}, -2))],
    *[("cache_accept", f, s) for f, s in (({"path": None}, -1), ({"path_len": -1}, -1), ({"path_len": (1 << 31) - 1, "cache.batch": 1 << 10}, -2))],
    *[("draft_tree", f, s) for f, s in (
        ({"batch": -1}, -1), ({"nodes": -1}, -1), ({"max_nodes": 0}, -2), ({"max_nodes": 1025}, -2), ({"max_nodes": 2}, -1),
        ({"parents": None}, -1), ({"tree_parents": None}, -1), ({"depths": None}, -1), ({"ancestors": None}, -1),
        ({"batch": (1 << 20) + 1}, -2))],
    *[("verify_drafts", f, s) for f, s in (
        ({"dtype": 3}, -2), ({"token_bytes": 2}, -2), ({"batch": -1}, -1), ({"nodes": -1}, -1), ({"vocab": 0}, -1),
        ({"vocab": (1 << 24) + 1}, -2), ({"max_nodes": 0}, -2), ({"max_nodes": 1025}, -2), ({"max_nodes": 2}, -1),
        ({"path_len": 2}, -1), ({"cu_seqlens": 4096, "total": 6}, -1), ({"batch": 1 << 16}, -2), ({"parents": None}, -1),
        ({"tokens": None}, -1), ({"uniforms": None}, -1), ({"target": None}, -1), ({"path": None}, -1),
        ({"accepted": None}, -1), ({"next_token": None}, -1), ({"workspace": None}, -1), ({"workspace": 4100}, -1),
        ({"workspace_bytes": 8}, -1))],
])
def test_every_call_refuses(call, fill, status):
    L = _lib.lib()
    p = params(call, fill)
    assert getattr(L, "rswa_" + call)(p, None) == status, L.rswa_last_error()
    assert call.encode() in L.rswa_last_error()


def test_null_parameters():
    L = _lib.lib()
    for call in CALLS:
        assert getattr(L, "rswa_" + call)(None, None) == -1
    assert L.rswa_cache_tree_attn_workspace_bytes(None) == L.rswa_verify_drafts_workspace_bytes(None) == 0


@pytest.mark.parametrize("call,fill", [
    ("draft_tree", {"batch": 0}), ("draft_tree", {"nodes": 0}), ("verify_drafts", {"batch": 0}),
    ("cache_accept", {"path_len": 0}), ("cache_accept", {"cache.max_pages": 0}), *[(c, {"cache.batch": 0}) for c in CACHED],
    *[(c, {"cache.seqlen_q": 0}) for c in CACHED]])
def test_nothing_to_do_is_no_error(call, fill):
    assert getattr(_lib.lib(), "rswa_" + call)(params(call, fill), None) == 0


# ---- compiled and traced programs ---------------------------------------------------------------
@pytest.fixture
def launches(monkeypatch):
    """Names of the entry points launched; the stub writes to each call's results and to what it changes in place."""
    names = []

    def launch(_, entry, p):
        name = entry.__name__[len("rswa_"):]
        names.append(name)
        if name == "draft_tree":
            rows = p.batch * p.nodes
            for at, size in ((p.tree_parents, 4), (p.depths, 4), (p.ancestors, 8)):
                ctypes.memset(at, size, size * rows)
        elif name == "cache_tree_attn":
            c = p.cache
            ctypes.memset(c.out, 0x3C, 2 * c.batch * c.seqlen_q * c.heads_q * c.head_dim)
            if c.lse:
                ctypes.memset(c.lse, 0x40, 4 * c.batch * c.seqlen_q * c.heads_q)
        elif name == "verify_drafts":
            ctypes.memset(p.path, 1, 4 * p.batch * p.path_len)
            ctypes.memset(p.accepted, 2, 4 * p.batch)
            ctypes.memset(p.next_token, 3, p.token_bytes * p.batch)
        elif name == "cache_accept":
            ctypes.memset(p.cache.k, 0x38, p.cache.head_dim)
            ctypes.memset(p.cache.v_scale, 0x7F, 1)
        else:
            ctypes.memset(p.new_k, 0x3D, 2 * p.head_dim)
            ctypes.memset(p.new_v, 0x3E, 2 * p.head_dim)

    monkeypatch.setattr(_lib, "require_device", lambda *t: t[0].device)
    monkeypatch.setattr(_lib, "launch", launch)
    return names


FIELDS = ["q", "k", "v", "parents", "table", "lens", "tokens", "target", "draft", "uniforms", "path"]


def flat():
    x = inputs()
    x.update({n: x[n].contiguous() for n in "qkv"})
    return (*x["cache"], *x["tree"], *(x[n] for n in FIELDS))


def program(call, **kw):
    def run(k, v, k_scale, v_scale, up, depths, ancestors, *rest):
        x = dict(zip(FIELDS, rest), cache=KVCache(k, v, k_scale, v_scale), tree=DraftTree(up, depths, ancestors))
        got = CALLS[call](x, **kw)
        if got is None:
            return x["k"] + 1
        return tuple(t + 1 for t in (got if isinstance(got, tuple) else (got,)))

    return run


def check(call, run, names):
    mine, want = flat(), flat()
    names.clear()
    results = run(*mine)
    assert names == [call]
    for x, y in zip((*results, *mine) if isinstance(results, tuple) else (results, *mine), _both(program(call)(*want), want)):
        assert x.dtype == y.dtype and torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


def _both(results, args):
    return (*results, *args) if isinstance(results, tuple) else (results, *args)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("call", CALLS)
def test_compiled(call, backend, launches):
    torch._dynamo.reset()
    run = torch.compile(program(call), backend=backend)
    for _ in range(2):
        check(call, run, launches)


@pytest.mark.parametrize("call", CALLS)
def test_traced(call, launches):
    from torch.fx.experimental.proxy_tensor import make_fx

    run = torch.jit.trace(program(call), flat(), check_trace=False)
    assert "ring_swa::" + call in str(run.graph)
    check(call, run, launches)
    for mode in ("real", "fake"):
        check(call, make_fx(program(call), tracing_mode=mode)(*flat()), launches)


# ---- the restatements ---------------------------------------------------------------------------
def test_the_restated_tree():
    assert R.tree([-1, 0, 0, 2, 4, 4, -1, 9, 7, -3], 6) == (
        [-1, 0, 0, 2, -2, -2, -2, -2, -2, -2], [0, 1, 1, 2] + [-1] * 6, [[1], [3], [5], [13]] + [[0]] * 6)
    got = R.tree(list(range(-1, 127)), 128)
    assert got[1] == list(range(128)) and got[2][127] == [-1, -1] and got[2][64] == [-1, 1]
    see = R.seen([-1, 0, 1], 4, 2, 1, torch.tensor([True, True, False, True]))
    assert see.tolist() == [[True, False, False, True, True, False, False], [True, False, False, True, True, True, False],
                            [True, False, False, False, True, True, True]]


@pytest.mark.parametrize("sampled", [True, False])
def test_the_restated_choice_has_the_targets_distribution(sampled):
    """Exactly, by the formula: with the uniforms' lengths in the place of draws the probability of each token of the first
    choice is the target's.  Three children, drawn independently from q or named outright."""
    p = torch.tensor([0.1, 0.4, 0.05, 0.25, 0.2], dtype=torch.float64)
    q = torch.tensor([0.3, 0.1, 0.2, 0.15, 0.25], dtype=torch.float64)
    found = torch.zeros(5, dtype=torch.float64)
    tokens = [(i, j, k) for i in range(5) for j in range(5) for k in range(5)] if sampled else [(4, 1, 2)]
    for drafts in tokens:
        chance = math.prod(float(q[t]) for t in drafts) if sampled else 1.0
        left, mass, a = p.clone(), 1.0, 0.0
        for x in drafts:
            take = float(min(1.0, left[x] / (mass * q[x]))) if sampled else float(left[x]) / mass
            found[x] += chance * take
            chance *= 1 - take
            if sampled:
                a += mass
                left = torch.clamp(p - a * q, min=0)
                mass = float(left.sum())
            else:
                mass -= float(left[x])
                left[x] = 0
            if chance < 1e-15:
                break
        else:
            found += chance * left / left.sum()
    assert bool(((found - p).abs() < 1e-12).all())


def test_the_restated_choice_follows_the_formula_step_by_step():
    """``R.verify`` against residuals that are written out and normalised after every rejection."""
    rng = random.Random(3)
    g = torch.Generator().manual_seed(3)
    for trial in range(200):
        n, vocab = rng.randint(1, 12), rng.randint(1, 9)
        parents = [-1] + [rng.randrange(0, i) for i in range(1, n)]
        p, q = (torch.softmax(torch.randn(n, vocab, generator=g, dtype=torch.float64), -1) for _ in range(2))
        tokens = [rng.randrange(vocab) for _ in range(n)]
        u = [rng.random() for _ in range(n)]
        cur, path, left = 0, [0], p[0]
        for i in range(1, n):
            if parents[i] != cur:
                continue
            x = tokens[i]
            if u[i] * q[cur, x] < left[x]:
                cur, left = i, p[i]
                path.append(i)
            else:
                left = torch.clamp(left - q[cur], min=0)
                left = left / left.sum()
        token = int((left.cumsum(0) > u[0]).nonzero()[0])
        assert R.verify(parents, tokens, p, q, u) == (path, token)


def test_the_restated_read_and_accept():
    cache = KVCache.empty(4, 2, 64, 16)
    for t in cache[:2]:
        t.view(torch.uint8).zero_()
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randint(-8, 9, (1, 20, 2, 64), generator=g) / 4 for _ in range(2))
    table, lens = torch.tensor([[2, 0, 3]], dtype=torch.int32), torch.tensor([5], dtype=torch.int32)
    after = R.accept(cache, k.bfloat16(), v.bfloat16(), torch.tensor([[3, 7, 7, 0, 20, 1]]), table, lens)
    got = R.read(after, table, torch.tensor([5]), [4])[0]
    for x, y in zip((k, v), got):
        assert torch.equal(x[0, [3, 7, 7, 0]].double(), y)
    beyond = R.read(after, table, torch.tensor([40]), [30])[0]
    assert all(bool((y == 0).all()) for y in beyond)
    assert O.same_bytes(R.accept(cache, k, v, torch.tensor([[-1, 3]]), table, lens), cache)
