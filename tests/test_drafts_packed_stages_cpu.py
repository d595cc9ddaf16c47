"""Packed drafts are verified by the launches that the same drafts take in rows of one length (the scratch says which)."""
import pytest

from ring_swa import _lib

P = 4096  # (no launch is made: an address is all that is asked for)


def scratch(batch, nodes, vocab, packed, draft=True):
    p = _lib.VerifyParams(dtype=2, token_bytes=4, batch=batch, vocab=vocab, draft=P if draft else None)
    if packed:  # (max_nodes as the calls have it: that of whole words of ancestors)
        p.total, p.cu_seqlens, p.max_nodes = batch * nodes, P, (nodes + 63) // 64 * 64
    else:
        p.nodes = p.max_nodes = nodes
    return _lib.lib().rswa_verify_drafts_workspace_bytes(p)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("vocab", [1000, 65535, 65536, 131072])
@pytest.mark.parametrize("batch,nodes", [(1, 1), (1, 6), (8, 8), (8, 9), (3, 64), (2, 65), (64, 32)])
def test_packed_as_dense(batch, nodes, vocab, draft):
    assert scratch(batch, nodes, vocab, True, draft) == scratch(batch, nodes, vocab, False, draft) > 0


def test_a_pack_goes_by_its_mean():
    L = _lib.lib()
    p = _lib.VerifyParams(dtype=2, token_bytes=4, batch=4, vocab=131072, draft=P, cu_seqlens=P, max_nodes=64)
    sizes = {}
    for total in (0, 1, 32, 33, 256, (1 << 31) - 1):
        p.total = total
        sizes[total] = L.rswa_verify_drafts_workspace_bytes(p)
    assert sizes[0] == sizes[1] == sizes[32] and sizes[33] == sizes[256] == sizes[(1 << 31) - 1] == 4 * sizes[32]
