"""Packs whose first sequence begins behind the first row of the tensors (cu_seqlens[0] > 0): the results of the same
pack from its first row on.  Bounds as in the other tests of the attention."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CASES = [
    # cu_seqlens, rows, q heads, kv heads, dim, window, sinks
    ([300, 700, 1001], 1100, 4, 2, 64, 128, 0),
    ([2000, 2300, 4000], 4096, 8, 2, 128, 500, 0),
    ([900, 900, 1500, 1501], 1600, 4, 4, 128, 100, 4),
    ([5000, 9000], 9000, 8, 8, 128, 1024, 1),
    ([700 + 20 * i for i in range(90)], 2600, 4, 1, 64, 64, 0),
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward_and_backward(case):
    from ring_swa import ring_sliding_window_attn_varlen, ring_streaming_llm_attn_varlen

    cu, rows, hq, hk, dim, window, sinks = CASES[case]
    g = torch.Generator().manual_seed(case)
    at, end = cu[0], cu[-1]
    shapes = ((rows, hq, dim), (rows, hk, dim), (rows, hk, dim), (rows, hq, dim))
    q, k, v, do = (torch.randn(*s, generator=g).bfloat16().cuda() for s in shapes)

    def run(lo, offsets):
        leaves = [t[lo:end].clone().requires_grad_() for t in (q, k, v)]
        offsets = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        if sinks:
            out = ring_streaming_llm_attn_varlen(*leaves, window, offsets, num_sink_tokens=sinks)
        else:
            out = ring_sliding_window_attn_varlen(*leaves, window, offsets)
        grads = torch.autograd.grad(out, leaves, do[lo:end])
        return [t[at - lo:].float() for t in (out, *grads)]

    want = run(at, [x - at for x in cu])
    got = run(0, cu)
    assert (got[0] - want[0]).abs().max() <= 2e-2
    for x, y in zip(got[1:], want[1:]):
        assert (x - y).norm() <= 1e-2 * y.norm()
