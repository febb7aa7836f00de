"""How the product kernels end: nothing of a launch reaches the shared memory of the next one, and a launch whose waits ran out, or
that starts while the status word is raised, leaves its outputs alone.  In forms that neither fault nor hang a GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device="cuda")


def bits(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def test_short_launches_one_behind_the_other():
    """Products of one K block and of a ring's worth of them, in CTA pairs and in clusters, back to back without a gap: each starts on
    SMs that the one before has just left, with barriers where the other had its own.  Every result keeps its bits."""
    from come_b200 import _lib
    from come_b200.block_scaled import block_scaled_gated_linear, block_scaled_linear, quantize_rows, quantize_weight
    from come_b200.feed_forward import gated_linear
    randn = gen(1)
    calls = []

    def step(*tensors):
        leaves = [t.detach().requires_grad_(True) for t in tensors[:3]]
        return list(torch.autograd.grad(gated_linear(*leaves), leaves, tensors[3]))

    for T, K, F in ((5003, 64, 1010), (5003, 128, 1010), (4700, 776, 520), (3, 128, 200), (130, 1024, 512)):
        x, wg, wu = randn(T, K), randn(F, K) / 8, randn(F, K) / 8
        x8, g8, u8 = quantize_rows(x), quantize_weight(wg), quantize_weight(wu)
        xb, gb, ub, dh = (t.bfloat16() for t in (x, wg, wu, randn(T, F)))
        calls += [lambda x8=x8, g8=g8: [block_scaled_linear(x8, g8)],
                  lambda x8=x8, g8=g8, u8=u8: list(block_scaled_gated_linear(x8, g8, u8)),
                  lambda xb=xb, gb=gb, ub=ub: [gated_linear(xb, gb, ub)],
                  lambda xb=xb, gb=gb, ub=ub, dh=dh: step(xb, gb, ub, dh)]
    want = []
    for call in calls:
        want.append(call())
        torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()  # launches from a graph follow each other without the host between them
    with torch.cuda.graph(graph):
        got = [[call() for call in calls] for _ in range(4)]
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    for round_ in got:
        for results, first in zip(round_, want):
            assert all(torch.equal(bits(a), bits(b)) for a, b in zip(results, first))
    assert _lib.device_status(clear=True) == 0
