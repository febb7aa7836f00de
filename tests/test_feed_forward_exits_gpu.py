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


# tokens, features, channels, and how many K blocks of 16- and 8-bit operands a CTA has (per tile, where it has several)
SPLIT, PAIR = (130, 192, 1024), (5000, 1008, 1024)


def stall(x, w, v, k_blocks, ctas, out, out_scale=None, ticks=1 << 20):
    from come_b200 import _lib
    st = torch.cuda.current_stream().cuda_stream
    (T, K), F = x[0].shape, w[0].shape[0]
    assert all(t[0].is_contiguous() and (t[1] is None or t[1].is_contiguous()) for t in (x, w, v))
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    _lib.check(_lib.lib().come_selftest_matmul_stall(ptr(x[0]), ptr(x[1]), ptr(w[0]), ptr(v[0]), ptr(w[1]), T, F, K, k_blocks, ctas, ticks, ptr(out), ptr(out_scale), st))


def operands(form, T, F, K):
    from come_b200.block_scaled import quantize_rows, quantize_weight
    randn = gen(T)
    x, w, v = randn(T, K), randn(F, K) / K ** 0.5, randn(F, K) / K ** 0.5
    if form == "16":
        return tuple((t.bfloat16(), None) for t in (x, w, v))
    x8, w8, v8 = quantize_rows(x), quantize_weight(w), quantize_weight(v)
    return (x8.data, x8.scale.contiguous()), (w8.data, w8.scale), (v8.data, w8.scale)  # one scale tensor for both weights


def product(form, x, w, v):
    from come_b200.block_scaled import BlockScaled, block_scaled_gated_linear
    from come_b200.feed_forward import gated_linear
    if form == "16":
        return gated_linear(x[0], w[0], v[0])
    got = block_scaled_gated_linear(BlockScaled(*x), BlockScaled(*w), BlockScaled(*v), out_dtype=torch.bfloat16 if form == "8 to 16" else None)
    return got if form == "8 to 16" else (got.data.view(torch.uint8), got.scale)


@pytest.mark.parametrize("form", ["16", "8 to 16", "8 to 8"])
@pytest.mark.parametrize("sizes,ctas,k_blocks", [(SPLIT, 0xff, 0), (SPLIT, 1, 0), (SPLIT, 0x80, 1), (SPLIT, 4, 1), (SPLIT, 0xff, 99),
                                                 (PAIR, 3, 0), (PAIR, 1, 1), (PAIR, 2, 1), (PAIR, 1, 5), (PAIR, 2, 7), (PAIR, 3, 8), (PAIR, 2, 15), (PAIR, 1, 16), (PAIR, 2, 17),
                                                 (PAIR, 3, 31), (PAIR, 3, 99)])
def test_a_product_whose_waits_run_out_leaves_tiles_right_or_untouched(sizes, ctas, k_blocks, form):
    """Loads withheld by one CTA of a cluster or by all, in front of the first block, inside a tile, at its end and in a later tile; a CTA
    of the 130 rows has two blocks of 16-bit operands or one of 8-bit ones, a pair of the 5000 two or three tiles of 16 or 8."""
    from come_b200 import _lib
    T, F, K = sizes
    x, w, v = operands(form, T, F, K)
    assert _lib.device_status(clear=True) == 0
    want = product(form, x, w, v)
    eight = form == "8 to 8"
    out = torch.full((T, F), 0x7f if eight else 7.0, dtype=torch.uint8 if eight else torch.bfloat16, device="cuda")  # 0x7f: NaN, which no result is
    scale = torch.full((T, -(-F // 128)), 7.0, device="cuda") if eight else None
    try:
        stall(x, w, v, k_blocks, ctas, out, scale)
        torch.cuda.synchronize()  # the kernel returned by itself
        status = _lib.device_status(clear=False)
        per_tile = (16 if form == "16" else 8) // (8 if sizes is SPLIT else 1)
        stalls = k_blocks < per_tile * (1 if sizes is SPLIT else 3)
        assert (status != 0) == stalls and status & ~0x380000 == 0, hex(status)
        if stalls:
            with pytest.raises(RuntimeError, match="product kernel"):
                _lib.raise_on_device_error(clear=False)
    finally:
        _lib.device_status(clear=True)
    values, blank = (want[0], 0x7f) if eight else (want, 7.0)
    rows = 128 if sizes is SPLIT else 256
    tiles = [(slice(r, r + rows), slice(c, c + 128)) for r in range(0, T, rows) for c in range(0, F, 128)]
    right, untouched = [torch.equal(out[t], values[t]) for t in tiles], [bool((out[t] == blank).all()) for t in tiles]
    assert all(r or u for r, u in zip(right, untouched)) and any(untouched) == stalls
    assert any(right) == (not stalls or (sizes is PAIR and k_blocks >= per_tile))
    if eight:
        block = torch.stack([(out[:, c: c + 128] == blank).all(1) for c in range(0, F, 128)], 1)
        assert bool(torch.where(block, scale == 7.0, scale == want[1]).all())
    again = product(form, x, w, v)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1]) if eight else torch.equal(again, want)
    assert _lib.device_status(clear=True) == 0


def raise_status():
    """Leaves bits of the product kernels in the status word."""
    from come_b200 import _lib
    x, w, v = operands("16", 130, 192, 128)
    stall(x, w, v, 0, 1, torch.empty(130, 192, dtype=torch.bfloat16, device="cuda"))
    assert _lib.device_status(clear=False) & 0x380000


@pytest.mark.parametrize("T,K,F", [(3, 128, 200), (130, 256, 192), (5003, 128, 1010)])
def test_products_leave_their_outputs_alone_while_the_status_word_is_raised(T, K, F):
    from come_b200 import _lib
    from come_b200.block_scaled import quantize_rows, quantize_weight
    lib, randn, st = _lib.lib(), gen(5), torch.cuda.current_stream().cuda_stream
    assert _lib.device_status(clear=True) == 0
    x, wg, wu = randn(T, K), randn(F, K) / 8, randn(F, K) / 8
    x8, g8, u8 = quantize_rows(x), quantize_weight(wg), quantize_weight(wu)
    xb, gb, ub, dh = (t.bfloat16() for t in (x, wg, wu, randn(T, F)))
    xa = (x8.data.data_ptr(), x8.data.stride(0), x8.scale.data_ptr(), *x8.scale.stride())
    ga, ua = ((t.data.data_ptr(), t.data.stride(0), t.scale.data_ptr(), t.scale.stride(0)) for t in (g8, u8))
    wide = (xb.data_ptr(), K, gb.data_ptr(), K, ub.data_ptr(), K, None, None, _lib.COME_BF16, 0, T, F, K)
    made = []

    def full(*shape, dtype=torch.bfloat16):
        made.append(torch.full(shape, 7, dtype=dtype, device="cuda"))
        return made[-1].data_ptr()

    stride = -(-F // 16) * 16

    def run():
        made.clear()
        _lib.check(lib.come_matmul_e4m3(*xa, *ga, None, T, F, K, full(T, F, dtype=torch.float32), F, _lib.COME_F32, st))
        _lib.check(lib.come_gated_matmul_e4m3(*xa, *ga, *ua, None, None, 0, T, F, K, full(T, F), F, _lib.COME_BF16, None, 0, 0, st))
        _lib.check(lib.come_gated_matmul_e4m3(*xa, *ga, *ua, None, None, 0, T, F, K, full(T, stride, dtype=torch.uint8), stride, _lib.COME_E4M3,
                                              full(T, -(-F // 128), dtype=torch.float32), -(-F // 128), 1, st))
        _lib.check(lib.come_gated_matmul(*wide, full(T, F), F, st))
        rows = lib.come_gated_backward_rows(T, F)
        _lib.check(lib.come_gated_matmul_backward(*wide, dh.data_ptr(), F, full(rows, stride), full(rows, stride), stride, full(T, K), K, full(F, K), full(F, K), K,
                                                  None, None, st))
        return made

    try:
        raise_status()
        assert all(bool((t == 7).all()) for t in run())
    finally:
        _lib.device_status(clear=True)
    assert all(not bool((t[..., :1] == 7).all()) for t in run())  # cleared: the same launches compute
    assert _lib.device_status(clear=True) == 0


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("T,K,F", [(3, 128, 200), (130, 256, 192), (5003, 128, 1010)])
def test_no_gradient_is_written_while_the_status_word_is_raised(T, K, F, kind):
    """All five results of the backward pass, the biases' among them: their sums would be those of workspaces that nothing has filled."""
    from come_b200 import _lib
    lib, randn, st = _lib.lib(), gen(6), torch.cuda.current_stream().cuda_stream
    dtype = torch.float16 if kind == "f16" else torch.bfloat16
    assert _lib.device_status(clear=True) == 0
    x, wg, wu, dh, b = (t.to(dtype) for t in (randn(T, K), randn(F, K) / 8, randn(F, K) / 8, randn(T, F), randn(F)))
    rows, stride = lib.come_gated_backward_rows(T, F), -(-F // 8) * 8

    def run():
        made = [torch.full(s, 7, dtype=dtype, device="cuda") for s in ((rows, stride), (rows, stride), (T, K), (F, K), (F, K), (F,), (F,))]
        dg, du, dx, dwg, dwu, dbg, dbu = (t.data_ptr() for t in made)
        _lib.check(lib.come_gated_matmul_backward(x.data_ptr(), K, wg.data_ptr(), K, wu.data_ptr(), K, b.data_ptr(), b.data_ptr(), _lib.COME_F16 if kind == "f16" else _lib.COME_BF16, 0,
                                                  T, F, K, dh.data_ptr(), F, dg, du, stride, dx, K, dwg, dwu, K, dbg, dbu, st))
        return made

    try:
        raise_status()
        assert all(bool((t == 7).all()) for t in run())
    finally:
        _lib.device_status(clear=True)
    assert all(not bool((t == 7).all()) for t in run())
    assert _lib.device_status(clear=True) == 0


def test_products_beside_library_products_on_another_stream():
    """Both need tensor memory: the clusters of one and the CTA pairs of the other must not hold parts of each other's SMs."""
    from come_b200 import _lib
    from come_b200.block_scaled import block_scaled_linear, quantize_rows, quantize_weight
    from come_b200.feed_forward import gated_linear
    randn = gen(8)
    few, many = randn(60, 1024).bfloat16(), randn(5000, 1024).bfloat16()
    w, v = (randn(1040, 1024).bfloat16() / 32 for _ in range(2))
    few8, many8, w8 = quantize_rows(few), quantize_rows(many), quantize_weight(w)
    calls = (lambda: gated_linear(few, w, v), lambda: block_scaled_linear(few8, w8), lambda: gated_linear(many, w, v), lambda: block_scaled_linear(many8, w8))
    sizes = [(randn(m, 1024).bfloat16(), randn(n, 1024).bfloat16()) for m, n in ((64, 64), (128, 512), (300, 4096), (5000, 1040))]
    want, library = [c() for c in calls], [a @ b.t() for a, b in sizes]
    torch.cuda.synchronize()
    streams, got, theirs = [torch.cuda.Stream() for _ in range(2)], [], []
    for _ in range(30):
        with torch.cuda.stream(streams[0]):
            got.append([c() for c in calls])
        with torch.cuda.stream(streams[1]):
            theirs.append([a @ b.t() for a, b in sizes])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want)) and all(torch.equal(a, b) for r in theirs for a, b in zip(r, library))
    assert _lib.device_status(clear=True) == 0
