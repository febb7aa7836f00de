"""The feed-forward operators (RMSNorm with residual and 8-bit output, block-scaled products, gated projections with their
backward pass) against plain float64 formulas, element by element, with bounds derived from the roundings each kernel makes.

Roundings: a result in type t is off by at most half a step, eps_t / 2 relative (bf16 2^-8, fp16 2^-11, fp32 2^-24, e4m3 2^-4, or half
its smallest step, 2^-10, below 2^-6).  A tensor-core instruction adds 16 (16-bit) or 32 (8-bit) products to a float32 sum with an error
of at most 2^-22 of the largest magnitude in it; a sum of K products of magnitudes adding up to S is therefore off by at most
(K / 16 + 8) 2^-22 S, the eight covering the scales, the bias and the sums of a cluster's shares.  The logistic function and the normal
distribution are good to 2^-20.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half the smallest step


def rnd(kind):
    return torch.finfo(DT[kind]).eps / 2


def chain(K):
    return (K / 16 + 8) * 2.0 ** -22


def gen(seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device="cuda")


def d(t):
    return t.detach().double()


def within(got, want, bound, what):
    got, want = d(got), d(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"{what}: off by {(got - want).abs().flatten()[over.argmax()].item():.3g} at {over.argmax().item()}, allowed {torch.as_tensor(bound).expand_as(want).flatten()[over.argmax()].item():.3g}"


def act64(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = torch.special.erfc(-g / math.sqrt(2)) / 2
    return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def check_rows8(q, want, slack, what):
    """8-bit rows against the float64 values they were made from; ``slack``: how far the kernel's own values may be from those."""
    rows, cols = want.shape
    assert q.data.dtype == torch.float8_e4m3fn and q.data.shape == want.shape and q.scale.shape == (rows, -(-cols // 128)) and q.data.stride(0) % 16 == 0
    pad = torch.nn.functional.pad(want, (0, -cols % 128)).view(rows, -1, 128)
    loose = torch.nn.functional.pad(slack.expand_as(want), (0, -cols % 128)).view(rows, -1, 128).amax(-1)
    scale = pad.abs().amax(-1).clamp_min(448.0 * 2.0 ** -126) / 448.0
    within(q.scale, scale, loose / 448.0 + scale * 2.0 ** -21, what + " scale")
    wide = d(q.scale).repeat_interleave(128, 1)[:, :cols]
    value = d(q.data.float()) * wide
    within(value, want, want.abs() * 2.0 ** -4 + wide * 2.0 ** -10 + slack * (1 + 2.0 ** -4) + want.abs() * 2.0 ** -20, what + " values")
    assert d(q.data.float()).abs().max() <= 448


# ---- norm -------------------------------------------------------------------------------------------------------------------
NORM_SHAPES = [(1, 8), (4001, 24), (3001, 56), (2999, 64), (1003, 100), (1, 1024), (2, 40), (3, 127), (5, 128), (7, 129), (64, 1000), (600, 136), (593, 1024), (1200, 250), (9, 2052), (700, 4096), (3, 8192)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_residual_rmsnorm(rows, cols, kind):
    from come_b200.block import residual_rmsnorm
    randn = gen(rows * 10007 + cols)
    x, b, g = (3 * randn(rows, cols)).to(DT[kind]), randn(rows, cols).to(DT[kind]), (0.5 * randn(cols)).to(DT[kind])
    norm = torch.nn.RMSNorm(cols, eps=1e-5, device="cuda").requires_grad_(False)
    norm.weight.copy_(1 + 0.3 * randn(cols))
    w = norm.weight.to(DT[kind])
    e = rnd(kind)
    for branch, scale in ((b, g), (b, None), (None, None)):
        out, normed = residual_rmsnorm(x, branch, scale, norm)
        step = torch.zeros_like(d(x)) if branch is None else d(b) * (1 if scale is None else d(g))
        within(out, d(x) + step, e * (d(x) + step).abs() + 2.0 ** -23 * (d(x).abs() + step.abs()) + TINY[kind], "stream")
        stored = d(out)  # the norm is that of the stored stream
        y = stored / torch.sqrt(stored.pow(2).mean(1, keepdim=True) + 1e-5) * d(w)
        within(normed, y, (e + cols * 2.0 ** -24 + 2.0 ** -20) * y.abs() + TINY[kind], "normed")
        out8, q = residual_rmsnorm(x, branch, scale, norm, quantize=True)
        assert torch.equal(out8, out)
        check_rows8(q, y, y.abs() * (cols * 2.0 ** -24 + 2.0 ** -20), "normed")
    none, again = residual_rmsnorm(x, b, g, norm, store_stream=False)
    assert none is None and torch.equal(again, residual_rmsnorm(x, b, g, norm)[1])


def test_residual_rmsnorm_without_weight_and_eps():
    from come_b200.block import residual_rmsnorm
    x = gen(1)(33, 96).bfloat16()
    norm = torch.nn.RMSNorm(96, eps=None, elementwise_affine=False)
    _, normed = residual_rmsnorm(x, None, None, norm)
    y = d(x) / torch.sqrt(d(x).pow(2).mean(1, keepdim=True) + torch.finfo(torch.bfloat16).eps)
    within(normed, y, (2.0 ** -8 + 2.0 ** -17) * y.abs(), "normed")


def test_residual_rmsnorm_special_rows():
    """A zero row stays zero, a row with a NaN or an infinity is its own affair, and the smallest numbers keep finite scales."""
    from come_b200.block import residual_rmsnorm
    from come_b200.block_scaled import quantize_rows
    norm = torch.nn.RMSNorm(256, eps=1e-6, device="cuda").requires_grad_(False)
    x = gen(2)(6, 256)
    clean, clean8 = residual_rmsnorm(x, None, None, norm)[1], residual_rmsnorm(x, None, None, norm, quantize=True)[1]
    bad = x.clone()
    bad[1] = 0
    bad[2, 7] = float("nan")
    bad[3, 200] = float("inf")
    normed, q = residual_rmsnorm(bad, None, None, norm)[1], residual_rmsnorm(bad, None, None, norm, quantize=True)[1]
    keep = [0, 4, 5]
    assert torch.equal(normed[keep], clean[keep]) and torch.equal(q.data.float()[keep], clean8.data.float()[keep]) and torch.equal(q.scale[keep], clean8.scale[keep])
    assert (normed[1] == 0).all() and (q.data.float()[1] == 0).all() and torch.isfinite(q.scale[1]).all()
    assert normed[2].isnan().all() and q.data.float()[2].isnan().all()
    assert normed[3, 200].isnan() and (normed[3, :200] == 0).all() and q.data.float()[3, 200].isnan()
    # the quantiser alone: an infinity makes its block NaN, a NaN only itself
    r = quantize_rows(bad)
    v = r.dequantize()
    assert v[2, 7].isnan() and torch.isfinite(v[2, :7]).all() and torch.isfinite(v[2, 8:]).all()
    assert torch.isfinite(v[3, :128]).all() and v[3, 128:].isnan().all()
    large = torch.tensor([[3.4e38, 1e38, -9e37, 1e37] * 32], device="cuda")  # the largest numbers keep their values
    check_rows8(quantize_rows(large), d(large), torch.zeros((), device="cuda", dtype=torch.float64), "large")
    small = quantize_rows(torch.full((1, 128), 1e-41, device="cuda"))
    assert torch.isfinite(small.scale).all() and (small.scale >= 2.0 ** -126).all() and torch.isfinite(small.dequantize()).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 15), (130, 130), (128, 256), (257, 640), (1, 4000)])
def test_quantizers(rows, cols, kind):
    from come_b200.block_scaled import quantize_rows, quantize_weight
    t = (gen(rows + cols)(rows, cols + 3) * torch.exp(gen(5)(rows, 1))).to(DT[kind])[:, 1: cols + 1]  # rows that begin at odd addresses
    check_rows8(quantize_rows(t), d(t), torch.zeros((), device="cuda", dtype=torch.float64), "rows")
    q = quantize_weight(t)
    pad = torch.nn.functional.pad(d(t), (0, -cols % 128, 0, -rows % 128))
    blocks = pad.view(pad.shape[0] // 128, 128, pad.shape[1] // 128, 128)
    scale = blocks.abs().amax((1, 3)) / 448
    within(q.scale, scale, scale * 2.0 ** -21, "scale")
    wide = d(q.scale).repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    within(d(q.data.float()) * wide, d(t), d(t).abs() * (2.0 ** -4 + 2.0 ** -20) + wide * 2.0 ** -10, "values")
    assert torch.equal(q.dequantize(), (q.data.float() * wide.float()))


# ---- products of 8-bit operands -------------------------------------------------------------------------------------------------
def tokens8(randn, rows, cols):
    from come_b200.block_scaled import quantize_rows
    return quantize_rows(randn(rows, cols) * torch.exp(0.5 * randn(rows, 1)))


def weight8(randn, rows, cols):
    from come_b200.block_scaled import quantize_weight
    return quantize_weight(randn(rows, cols) / math.sqrt(cols))


def values(t):
    rows, cols = t.data.shape
    scale = t.scale if t.scale.shape[0] == rows and rows != -(-rows // 128) else t.scale.repeat_interleave(128, 0)[:rows] if t.scale.shape[0] != rows else t.scale
    return d(t.data.float()) * d(scale).repeat_interleave(128, 1)[:, :cols]


# from one token to more tiles than the GPU has SMs: both kernels, full and partial tiles, split contractions
LINEAR_SHAPES = [(1, 1, 1), (1, 16, 8), (1, 2736, 1024), (2, 129, 130), (7, 128, 128), (64, 500, 257), (127, 384, 300), (129, 1000, 40), (300, 64, 1100), (1374, 256, 384),
                 (2600, 257, 1003), (5000, 130, 1040), (9473, 384, 512),
                 (5000, 72, 1010), (5000, 72, 1012)]  # rows of the result at multiples of 4 and of 8 bytes


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,K,N", LINEAR_SHAPES)
def test_block_scaled_linear(T, K, N, kind):
    from come_b200.block_scaled import block_scaled_linear
    randn = gen(T * 31 + K * 7 + N)
    x, w, bias = tokens8(randn, T, K), weight8(randn, N, K), randn(N)
    xv, wv = values(x), d(w.dequantize(torch.float32))
    y, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    for b in (None, bias):
        out = block_scaled_linear(x, w, b, out_dtype=DT[kind])
        want, s = (y, size) if b is None else (y + d(b), size + d(b).abs())
        assert out.dtype == DT[kind] and out.is_contiguous()
        within(out, want, rnd(kind) * want.abs() + (1 + rnd(kind)) * chain(K) * s + TINY[kind], "out")
        assert torch.equal(out, block_scaled_linear(x, w, b, out_dtype=DT[kind])), "another run, other bits"


def test_block_scaled_linear_takes_any_scale_strides_and_row_strides():
    from come_b200.block_scaled import BlockScaled, block_scaled_linear
    randn = gen(77)
    for T, K, N in ((5, 300, 70), (5000, 300, 1040)):
        x, w = tokens8(randn, T, K), weight8(randn, N, K)
        want = block_scaled_linear(x, w)
        wide = torch.full((T, 448), 127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)  # NaN around the rows
        wide[:, 16: 16 + K] = x.data
        moved = BlockScaled(wide[:, 16: 16 + K], x.scale.contiguous())
        assert torch.equal(block_scaled_linear(moved, w), want)
        part = BlockScaled(x.data[2:], x.scale[2:])
        assert torch.equal(block_scaled_linear(part, w)[: 3], want[2: 5])
        stacked = torch.zeros((w.scale.shape[0], 9), device="cuda")
        stacked[:, : w.scale.shape[1]] = w.scale
        assert torch.equal(block_scaled_linear(x, BlockScaled(w.data, stacked[:, : w.scale.shape[1]])), want)


GATED_SHAPES = [(1, 8, 1), (1, 1024, 2736), (2, 72, 129), (65, 392, 130), (128, 128, 128), (130, 200, 500), (900, 264, 257), (2600, 136, 1003), (5200, 72, 520), (4700, 200, 640)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("T,K,F", GATED_SHAPES)
def test_block_scaled_gated_linear(T, K, F, act):
    from come_b200.block_scaled import block_scaled_gated_linear
    randn = gen(T + K + F)
    x, wg, wu = tokens8(randn, T, K), weight8(randn, F, K), weight8(randn, F, K)
    bg, bu = 0.5 * randn(F), 0.5 * randn(F)
    xv, gv, uv = values(x), d(wg.dequantize()), d(wu.dequantize())
    for biases in ((None, None), (bg, bu), (None, bu)):
        zero = torch.zeros(F, device="cuda", dtype=torch.float64)
        b0, b1 = (zero if b is None else d(b) for b in biases)
        g, u = xv @ gv.t() + b0, xv @ uv.t() + b1
        eg, eu = chain(K) * (xv.abs() @ gv.abs().t() + b0.abs()), chain(K) * (xv.abs() @ uv.abs().t() + b1.abs())
        a, _ = act64(g, act)
        h = a * u
        slack = 1.2 * eg * (u.abs() + eu) + a.abs() * eu + 2.0 ** -19 * (h.abs() + u.abs() * 2.0 ** -126)  # |act'| <= 1.13
        q = block_scaled_gated_linear(x, wg, wu, *biases, activation=act)
        check_rows8(q, h, slack, "h")
        for kind in ("f16", "bf16"):
            out = block_scaled_gated_linear(x, wg, wu, *biases, activation=act, out_dtype=DT[kind])
            within(out, h, rnd(kind) * h.abs() + (1 + rnd(kind)) * slack + TINY[kind], "h")
    again = block_scaled_gated_linear(x, wg, wu, None, bu, activation=act)
    assert torch.equal(again.data.view(torch.uint8), q.data.view(torch.uint8)) and torch.equal(again.scale, q.scale)


def test_a_row_with_nan_spoils_only_itself():
    from come_b200.block_scaled import BlockScaled, block_scaled_gated_linear, block_scaled_linear
    from come_b200.feed_forward import gated_linear
    randn = gen(9)
    for T in (40, 5000):
        x, w, v = tokens8(randn, T, 256), weight8(randn, 1040, 256), weight8(randn, 1040, 256)
        bits = x.data.view(torch.uint8).clone()
        bits[3, 5] = 0x7f
        spoiled = BlockScaled(bits.view(torch.float8_e4m3fn), x.scale)
        rest = torch.arange(T, device="cuda") != 3
        out, want = block_scaled_linear(spoiled, w), block_scaled_linear(x, w)
        assert out[3].isnan().all() and torch.equal(out[rest], want[rest])
        h, good = block_scaled_gated_linear(spoiled, w, v), block_scaled_gated_linear(x, w, v)
        assert h.data.float()[3].isnan().all() and torch.equal(h.data.view(torch.uint8)[rest], good.data.view(torch.uint8)[rest])
        xb, wb, vb = randn(T, 256).bfloat16(), randn(520, 256).bfloat16(), randn(520, 256).bfloat16()
        want = gated_linear(xb, wb, vb)
        xb[3, 5] = float("nan")
        out = gated_linear(xb, wb, vb)
        assert out[3].isnan().all() and torch.equal(out[rest], want[rest])


def test_rows_behind_the_last_stay_as_they_were():
    """The C entries write the rows and columns of the result and nothing around them."""
    from come_b200 import _lib
    lib, randn = _lib.lib(), gen(4)
    st = torch.cuda.current_stream().cuda_stream
    for T, K, F in ((3, 64, 70), (130, 64, 70), (5003, 64, 1010)):
        x, wg, wu = tokens8(randn, T, K), weight8(randn, F, K), weight8(randn, F, K)
        args = (x.data.data_ptr(), x.data.stride(0), x.scale.data_ptr(), *x.scale.stride())
        for dtype, code in ((torch.float32, 0), (torch.bfloat16, 2)):
            out = torch.full((T + 2, F + 14), 7.0, dtype=dtype, device="cuda")
            _lib.check(lib.come_matmul_e4m3(*args, wg.data.data_ptr(), wg.data.stride(0), wg.scale.data_ptr(), wg.scale.stride(0), None, T, F, K, out[1:].data_ptr(), F + 14, code, st))
            assert (out[0] == 7).all() and (out[T + 1] == 7).all() and (out[:, F:] == 7).all() and not (out[1: T + 1, :F] == 7).all()
        q = torch.full((T + 2, F + 128 - F % 16), 0x55, dtype=torch.uint8, device="cuda")
        s = torch.full((-(-F // 128) + 1, T + 2), 7.0, device="cuda")
        _lib.check(lib.come_gated_matmul_e4m3(*args, wg.data.data_ptr(), wg.data.stride(0), wg.scale.data_ptr(), wg.scale.stride(0), wu.data.data_ptr(), wu.data.stride(0),
                                              wu.scale.data_ptr(), wu.scale.stride(0), None, None, 0, T, F, K, q[1:].data_ptr(), q.stride(0), _lib.COME_E4M3,
                                              s[:, 1:].data_ptr(), 1, s.stride(0), st))
        assert (q[0] == 0x55).all() and (q[T + 1] == 0x55).all() and (q[:, F:] == 0x55).all()
        assert (s[:, 0] == 7).all() and (s[:, T + 1] == 7).all() and (s[-1] == 7).all() and not (s[:-1, 1: T + 1] == 7).any()


# ---- gated projections in 16 bits, and their gradients ------------------------------------------------------------------------------
def gated64(x, wg, wu, bg, bu, act, dh=None):
    """float64 result and gradients with bounds of the kernels' float32 sums: (h, slack of h), {name: (gradient, slack)}."""
    K, T = x.shape[1], x.shape[0]
    g, u = x @ wg.t() + bg, x @ wu.t() + bu
    eg, eu = chain(K) * (x.abs() @ wg.abs().t() + bg.abs()), chain(K) * (x.abs() @ wu.abs().t() + bu.abs())
    a, slope = act64(g, act)
    h = a * u
    slack = 1.2 * eg * (u.abs() + eu) + a.abs() * eu + 2.0 ** -19 * (h.abs() + u.abs() * 2.0 ** -126)
    if dh is None:
        return h, slack
    return h, slack, g, u, a, slope, eg, eu


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("T,K,F", GATED_SHAPES)
def test_gated_linear_and_its_gradients(T, K, F, act, kind):
    from come_b200.feed_forward import gated_linear
    randn = gen(T * 3 + K + F)
    dtype, e = DT[kind], rnd(kind)
    x, wg, wu = randn(T, K).to(dtype), (randn(F, K) * 1.5 / math.sqrt(K)).to(dtype), (randn(F, K) * 1.5 / math.sqrt(K)).to(dtype)
    bg, bu, dh = (0.3 * randn(F)).to(dtype), (0.3 * randn(F)).to(dtype), randn(T, F).to(dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, bg, bu)]
    out = gated_linear(*leaves, activation=act)
    grads = torch.autograd.grad(out, leaves, dh)
    h, slack, g, u, a, slope, eg, eu = gated64(d(x), d(wg), d(wu), d(bg), d(bu), act, d(dh))
    within(out, h, e * h.abs() + (1 + e) * slack + TINY[kind], "h")
    assert torch.equal(out.detach(), gated_linear(x, wg, wu, bg, bu, activation=act)), "without a graph, other bits"
    # gradients of the projections: |act''| <= 0.8 (gelu), rounded once to the type of the tokens
    dg, du = d(dh) * u * slope, d(dh) * a
    edg = d(dh).abs() * (slope.abs() * eu + (u.abs() + eu) * (0.85 * eg + 2.0 ** -18 * (1 + g.abs())))
    edu = d(dh).abs() * (1.2 * eg + 2.0 ** -19 * a.abs() + 2.0 ** -140)
    edg, edu = edg + e * (dg.abs() + edg) + TINY[kind], edu + e * (du.abs() + edu) + TINY[kind]
    ag, au = dg.abs() + edg, du.abs() + edu
    for name, got, want, wobble, size, terms in (
            ("dx", grads[0], dg @ d(wg) + du @ d(wu), edg @ d(wg).abs() + edu @ d(wu).abs(), ag @ d(wg).abs() + au @ d(wu).abs(), 2 * F),
            ("dgate", grads[1], dg.t() @ d(x), edg.t() @ d(x).abs(), ag.t() @ d(x).abs(), T),
            ("dup", grads[2], du.t() @ d(x), edu.t() @ d(x).abs(), au.t() @ d(x).abs(), T),
            ("dgate_bias", grads[3], dg.sum(0), edg.sum(0), ag.sum(0), T),
            ("dup_bias", grads[4], du.sum(0), edu.sum(0), au.sum(0), T)):
        assert got.dtype == dtype
        within(got, want, wobble + chain(terms) * size + e * (want.abs() + wobble + chain(terms) * size) + TINY[kind], name)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_the_gradient_formula_against_differences(act):
    """The float64 gradients that the kernels are held to, against central differences of the float64 result along random directions."""
    randn = gen(21)
    x, wg, wu, bg, bu, dh = (d(randn(*s)) for s in ((6, 16), (10, 16), (10, 16), (10,), (10,), (6, 10)))
    f = lambda *t: (act64(t[0] @ t[1].t() + t[3], act)[0] * (t[0] @ t[2].t() + t[4]) * dh).sum()  # noqa: E731
    _, _, g, u, a, slope, _, _ = gated64(x, wg, wu, bg, bu, act, dh)
    dg, du = dh * u * slope, dh * a
    formula = (dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dg.sum(0), du.sum(0))
    at, step = [x, wg, wu, bg, bu], 1e-5
    for i, grad in enumerate(formula):
        v = d(randn(*at[i].shape))
        up, down = ([t + s * v if j == i else t for j, t in enumerate(at)] for s in (step, -step))
        slope_there = (f(*up) - f(*down)) / (2 * step)
        # third derivatives of a few hundred: error step^2 * 1e3, and cancellation 1e-16 * |f| / step
        assert abs((grad * v).sum() - slope_there) <= 1e-6 * (1 + abs(slope_there))


@pytest.mark.parametrize("T,K,F", [(16, 1024, 2736), (64, 1024, 2736), (65, 1024, 2736)])
def test_gradient_of_one_weight_of_few_tokens(T, K, F):
    """One weight of two learns, with and without the second part of the operands, in results that have enough tiles for either kernel."""
    from come_b200.feed_forward import gated_linear
    randn = gen(T)
    x, wg, wu, dh = randn(T, K).bfloat16(), (randn(F, K) / 32).bfloat16(), (randn(F, K) / 32).bfloat16(), randn(T, F).bfloat16()
    both = [t.clone().requires_grad_(True) for t in (wg, wu)]
    want = torch.autograd.grad(gated_linear(x, *both), both, dh)
    for i in range(2):
        one = [t.clone().requires_grad_(j == i) for j, t in enumerate((wg, wu))]
        (got,) = torch.autograd.grad(gated_linear(x, *one), one[i], dh)
        # the two kernels add the same float32 terms in other orders
        within(got, want[i], 2.0 ** -8 * d(want[i]).abs() + chain(2 * T) * 4 * d(want[i]).abs().amax(), "one weight")


def test_gated_linear_forms_of_its_inputs():
    """Strided, misaligned, broadcast and three-dimensional tokens, weights that are halves of one tensor, gradients of some inputs only,
    of a broadcast result gradient and of a weight used twice."""
    from come_b200.feed_forward import gated_linear
    randn = gen(33)
    for T in (37, 5000):
        K, F = 72, 520
        x, w12 = randn(T, K).bfloat16(), (0.2 * randn(2 * F, K)).bfloat16()
        wg, wu = w12.chunk(2)
        want = gated_linear(x, wg.clone(), wu.clone())
        wide = torch.full((T, 96), float("nan"), device="cuda", dtype=torch.bfloat16)
        wide[:, 8: 80] = x
        odd = torch.full((T, 97), float("nan"), device="cuda", dtype=torch.bfloat16)
        odd[:, 3: 75] = x
        assert torch.equal(gated_linear(wide[:, 8: 80], wg, wu), want) and torch.equal(gated_linear(odd[:, 3: 75], wg, wu), want)
        assert torch.equal(gated_linear(x.t().contiguous().t(), wg.t().contiguous().t(), wu), want)
        assert torch.equal(gated_linear(x[None], wg, wu)[0], want)
        one = gated_linear(x[:1], wg, wu)
        same = gated_linear(x[:1].expand(T, K), wg, wu)
        assert (same == same[:1]).all() and (T < 1000 or torch.allclose(same[:1].float(), one.float(), rtol=2.0 ** -7, atol=1e-6))
        # gradients: some inputs only, and a broadcast gradient
        ones = torch.ones(T, F, device="cuda", dtype=torch.bfloat16)
        full = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
        all_three = torch.autograd.grad(gated_linear(*full), full, ones)
        for i in range(3):
            some = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, wg, wu))]
            gated_linear(*some).sum().backward()
            assert torch.equal(some[i].grad, all_three[i]) and all(some[j].grad is None for j in range(3) if j != i)
        both = wg.clone().requires_grad_(True)
        gx, gw = torch.autograd.grad(gated_linear(full[0], both, both), (full[0], both), ones)
        separate = [t.clone().requires_grad_(True) for t in (x, wg, wg)]
        sx, sg, su = torch.autograd.grad(gated_linear(*separate), separate, ones)
        assert torch.equal(gx, sx) and torch.equal(gw, sg + su)
        biases = [torch.zeros(F, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(2)]
        gated_linear(x, wg, wu, *biases).sum().backward()  # nothing but the biases learns
        every = [t.clone().requires_grad_(True) for t in (x, wg, wu, *(b.detach() for b in biases))]
        gated_linear(*every).sum().backward()
        assert torch.equal(biases[0].grad, every[3].grad) and torch.equal(biases[1].grad, every[4].grad)
        shared = x[:1].clone().requires_grad_(True)
        (gs,) = torch.autograd.grad(gated_linear(shared.expand(T, K), wg, wu), shared, ones)
        assert gs.shape == (1, K) and torch.isfinite(gs).all()


def test_empty_sizes():
    from come_b200.block import residual_rmsnorm
    from come_b200.block_scaled import block_scaled_gated_linear, block_scaled_linear, quantize_rows, quantize_weight
    from come_b200.feed_forward import gated_linear
    w = torch.randn(24, 64, device="cuda")
    none = quantize_rows(torch.empty(0, 64, device="cuda"))
    assert block_scaled_linear(none, quantize_weight(w)).shape == (0, 24)
    h = block_scaled_gated_linear(none, quantize_weight(w), quantize_weight(w))
    assert h.data.shape == (0, 24) and h.scale.shape == (0, 1)
    out, normed = residual_rmsnorm(torch.empty(0, 64, device="cuda"), None, None, torch.nn.RMSNorm(64, device="cuda"))
    assert normed.shape == (0, 64)
    wb = w.bfloat16().requires_grad_(True)
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = gated_linear(x, wb, wb)
    y.sum().backward()
    assert y.shape == (0, 24) and x.grad.shape == (0, 64) and (wb.grad == 0).all()


def test_refusals_on_the_gpu():
    from come_b200.block import residual_rmsnorm
    from come_b200.block_scaled import BlockScaled, block_scaled_gated_linear, block_scaled_linear, quantize_rows, quantize_weight
    from come_b200.feed_forward import gated_linear
    x = torch.randn(4, 64, device="cuda")
    norm = torch.nn.RMSNorm(64, device="cuda")
    with pytest.raises(ValueError, match="contiguous"):
        residual_rmsnorm(x.t(), None, None, norm)
    with pytest.raises(ValueError, match="branch must be"):
        residual_rmsnorm(x, x.bfloat16(), None, norm)
    with pytest.raises(ValueError, match="scale without a branch"):
        residual_rmsnorm(x, None, x[0], norm)
    with pytest.raises(ValueError, match="scale must be"):
        residual_rmsnorm(x, x, x[0, :5], norm)
    with pytest.raises(NotImplementedError, match="nn.RMSNorm"):
        residual_rmsnorm(x, None, None, torch.nn.LayerNorm(64, device="cuda"))
    with pytest.raises(NotImplementedError, match="at most"):
        residual_rmsnorm(torch.zeros(1, 8196, device="cuda"), None, None, torch.nn.RMSNorm(8196, device="cuda"))
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        residual_rmsnorm(x.double(), None, None, norm)
    with pytest.raises(RuntimeError, match="no autograd"):
        residual_rmsnorm(x.clone().requires_grad_(True), None, None, norm)
    with pytest.raises(RuntimeError, match="no autograd"):
        quantize_rows(x.clone().requires_grad_(True))
    with pytest.raises(ValueError, match=r"\[rows, C\]"):
        quantize_rows(x[0])
    x8, w8 = quantize_rows(x), quantize_weight(torch.randn(16, 64, device="cuda"))
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        block_scaled_linear(BlockScaled(x, x8.scale), w8)
    with pytest.raises(ValueError, match="scales must be"):
        block_scaled_linear(BlockScaled(x8.data, x8.scale[:3]), w8)
    with pytest.raises(ValueError, match="weight must be"):
        block_scaled_linear(x8, quantize_weight(torch.randn(16, 80, device="cuda")))
    with pytest.raises(ValueError, match="multiples of 16 bytes"):
        block_scaled_linear(BlockScaled(x8.data.view(torch.uint8).view(-1)[: 4 * 40].view(torch.float8_e4m3fn).view(4, 40), x8.scale), quantize_weight(torch.randn(16, 40, device="cuda")))
    with pytest.raises(ValueError, match="bias must be"):
        block_scaled_linear(x8, w8, torch.zeros(16, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        block_scaled_linear(x8, w8, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="same features"):
        block_scaled_gated_linear(x8, w8, quantize_weight(torch.randn(17, 64, device="cuda")))
    with pytest.raises(ValueError, match="activation"):
        block_scaled_gated_linear(x8, w8, w8, activation="tanh")
    with pytest.raises(RuntimeError, match="out_dtype"):
        block_scaled_gated_linear(x8, w8, w8, out_dtype=torch.float32)
    xb, wb = x.bfloat16(), torch.randn(16, 64, device="cuda").bfloat16()
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        gated_linear(x, wb.float(), wb.float())
    with pytest.raises(ValueError, match="w_gate and w_up must be"):
        gated_linear(xb, wb, wb[:5])
    with pytest.raises(NotImplementedError, match="multiple of 8"):
        gated_linear(xb[:, :60], wb[:, :60], wb[:, :60])
    with pytest.raises(ValueError, match="b_up must be"):
        gated_linear(xb, wb, wb, None, wb[0, :16].float())
    with pytest.raises(ValueError, match="w_gate must be"):
        gated_linear(xb, wb.half(), wb.half())
    xg = xb.clone().requires_grad_(True)
    (gx,) = torch.autograd.grad(gated_linear(xg, wb, wb).float().square().sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.float().sum().backward()


# ---- streams, graphs ------------------------------------------------------------------------------------------------------------------
def _chain(x, branch, gamma, norm, gate, up, down, bias):
    from come_b200.block import residual_rmsnorm
    from come_b200.block_scaled import block_scaled_gated_linear, block_scaled_linear
    stream, x8 = residual_rmsnorm(x, branch, gamma, norm, quantize=True)
    h = block_scaled_gated_linear(x8, gate, up)
    return residual_rmsnorm(stream, block_scaled_linear(h, down, bias, out_dtype=x.dtype), gamma, norm)


def _chain_parts(seed, T, C, F):
    randn = gen(seed)
    norm = torch.nn.RMSNorm(C, eps=1e-6, device="cuda", dtype=torch.bfloat16).requires_grad_(False)
    return (randn(T, C).bfloat16(), randn(T, C).bfloat16(), (0.1 * randn(C)).bfloat16(), norm, weight8(randn, F, C), weight8(randn, F, C), weight8(randn, C, F), randn(C))


@pytest.mark.parametrize("T", [1, 70, 5000])
def test_chain_in_two_graphs_and_on_another_stream(T):
    """The feed-forward half of a block as it is used: eager, on a side stream, and captured twice; replays of the two graphs in turn on
    new inputs give the eager bits."""
    parts = _chain_parts(T, T, 256, 1040)
    other = _chain_parts(T + 1, T, 256, 1040)
    want, want2 = _chain(*parts), _chain(*other[:2], *parts[2:])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _chain(*parts)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    slots, graphs = [], []
    for _ in range(2):
        x, b = parts[0].clone(), parts[1].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _chain(x, b, *parts[2:])
        slots.append((x, b, out))
        graphs.append(g)
    slots[1][0].copy_(other[0])
    slots[1][1].copy_(other[1])
    for _ in range(3):
        graphs[0].replay()
        graphs[1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(slots[0][2], want)) and all(torch.equal(a, b) for a, b in zip(slots[1][2], want2))


@pytest.mark.parametrize("T", [60, 5000])
def test_two_streams_at_once(T):
    """Launches of both product kernels on two streams at the same time give the bits of one after the other."""
    sets = [_chain_parts(i, T, 256, 1040) for i in range(2)]
    want = [_chain(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(_chain(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for r in got[i] for a, b in zip(r, want[i]))


def test_training_step_in_a_graph():
    from come_b200.feed_forward import gated_linear
    randn = gen(8)
    for T in (50, 4700):
        data = [randn(T, 200).bfloat16(), (0.1 * randn(640, 200)).bfloat16(), (0.1 * randn(640, 200)).bfloat16()]
        dh = randn(T, 640).bfloat16()

        def step(ts):
            leaves = [t.detach().requires_grad_(True) for t in ts]
            return torch.autograd.grad(gated_linear(*leaves, activation="gelu"), leaves, dh)

        want = [t.clone() for t in step(data)]
        x = torch.zeros_like(data[0])
        static = [x, *data[1:]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            grads = step(static)
        x.copy_(data[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


# ---- offsets beyond 32 bits ------------------------------------------------------------------------------------------------------------
def test_results_of_more_than_2_31_elements():
    """The last rows of a result with more than 2^31 elements are those of a call on these rows alone.  Two ways to the same real number,
    each with float32 sums and one rounding: a step of the result's type apart at most, with room for the sums near zero."""
    from come_b200.block import residual_rmsnorm
    from come_b200.block_scaled import block_scaled_gated_linear, block_scaled_linear, quantize_rows, quantize_weight
    from come_b200.feed_forward import gated_linear
    torch.manual_seed(11)
    T, K, F, tail = 1_050_000, 64, 2056, 200
    assert T * F > 2 ** 31
    x = torch.randn(T, K, device="cuda").bfloat16()
    wg, wu = (torch.randn(F, K, device="cuda").div_(8).bfloat16() for _ in range(2))
    last = x[-tail:].clone()

    def near(got, want, what):
        got, want = got.double(), want.double()
        assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + 1e-5 * want.abs().max()).all(), what

    x8, last8, g8, u8 = quantize_rows(x), quantize_rows(last), quantize_weight(wg), quantize_weight(wu)
    near(block_scaled_linear(x8, g8)[-tail:], block_scaled_linear(last8, g8), "8-bit product")
    near(block_scaled_gated_linear(x8, g8, u8, out_dtype=torch.bfloat16)[-tail:], block_scaled_gated_linear(last8, g8, u8, out_dtype=torch.bfloat16), "8-bit gated")
    q, want = block_scaled_gated_linear(x8, g8, u8), block_scaled_gated_linear(last8, g8, u8)
    assert ((q.scale[-tail:] - want.scale).abs() <= 2.0 ** -20 * want.scale).all()
    got, want = q.data[-tail:].float() * q.scale[-tail:].repeat_interleave(128, 1)[:, :F], want.dequantize()
    assert ((got - want).abs() <= 2.0 ** -3 * want.abs() + want.abs().max() * 2.0 ** -16).all()
    del q, got

    def grads(x, dh):
        x = x.detach().requires_grad_()
        w = wg.detach().requires_grad_()
        out = gated_linear(x, w, wu)
        out.backward(dh)
        return out.detach()[-tail:].clone(), x.grad[-tail:].clone(), w.grad

    dh = torch.zeros(T, F, device="cuda", dtype=torch.bfloat16)
    dh[-tail:] = torch.randn(tail, F, device="cuda")
    out, dx, dw = grads(x, dh)
    some = 2 ** 18 // F + 1  # as many rows keep the operands of the gradients in one part, like the long call
    assert tail > some and tail > 64
    out1, dx1, dw1 = grads(last, dh[-tail:].clone())
    near(out, out1, "gated")
    near(dx, dx1, "dx")
    near(dw, dw1, "dw")
    del dh, x8, out, dx, dw
    torch.cuda.empty_cache()

    rows, C = 2_100_000, 1032
    x = torch.randn(rows, C, device="cuda", dtype=torch.bfloat16)
    norm = torch.nn.RMSNorm(C, eps=1e-6).cuda().bfloat16()
    with torch.no_grad():
        stream, normed = residual_rmsnorm(x, x, None, norm)
        s1, n1 = residual_rmsnorm(x[-tail:].clone(), x[-tail:].clone(), None, norm)
        assert torch.equal(stream[-tail:], s1)
        near(normed[-tail:], n1, "norm")
        del normed, stream
        q = residual_rmsnorm(x, None, None, norm, quantize=True)[1]
        q1 = residual_rmsnorm(x[-tail:].clone(), None, None, norm, quantize=True)[1]
        got, want = q.data[-tail:].float() * q.scale[-tail:].repeat_interleave(128, 1)[:, :C], q1.dequantize()
        assert ((got - want).abs() <= 2.0 ** -3 * want.abs() + want.abs().max() * 2.0 ** -16).all()
    del q, x
    torch.cuda.empty_cache()


# ---- modules and the aggregator ---------------------------------------------------------------------------------------------------------
def test_gated_mlp_in_16_and_8_bits():
    """The module against its formula, and the 8-bit module against the formula on its own (quantised) weights, activations quantised as
    it documents."""
    from come_b200.block_scaled import BlockScaledGatedMlp, BlockScaledLinear, quantize_rows
    from come_b200.feed_forward import GatedMlp
    torch.manual_seed(3)
    mlp = GatedMlp(192, 328, activation="gelu").cuda()
    x = torch.randn(2, 50, 192, device="cuda")
    m16 = GatedMlp(192, 328, activation="gelu").cuda().bfloat16()
    m16.load_state_dict(mlp.state_dict())
    with torch.no_grad():
        y = m16(x.bfloat16())
    w12, b12, w3, b3 = (d(m16.state_dict()[k]) for k in ("w12.weight", "w12.bias", "w3.weight", "w3.bias"))
    g, u = (d(x.bfloat16()) @ w12.t() + b12).chunk(2, -1)
    h = act64(g, "gelu")[0] * u
    # h is rounded once to bfloat16, the product once more; float32 sums add chain(...) of the magnitudes
    want, size = h @ w3.t() + b3, h.abs() @ w3.abs().t() + b3.abs()
    within(y, want, (2.0 ** -8 + 16 * chain(328)) * size + 2.0 ** -8 * want.abs(), "bf16 module")
    m8 = BlockScaledGatedMlp(mlp, out_dtype=torch.float32)
    from come_b200.block_scaled import to_block_scaled
    assert isinstance(to_block_scaled(mlp), BlockScaledGatedMlp) and isinstance(to_block_scaled(torch.nn.Sequential(m16))[0], BlockScaledGatedMlp)
    assert m8.to(torch.bfloat16).gate_scale.dtype == torch.float32 and m8.gate.dtype == torch.float8_e4m3fn  # a cast leaves 8-bit weights alone
    y8 = m8(x)
    assert y8.dtype == torch.float32 and y8.shape == x.shape
    x8 = d(quantize_rows(x.view(-1, 192)).dequantize())
    wide = lambda n: d(m8._weight(n).dequantize())  # noqa: E731
    g, u = x8 @ wide("gate").t() + d(m8.gate_bias), x8 @ wide("up").t() + d(m8.up_bias)
    h = act64(g, "gelu")[0] * u
    # an element of h is rounded to 8 bits: 2^-4 of itself or 2^-10 of its block's scale, which is at most max|h| / 448
    room = h.abs() * 2.0 ** -4 + h.abs().amax(1, keepdim=True) / 448 * 2.0 ** -9 + 16 * chain(192) * (x8.abs() @ wide("gate").abs().t() + 1) * (1 + u.abs())
    within(y8.view(-1, 192), h @ wide("down").t() + d(m8.down_bias), room @ wide("down").abs().t() + chain(328) * (h.abs() @ wide("down").abs().t() + 1), "8-bit module")
    lin = torch.nn.Linear(192, 70).cuda()
    l8 = BlockScaledLinear(lin, out_dtype=torch.float32)
    want = x8 @ d(l8._weight("weight").dequantize()).t() + d(lin.bias)
    within(l8(x).view(-1, 70), want, chain(192) * (x8.abs() @ d(l8._weight("weight").dequantize()).abs().t() + 1) * 2 + 2.0 ** -23 * want.abs(), "8-bit linear")


@pytest.mark.parametrize("cols", [320, 328, 250])
def test_8_bit_modules_move_between_devices_and_through_state_dicts(cols):
    """The buffers keep their numbers and the rows their alignment when a module goes to the host and back, is copied, or is filled from
    contiguous tensors of its state dict, for widths that are not whole 16 bytes too."""
    import copy
    from come_b200.block_scaled import BlockScaledLinear
    torch.manual_seed(4)
    lin = torch.nn.Linear(cols, 130).cuda()
    x = torch.randn(9, cols, device="cuda")
    module = BlockScaledLinear(lin, out_dtype=torch.float32)
    want = module(x)
    state = {k: v.cpu().contiguous() for k, v in module.state_dict().items()}
    assert torch.equal(copy.deepcopy(module)(x), want)
    assert torch.equal(module.cpu().cuda()(x), want)
    assert torch.equal(module.half().cpu().float().cuda()(x), want)
    other = BlockScaledLinear(torch.nn.Linear(cols, 130).cuda(), out_dtype=torch.float32)
    other.load_state_dict(state, assign=True)
    assert torch.equal(other.cuda()(x), want)
    other.load_state_dict(BlockScaledLinear(lin).state_dict())
    assert torch.equal(other(x), want)


@pytest.mark.parametrize("eight", [False, True])
def test_aggregator_with_rms_norms_and_gated_mlps(eight):
    """The fused aggregator (norms with their residuals in one kernel, 8-bit rows straight from the norm) against the same modules run one
    by one, and its graph replay against itself."""
    from come_b200 import _lib
    from come_b200.block_scaled import BlockScaledGatedMlp, to_block_scaled
    from come_b200.fused import CapturedForward, FusedAggregator
    from come_b200.token_merger import MergePlan
    from come_b200.vggt_arch import AggregatorCore
    C, depth, start, side, B, S = 128, 2, 5, 7, 1, 3
    N, M = start + side * side, 4
    core = AggregatorCore(embed_dim=C, depth=depth, num_heads=2, mlp_ratio=2.0, init_values=0.5, retain_layers=None, patch_start_idx=start, norm="rms", mlp="gated").cuda().bfloat16().eval()
    if eight:
        to_block_scaled(core)
        assert sum(isinstance(m, BlockScaledGatedMlp) for m in core.modules()) == 2 * depth
    gen_cpu = torch.Generator().manual_seed(6)
    tokens = torch.randn(B, S, N, C, generator=gen_cpu).cuda().bfloat16()
    mask = (torch.rand(B * S, M, generator=gen_cpu) < 0.5).cuda()
    layout = _lib.Layout.two_d(start, side, side, 3, 3)
    with torch.no_grad():
        fused, _ = FusedAggregator(core)(tokens, MergePlan(mask, layout))
        plain, _ = FusedAggregator(core, fuse_elementwise=False)(tokens, MergePlan(mask, layout))
        model = FusedAggregator(core)
        replay, _ = CapturedForward(model)(tokens, MergePlan(mask, layout))
    for layer in range(depth):
        f, p = d(fused[layer]), d(plain[layer])
        # both round every branch to bfloat16 (2^-9 in the mean), at other places; in 8 bits an element that falls to the other side of a
        # rounding moves by 2^-4 of itself, in the norm's rows, in h and through LayerScale 0.5
        assert (f - p).norm() / p.norm() < (4e-2 if eight else 2e-2)
        assert torch.equal(replay[layer], fused[layer])
    assert _lib.device_status() == 0
