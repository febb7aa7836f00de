"""Feed-forward operators at the edges of what they take: widths, lengths, ranges of gradients, norms and modules as users build them.
Plain float64 formulas; roundings as in test_feed_forward_gpu.py."""
import math

import pytest
import torch

from test_feed_forward_gpu import DT, TINY, chain, check_rows8, d, gated64, gen, rnd, within

pytestmark = pytest.mark.gpu


# ---- norms as modules have them ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("quantize", [False, True])
def test_a_norm_without_an_eps_is_the_module_s(kind, quantize):
    """Where the framework runs a block's norm in place of the module (residual_norm), an nn.RMSNorm without an eps has float32's, as the
    module itself; with small streams another one shows in the first digit."""
    from come_b200.block import residual_norm
    x = (gen(1)(33, 96) * 2.0 ** -8).to(DT[kind])
    norm = torch.nn.RMSNorm(96, device="cuda").requires_grad_(False)
    y = d(x) / torch.sqrt(d(x).pow(2).mean(1, keepdim=True) + torch.finfo(torch.float32).eps)
    _, normed = residual_norm(x, None, None, norm, quantize=quantize)
    if quantize:
        check_rows8(normed, y, y.abs() * 2.0 ** -17, "normed")
    else:
        within(normed, y, (rnd(kind) + 2.0 ** -17) * y.abs() + TINY[kind], "normed")
        within(norm.to(DT[kind])(x), y, (rnd(kind) + 2.0 ** -17) * y.abs() + TINY[kind], "the module")


# ---- quantisers -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,rows,cols", [("f32", 3, 8193), ("f32", 5, 11008), ("bf16", 3, 16392), ("bf16", 4, 28672), ("f16", 2, 20001), ("f32", 700, 9000), ("f32", 1, 100_000)])
def test_rows_of_any_width_are_quantised(kind, rows, cols):
    from come_b200.block_scaled import quantize_rows
    t = (gen(cols)(rows, cols + 7) * torch.exp(gen(5)(rows, 1))).to(DT[kind])
    none = torch.zeros((), device="cuda", dtype=torch.float64)
    q = quantize_rows(t[:, :cols])  # rows further apart than they are wide
    check_rows8(q, d(t[:, :cols]), none, "rows")
    again = quantize_rows(t[:, :cols].contiguous())
    assert torch.equal(q.data.view(torch.uint8), again.data.view(torch.uint8)) and torch.equal(q.scale, again.scale)


def test_wide_modules_quantise_their_tokens():
    from come_b200.block_scaled import BlockScaledLinear, quantize_rows
    torch.manual_seed(7)
    lin = torch.nn.Linear(11008, 40).cuda()
    x = torch.randn(5, 11008, device="cuda")
    module = BlockScaledLinear(lin)
    xv, wv = d(quantize_rows(x).dequantize()), d(module._weight("weight").dequantize())
    with torch.no_grad():
        within(module(x), xv @ wv.t() + d(lin.bias), chain(11008) * (xv.abs() @ wv.abs().t() + 1) + 2.0 ** -23, "out")


@pytest.mark.parametrize("rows,cols", [(8_388_481, 8), (8_388_607, 1), (8_388_736, 8), (3, 8_400_000)])
def test_weights_of_many_rows_or_columns_are_quantised(rows, cols):
    from come_b200.block_scaled import quantize_weight
    w = torch.randn(rows, cols, device="cuda", dtype=torch.bfloat16)
    q = quantize_weight(w)
    tops = torch.nn.functional.pad(w.float().abs(), (0, -cols % 128, 0, -rows % 128)).view(-(-rows // 128), 128, -(-cols // 128), 128).amax((1, 3))
    within(q.scale, tops / 448, tops / 448 * 2.0 ** -21, "scale")
    for part in (slice(0, 300), slice(rows - 300 if rows > 300 else 0, rows)):
        start = part.start // 128 * 128
        at = slice(start, part.stop)
        wide = d(q.scale[start // 128:]).repeat_interleave(128, 0)[: q.data[at].shape[0]].repeat_interleave(128, 1)[:, :cols]
        within(d(q.data[at].float()) * wide, w[at], d(w[at]).abs() * (2.0 ** -4 + 2.0 ** -20) + wide * 2.0 ** -10, "values")


# ---- gradients ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,K,F", [(40, 72, 130), (1001, 200, 1003), (5000, 72, 520)])
@pytest.mark.parametrize("step", [-24, -18, -10, 0, 6])
def test_float16_gradients_of_any_size(T, K, F, step):
    """Gradients of the result from float16's smallest numbers (a mean over many elements without loss scaling) up: those of the projections
    keep their digits.  Brought to [1/2, 1) by a power of two where it is smaller, the largest |dh| leaves every gradient of a projection at most
    half a step off, or half the type's smallest, 2^-25, of that range: 2^-24 of the largest |dh|, and 2^-25 from 1/2 on."""
    from come_b200.feed_forward import gated_linear
    randn = gen(T + step)
    e = rnd("f16")
    x, wg, wu = randn(T, K).half(), (randn(F, K) * 1.5 / math.sqrt(K)).half(), (randn(F, K) * 1.5 / math.sqrt(K)).half()
    bg, bu, dh = (0.3 * randn(F)).half(), (0.3 * randn(F)).half(), (randn(T, F) * 2.0 ** step).half()
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, bg, bu)]
    grads = torch.autograd.grad(gated_linear(*leaves), leaves, dh)
    h, slack, g, u, a, slope, eg, eu = gated64(d(x), d(wg), d(wu), d(bg), d(bu), "silu", d(dh))
    least = d(dh).abs().max().clamp(max=0.5) * 2.0 ** -24
    dg, du = d(dh) * u * slope, d(dh) * a
    edg = d(dh).abs() * (slope.abs() * eu + (u.abs() + eu) * (0.85 * eg + 2.0 ** -18 * (1 + g.abs())))
    edu = d(dh).abs() * (1.2 * eg + 2.0 ** -19 * a.abs() + 2.0 ** -140)
    edg, edu = edg + e * (dg.abs() + edg) + least, edu + e * (du.abs() + edu) + least
    ag, au = dg.abs() + edg, du.abs() + edu
    for name, got, want, wobble, size, terms in (
            ("dx", grads[0], dg @ d(wg) + du @ d(wu), edg @ d(wg).abs() + edu @ d(wu).abs(), ag @ d(wg).abs() + au @ d(wu).abs(), 2 * F),
            ("dgate", grads[1], dg.t() @ d(x), edg.t() @ d(x).abs(), ag.t() @ d(x).abs(), T),
            ("dup", grads[2], du.t() @ d(x), edu.t() @ d(x).abs(), au.t() @ d(x).abs(), T),
            ("dgate_bias", grads[3], dg.sum(0), edg.sum(0), ag.sum(0), T),
            ("dup_bias", grads[4], du.sum(0), edu.sum(0), au.sum(0), T)):
        within(got, want, wobble + chain(terms) * size + e * (want.abs() + wobble + chain(terms) * size) + TINY["f16"], name)
        # the sum of independent roundings of a thousand terms is far below the sum of their bounds
        rough = 4 * e + TINY["f16"] / want.abs().square().mean().sqrt()
        assert (d(got) - want).norm() / want.norm() <= rough, (name, ((d(got) - want).norm() / want.norm()).item(), rough.item())


def test_float16_gradients_do_not_overflow_on_their_way():
    """dh up = 180,000 has no float16 number; the gradients that it becomes have, where its product with a weight (0.1) or a token (0.25)
    lies below 65504.  Products with numbers above 0.36 exceed float16 themselves: those are infinite in any arithmetic."""
    from come_b200.feed_forward import gated_linear
    for T in (40, 5000):
        K, F = 72, 520
        randn = gen(T)
        x, wg, wu = (0.25 * randn(T, K)).half(), (0.1 * randn(F, K)).half(), (0.1 * randn(F, K)).half()
        bg, bu = torch.full((F,), 1.0, device="cuda").half(), torch.full((F,), 3.0, device="cuda").half()
        dh = torch.zeros(T, F, device="cuda").half()
        dh[T // 2, 5] = 60000.0
        leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
        grads = torch.autograd.grad(gated_linear(*leaves, bg, bu), leaves, dh)
        h, slack, g, u, a, slope, eg, eu = gated64(d(x), d(wg), d(wu), d(bg), d(bu), "silu", d(dh))
        dg, du = d(dh) * u * slope, d(dh) * a
        assert dg.abs().max() > 65504
        for got, want in zip(grads, (dg @ d(wg) + du @ d(wu), dg.t() @ d(x), du.t() @ d(x))):
            # one rounding of each projection's gradient, one of the result, float32 sums of a few terms
            size = (dg.abs() @ d(wg).abs() + du.abs() @ d(wu).abs()) if want.shape == (T, K) else (dg.abs() + du.abs()).t() @ d(x).abs()
            bound = (3 * rnd("f16") + 2.0 ** -16) * size + TINY["f16"]
            fits, beyond = want.abs() + bound < 65504, want.abs() - bound > 65520  # from 65520 on float16 rounds to infinity
            assert want[fits].abs().max() > 2000 and beyond.float().mean() < 0.01
            within(got[fits], want[fits], bound[fits], "gradient")
            assert torch.isinf(got[beyond]).all()


@pytest.mark.parametrize("special", [float("inf"), float("nan")])
def test_an_infinite_gradient_spoils_what_it_reaches(special):
    """A row of dh with an infinity or a NaN (loss scaling gone too far) shows in every gradient that it is part of, and only there."""
    from come_b200.feed_forward import gated_linear
    for T in (40, 5000):
        randn = gen(T)
        x, wg, wu, dh = randn(T, 72).half(), (0.2 * randn(520, 72)).half(), (0.2 * randn(520, 72)).half(), randn(T, 520).half()
        leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu)]
        want = torch.autograd.grad(gated_linear(*leaves), leaves, dh)
        dh[3, 7] = special
        got = torch.autograd.grad(gated_linear(*leaves), leaves, dh)
        assert not torch.isfinite(got[0][3]).any() and not torch.isfinite(got[1][7]).any() and not torch.isfinite(got[2][7]).any()
        rest = torch.arange(T, device="cuda") != 3
        within(got[0][rest], want[0][rest], 2.0 ** -9 * d(want[0][rest]).abs() + 2.0 ** -10 * d(want[0]).abs().max(), "dx")
        keep = torch.arange(520, device="cuda") != 7
        assert torch.isfinite(got[1][keep]).all() and torch.isfinite(got[2][keep]).all()


@pytest.mark.parametrize("T", [40, 5000])
def test_a_large_float16_gradient_of_one_token_leaves_the_others_their_digits(T):
    """One token's gradients are 2^18 times the others' and still far from the type's largest number: nothing has to make room for them.
    The other tokens' dx depends on their own gradients only, each at most half a step or half the type's smallest step off."""
    from come_b200.feed_forward import gated_linear
    K, F = 72, 520
    randn = gen(T + 1)
    e = rnd("f16")
    x, wg, wu = randn(T, K).half(), (randn(F, K) * 1.5 / math.sqrt(K)).half(), (randn(F, K) * 1.5 / math.sqrt(K)).half()
    dh = (randn(T, F) * 2.0 ** -10).half()
    dh[3] = (randn(F) * 2.0 ** 8).clamp(-900, 900).half()
    leaf = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(gated_linear(leaf, wg, wu), leaf, dh)
    zero = torch.zeros(F, device="cuda", dtype=torch.float64)
    h, slack, g, u, a, slope, eg, eu = gated64(d(x), d(wg), d(wu), zero, zero, "silu", d(dh))
    dg, du = d(dh) * u * slope, d(dh) * a
    edg = d(dh).abs() * (slope.abs() * eu + (u.abs() + eu) * (0.85 * eg + 2.0 ** -18 * (1 + g.abs())))
    edu = d(dh).abs() * (1.2 * eg + 2.0 ** -19 * a.abs() + 2.0 ** -140)
    edg, edu = edg + e * (dg.abs() + edg) + 2.0 ** -25, edu + e * (du.abs() + edu) + 2.0 ** -25
    want, wobble = dg @ d(wg) + du @ d(wu), edg @ d(wg).abs() + edu @ d(wu).abs()
    size = (dg.abs() + edg) @ d(wg).abs() + (du.abs() + edu) @ d(wu).abs()
    within(dx, want, wobble + chain(2 * F) * size + e * (want.abs() + wobble + chain(2 * F) * size) + TINY["f16"], "dx")
    others = torch.arange(T, device="cuda") != 3
    # independent roundings: half a step of a gradient around 2^-10, or of the smallest numbers, and half a step of dx
    assert (d(dx[others]) - want[others]).norm() / want[others].norm() <= 2.0 ** -10


@pytest.mark.parametrize("T", [50, 1001, 4700])
def test_float16_steps_in_two_graphs_find_their_range_anew(T):
    """Replays in turn, with result gradients of other magnitudes than at the capture, give the eager bits."""
    from come_b200.feed_forward import gated_linear
    randn = gen(T)
    data = randn(T, 200).half(), (0.1 * randn(520, 200)).half(), (0.1 * randn(520, 200)).half()
    steps = [(randn(T, 520) * 2.0 ** e).half() for e in (0, -20, 8, -24)]

    def step(dh):
        leaves = [t.detach().requires_grad_(True) for t in data]
        return torch.autograd.grad(gated_linear(*leaves), leaves, dh)

    want = [step(dh) for dh in steps]
    slots, graphs = [], []
    for _ in range(2):
        dh, g = steps[0].clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(dh)
        slots.append((dh, out))
        graphs.append(g)
    for first, second in ((0, 1), (2, 3), (1, 2), (3, 0)):
        for (dh, _), i in zip(slots, (first, second)):
            dh.copy_(steps[i])
        for g in graphs + graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, out), i in zip(slots, (first, second)):
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
    # rows of the result's gradient that are further apart than they are wide, at an odd address, and one broadcast row
    wide = torch.full((T, 533), float("nan"), device="cuda").half()
    wide[:, 7: 527] = steps[1]
    assert all(torch.equal(a, b) for a, b in zip(step(wide[:, 7: 527]), want[1]))
    row = steps[1][:1].expand(T, 520)
    assert all(torch.equal(a, b) for a, b in zip(step(row), step(row.contiguous())))


# ---- forward mode -------------------------------------------------------------------------------------------------------------
def test_forward_mode_is_refused_not_dropped():
    """A dual tensor has no requires_grad: without a look at the level its tangent would vanish without a word."""
    from torch.autograd import forward_ad
    from come_b200.block import residual_rmsnorm
    from come_b200.block_scaled import quantize_rows
    from come_b200.feed_forward import gated_linear
    randn = gen(3)
    x, w, b = randn(5, 64).bfloat16(), randn(24, 64).bfloat16(), randn(24).bfloat16()
    norm = torch.nn.RMSNorm(64, eps=1e-6, device="cuda").requires_grad_(False)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(x), w, w), (x, dual(w), w), (x, w, w, dual(b)), (x, w, w, b, dual(b)), (dual(x)[None], w, w)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                gated_linear(*args)
        with pytest.raises(RuntimeError, match="no autograd"):
            residual_rmsnorm(dual(x), None, None, norm)
        with pytest.raises(RuntimeError, match="no autograd"):
            residual_rmsnorm(x, dual(x), None, norm)
        with pytest.raises(RuntimeError, match="no autograd"):
            quantize_rows(dual(x))
        assert torch.equal(gated_linear(x, w, w), gated_linear(x, w, w))  # tensors without a tangent still go through
        with torch.no_grad():
            assert gated_linear(x, w, w).shape == (5, 24)


# ---- autocast -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gated_projections_under_autocast(dtype):
    """float32 parameters and tokens under autocast are cast as a linear layer casts them, and gradients arrive in float32."""
    from come_b200.feed_forward import GatedMlp, gated_linear
    torch.manual_seed(1)
    mlp = GatedMlp(64, 88).cuda()
    x = torch.randn(3, 7, 64, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=dtype):
        y = mlp(x)
        half = mlp(x.to(dtype))
    assert y.dtype == dtype and torch.equal(y, half)
    y.float().square().sum().backward()
    w_gate, w_up = (t.detach().to(dtype) for t in mlp.w12.weight.chunk(2))
    b_gate, b_up = (t.detach().to(dtype) for t in mlp.w12.bias.chunk(2))
    leaves = [t.requires_grad_(True) for t in (x.detach().to(dtype), w_gate, w_up, b_gate, b_up, mlp.w3.weight.detach().to(dtype), mlp.w3.bias.detach().to(dtype))]
    want = torch.nn.functional.linear(gated_linear(*leaves[:5]), *leaves[5:])
    assert torch.equal(want, y)
    want.float().square().sum().backward()
    assert x.grad.dtype == torch.float32 and torch.equal(x.grad, leaves[0].grad.float())
    assert torch.equal(mlp.w12.weight.grad, torch.cat([leaves[1].grad, leaves[2].grad]).float()) and torch.equal(mlp.w12.bias.grad, torch.cat([leaves[3].grad, leaves[4].grad]).float())


# ---- modules -------------------------------------------------------------------------------------------------------------------
def test_every_use_of_a_gated_mlp_is_replaced():
    """A module that stands in several places, under one parent or under two, is replaced in all of them, by one 8-bit module."""
    from come_b200.block_scaled import BlockScaledGatedMlp, to_block_scaled
    from come_b200.feed_forward import GatedMlp
    mlp = GatedMlp(64, 96).cuda().bfloat16().eval()
    model = torch.nn.ModuleList([torch.nn.Sequential(mlp, mlp), torch.nn.Sequential(mlp), GatedMlp(64, 96).cuda()]).eval()
    to_block_scaled(model)
    assert not any(isinstance(m, GatedMlp) for m in model.modules())
    assert model[0][0] is model[0][1] and model[0][0] is model[1][0] and isinstance(model[2], BlockScaledGatedMlp) and model[2] is not model[0][0]
    assert not any(m.training for m in model.modules())
    assert to_block_scaled(model) is model  # a second time there is nothing left to do


def test_a_converted_mlp_keeps_its_mode():
    from come_b200.block_scaled import to_block_scaled
    from come_b200.feed_forward import GatedMlp
    assert not to_block_scaled(GatedMlp(64, 96).cuda().eval()).training and to_block_scaled(GatedMlp(64, 96).cuda()).training
