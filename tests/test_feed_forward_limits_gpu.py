"""Feed-forward operators at the edges of what they take: widths, lengths, ranges of gradients, norms and modules as users build them.
Plain float64 formulas; roundings as in test_feed_forward_gpu.py."""
import math

import pytest
import torch

from test_feed_forward_gpu import DT, TINY, act64, chain, check_rows8, d, gated64, gen, rnd, within

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
