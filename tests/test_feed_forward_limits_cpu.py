"""Host-side checks of the feed-forward operators that need no GPU: refusals of the self-test, limits of sizes, and which modules the fused
path and the 8-bit conversion take."""
import pytest
import torch

from come_b200 import _lib

AT = 1 << 20  # an address that passes the checks of alignment; nothing reads it (the calls below end on the host)


def test_the_self_test_of_the_products_refuses_what_is_not_small():
    good = dict(x=AT, xs=AT, gate=AT, up=AT, ws=AT, tokens=64, features=128, channels=256, k_blocks=0, ctas=1, ticks=1000, out=AT, out_scale=AT, stream=None)
    for change, text in (({"x": None}, "must be given"), ({"out": None}, "must be given"), ({"xs": None}, "both operands or of none"), ({"xs": None, "ws": None}, "no 8-bit result"),
                         ({"tokens": 1 << 16}, "a small launch only"), ({"features": 24}, "a small launch only"), ({"channels": 192}, "a small launch only"),
                         ({"k_blocks": -1}, "must not be negative"), ({"ctas": 0}, "a mask"), ({"ctas": 256}, "a mask"), ({"ticks": 0}, "ticks must be"),
                         ({"ticks": (1 << 26) + 1}, "ticks must be"), ({"gate": AT + 8}, "16-byte aligned"), ({"out": AT + 8}, "16-byte aligned")):
        rc = _lib.lib().come_selftest_matmul_stall(*{**good, **change}.values())
        assert rc == _lib.COME_ERR_ARG and text in _lib.last_error(), (change, rc, _lib.last_error())


def _wrapper(norm1, norm2):
    """What `fusable` looks at of a wrapped block."""
    from types import SimpleNamespace
    none = torch.nn.Identity()
    return SimpleNamespace(block=SimpleNamespace(norm1=norm1, norm2=norm2, ls1=none, ls2=none), attn=SimpleNamespace(run_dtype=torch.bfloat16))


class _OneMore(torch.nn.RMSNorm):
    def forward(self, x):
        return torch.nn.functional.rms_norm(x, self.normalized_shape, 1 + self.weight, self.eps)


def test_norms_with_a_formula_of_their_own_are_not_fused():
    """A subclass that computes something else (weights stored as differences from one, say) runs as the module that it is."""
    from come_b200.block import fusable
    rms = torch.nn.RMSNorm(64)
    assert fusable(_wrapper(rms, rms), torch.bfloat16)
    assert not fusable(_wrapper(rms, rms), torch.float32)
    assert not fusable(_wrapper(_OneMore(64), rms), torch.bfloat16) and not fusable(_wrapper(rms, _OneMore(64)), torch.bfloat16)


def test_norms_wider_than_the_kernel_s_rows_are_not_fused():
    from come_b200.block import fusable
    narrow, wide = torch.nn.RMSNorm(16384, device="meta"), torch.nn.RMSNorm(16392, device="meta")
    assert fusable(_wrapper(narrow, narrow), torch.bfloat16)
    assert not fusable(_wrapper(wide, narrow), torch.bfloat16) and not fusable(_wrapper(narrow, wide), torch.bfloat16)


def test_a_conversion_that_finds_nothing_says_so():
    from come_b200.block_scaled import to_block_scaled
    from come_b200.vggt_arch import AggregatorCore
    with pytest.raises(ValueError, match="no gated MLP"):
        to_block_scaled(AggregatorCore(embed_dim=64, depth=1, num_heads=1))
    with pytest.raises(ValueError, match="no gated MLP"):
        to_block_scaled(torch.nn.Linear(4, 4))


def test_weights_beyond_the_grid_are_refused_by_name():
    """Sizes that the check accepts fit the launch: blocks of 128 x 128 are counted in one dimension of 2^31 - 1."""
    lib = _lib.lib()
    rc = lib.come_quantize_weight(AT, _lib.COME_BF16, (1 << 31) - 1, 1 << 20, 1 << 20, AT, 1 << 20, AT, 1 << 13, None)
    assert rc == _lib.COME_ERR_ARG and "blocks" in _lib.last_error(), _lib.last_error()


def test_the_backward_pass_in_range_refuses_what_the_other_refuses():
    lib = _lib.lib()
    good = dict(x=AT, x_row=128, g=AT, g_row=128, u=AT, u_row=128, gb=None, ub=None, dtype=_lib.COME_F16, act=0, tokens=4, features=16, channels=128, dout=AT, dout_row=16,
                dg=AT, du=AT, d_row=16, dx=AT, dx_row=128, dwg=AT, dwu=AT, dw_row=128, dbg=None, dbu=None, range=AT, stream=None)
    for change, text in (({"tokens": 0}, "zero or empty"), ({"dout": None}, "dout must be given"), ({"d_row": 20}, "dgate must be given"), ({"dw_row": 64}, "weights' gradients"),
                         ({"dtype": _lib.COME_F32}, "float16 or bfloat16"), ({"range": AT + 2}, "range_dev must be")):
        rc = lib.come_gated_matmul_backward_in_range(*{**good, **change}.values())
        assert rc == _lib.COME_ERR_ARG and text in _lib.last_error(), (change, rc, _lib.last_error())


def test_addresses_that_are_no_multiples_of_their_element_are_refused():
    """A kernel's access to such an address would fault; the check ends the call on the host."""
    lib, f32, bf16, e4m3 = _lib.lib(), _lib.COME_F32, _lib.COME_BF16, _lib.COME_E4M3
    norm = dict(x=AT, branch=AT, scale=AT, rows=4, channels=64, dtype=bf16, weight=AT, eps=1e-6, x_out=AT, normed=None, q=AT, q_row=64, qs=AT, qs_row=1, qs_block=4, stream=None)
    rows = dict(x=AT, dtype=f32, rows=4, channels=64, x_row=64, q=AT, q_row=64, qs=AT, qs_row=1, qs_block=4, stream=None)
    weight = dict(w=AT, dtype=f32, rows=4, channels=64, w_row=64, q=AT, q_row=64, qs=AT, qs_row=1, stream=None)
    linear = dict(x=AT, x_row=128, xs=AT, xs_row=1, xs_block=4, w=AT, w_row=128, ws=AT, ws_row=1, bias=AT, tokens=4, features=16, channels=128, out=AT, out_row=16, dtype=f32, stream=None)
    gated = dict(x=AT, x_row=128, xs=AT, xs_row=1, xs_block=4, g=AT, g_row=128, gs=AT, gs_row=1, u=AT, u_row=128, us=AT, us_row=1, gb=AT, ub=AT, act=0, tokens=4, features=16,
                 channels=128, out=AT, out_row=16, dtype=e4m3, os=AT, os_row=1, os_block=4, stream=None)
    wide = dict(x=AT, x_row=128, g=AT, g_row=128, u=AT, u_row=128, gb=AT, ub=AT, dtype=bf16, act=0, tokens=4, features=16, channels=128, out=AT, out_row=16, stream=None)
    back = dict(x=AT, x_row=128, g=AT, g_row=128, u=AT, u_row=128, gb=AT, ub=AT, dtype=bf16, act=0, tokens=4, features=16, channels=128, dout=AT, dout_row=16,
                dg=AT, du=AT, d_row=16, dx=AT, dx_row=128, dwg=AT, dwu=AT, dw_row=128, dbg=AT, dbu=AT, stream=None)
    for entry, good, pointers in ((lib.come_residual_rmsnorm, norm, ("x", "branch", "scale", "weight", "x_out", "qs")), (lib.come_quantize_rows, rows, ("x", "qs")),
                                  (lib.come_quantize_weight, weight, ("w", "qs")), (lib.come_matmul_e4m3, linear, ("xs", "ws", "bias", "out")),
                                  (lib.come_gated_matmul_e4m3, gated, ("xs", "gs", "us", "gb", "ub", "os")), (lib.come_gated_matmul_e4m3, {**gated, "dtype": bf16}, ("out",)),
                                  (lib.come_gated_matmul, wide, ("gb", "ub", "out")), (lib.come_gated_matmul_backward, back, ("gb", "ub", "dout", "dx", "dwg", "dwu", "dbg", "dbu"))):
        for name in pointers:
            rc = entry(*{**good, name: AT + 1}.values())
            assert rc == _lib.COME_ERR_ARG and "multiple" in _lib.last_error(), (entry, name, rc, _lib.last_error())
    for entry, good, strides in ((lib.come_residual_rmsnorm, norm, ("qs_row", "qs_block")), (lib.come_quantize_rows, rows, ("qs_row", "qs_block")),
                                 (lib.come_matmul_e4m3, linear, ("xs_row", "xs_block", "ws_row")), (lib.come_gated_matmul_e4m3, gated, ("xs_row", "xs_block", "gs_row", "us_row", "os_row", "os_block"))):
        for name in strides:
            rc = entry(*{**good, name: -1}.values())
            assert rc == _lib.COME_ERR_ARG and "negative" in _lib.last_error(), (entry, name, rc, _lib.last_error())
