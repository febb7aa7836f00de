"""Refusals of the feed-forward operators that need no GPU: the checks of the Python layer and those of the C entry points."""
import ctypes

import pytest
import torch

from come_b200 import _lib


def _e4m3(*shape):
    return torch.zeros(shape, dtype=torch.float8_e4m3fn)


def test_cpu_tensors_are_refused():
    from come_b200.block import residual_rmsnorm
    from come_b200.block_scaled import BlockScaled, block_scaled_gated_linear, block_scaled_linear, quantize_rows, quantize_weight
    from come_b200.feed_forward import gated_linear
    x, w = torch.zeros(4, 128), torch.zeros(16, 128)
    with pytest.raises(RuntimeError, match="on CUDA"):
        residual_rmsnorm(x, None, None, torch.nn.RMSNorm(128))
    with pytest.raises(RuntimeError, match="on CUDA"):
        quantize_rows(x)
    with pytest.raises(RuntimeError, match="on CUDA"):
        quantize_weight(w)
    with pytest.raises(RuntimeError, match="on CUDA"):
        gated_linear(x.bfloat16(), w.bfloat16(), w.bfloat16())
    x8, w8 = BlockScaled(_e4m3(4, 128), torch.ones(4, 1)), BlockScaled(_e4m3(16, 128), torch.ones(1, 1))
    with pytest.raises(RuntimeError, match="on CUDA"):
        block_scaled_linear(x8, w8)
    with pytest.raises(RuntimeError, match="on CUDA"):
        block_scaled_gated_linear(x8, w8, w8)


def test_gated_mlp_and_blocks_validate_their_choices():
    from come_b200.feed_forward import GatedMlp
    from come_b200.vggt_arch import Block
    with pytest.raises(ValueError, match="activation must be one of"):
        GatedMlp(64, 96, activation="relu")
    with pytest.raises(ValueError, match="norm must be"):
        Block(64, 1, norm="batch")
    blk = Block(64, 1, norm="rms", mlp="gated")
    assert isinstance(blk.norm1, torch.nn.RMSNorm) and blk.mlp.w3.in_features == (256 * 2 // 3 + 7) // 8 * 8
    plain = Block(64, 1)
    assert isinstance(plain.norm1, torch.nn.LayerNorm) and plain.mlp.fc1.out_features == 256


class _Memory:
    """Addresses that pass the checks of alignment; nothing reads them (the calls below are refused on the host)."""
    at = 1 << 20


def _refused(rc, text):
    assert rc == _lib.COME_ERR_ARG and text in _lib.last_error(), (rc, _lib.last_error())


def test_c_entries_refuse_bad_arguments_before_any_launch():
    lib, m = _lib.lib(), _Memory.at
    # the norm
    _refused(lib.come_residual_rmsnorm(m, None, m, 4, 64, _lib.COME_F32, m, 1e-6, None, m, None, 0, None, 0, 0, None), "scale without a branch")
    _refused(lib.come_residual_rmsnorm(m, None, None, 4, 64, 7, m, 1e-6, None, m, None, 0, None, 0, 0, None), "unknown dtype")
    _refused(lib.come_residual_rmsnorm(m, None, None, 4, 64, _lib.COME_F32, m, 1e-6, None, m, m, 64, m, 1, 4, None), "written once")
    _refused(lib.come_residual_rmsnorm(m, None, None, 4, 60, _lib.COME_F32, m, 1e-6, None, None, m, 60, m, 1, 4, None), "whole 16 bytes")
    _refused(lib.come_residual_rmsnorm(m, None, None, 4, 64, _lib.COME_F32, m, 1e-6, None, None, None, 0, None, 0, 0, None), "nothing to write")
    _refused(lib.come_residual_rmsnorm(None, None, None, 4, 64, _lib.COME_F32, m, 1e-6, None, m, None, 0, None, 0, 0, None), "x must not be NULL")
    assert lib.come_residual_rmsnorm(None, None, None, 0, 64, _lib.COME_F32, None, 1e-6, None, m, None, 0, None, 0, 0, None) == _lib.COME_OK
    rc = lib.come_residual_rmsnorm(m, None, None, 4, 16392, _lib.COME_BF16, m, 1e-6, None, m, None, 0, None, 0, 0, None)
    assert rc == _lib.COME_ERR_UNSUPPORTED and "16384" in _lib.last_error()
    # the quantisers
    _refused(lib.come_quantize_rows(m, _lib.COME_F32, 4, 64, 64, m, 72, m, 1, 4, None), "whole 16 bytes")
    _refused(lib.come_quantize_rows(m, _lib.COME_F32, 4, 64, 64, m + 8, 64, m, 1, 4, None), "16-byte aligned")
    _refused(lib.come_quantize_weight(m, _lib.COME_F32, 4, 64, 64, m, 32, m, 1, None), "bad strides")
    # the 8-bit product: sizes, dtype, alignment, strides, missing tensors
    good = dict(x=m, x_row=128, xs=m, xs_row=1, xs_block=4, w=m, w_row=128, ws=m, ws_row=1, bias=None, tokens=4, features=16, channels=128, out=m, out_row=16,
                dtype=_lib.COME_BF16, stream=None)
    for change, text in (({"channels": 0}, "sizes must be positive"), ({"tokens": -1}, "sizes must be positive"), ({"tokens": 1 << 31}, "sizes must be positive"),
                         ({"dtype": 3}, "unknown dtype"), ({"x": m + 4}, "x must be given"), ({"x_row": 120}, "x must be given"), ({"w_row": 136}, "w must be given"),
                         ({"w": None}, "w must be given"), ({"xs": None}, "scales and result"), ({"out_row": 8}, "scales and result")):
        _refused(lib.come_matmul_e4m3(*{**good, **change}.values()), text)
    assert lib.come_matmul_e4m3(*{**good, "tokens": 0}.values()) == _lib.COME_OK  # nothing to do, nothing launched
    gated = dict(x=m, x_row=128, xs=m, xs_row=1, xs_block=4, g=m, g_row=128, gs=m, gs_row=1, u=m, u_row=128, us=m, us_row=1, gb=None, ub=None, act=0, tokens=4,
                 features=16, channels=128, out=m, out_row=16, dtype=_lib.COME_E4M3, os=m, os_row=1, os_block=4, stream=None)
    for change, text in (({"act": 2}, "unknown activation"), ({"dtype": _lib.COME_F32}, "8 bits with scales"), ({"os": None}, "needs its scales"),
                         ({"out_row": 24}, "needs its scales"), ({"u_row": 100}, "up must be given"), ({"g": m + 1}, "gate must be given")):
        _refused(lib.come_gated_matmul_e4m3(*{**gated, **change}.values()), text)
    # 16 bits and the backward pass
    wide = dict(x=m, x_row=128, g=m, g_row=128, u=m, u_row=128, gb=None, ub=None, dtype=_lib.COME_BF16, act=0, tokens=4, features=16, channels=128, out=m, out_row=16, stream=None)
    for change, text in (({"dtype": _lib.COME_F32}, "float16 or bfloat16"), ({"act": -1}, "unknown activation"), ({"x_row": 124}, "x must be given"),
                         ({"out": None}, "out must be given"), ({"channels": 136}, "x must be given")):
        _refused(lib.come_gated_matmul(*{**wide, **change}.values()), text)
    back = dict(x=m, x_row=128, g=m, g_row=128, u=m, u_row=128, gb=None, ub=None, dtype=_lib.COME_BF16, act=0, tokens=4, features=16, channels=128, dout=m, dout_row=16,
                dg=m, du=m, d_row=16, dx=m, dx_row=128, dwg=m, dwu=m, dw_row=128, dbg=None, dbu=None, stream=None)
    for change, text in (({"tokens": 0}, "zero or empty"), ({"dout": None}, "dout must be given"), ({"d_row": 20}, "dgate must be given"), ({"du": m + 2}, "dup must be given"),
                         ({"dx_row": 64}, "dx must hold"), ({"dw_row": 64}, "weights' gradients")):
        _refused(lib.come_gated_matmul_backward(*{**back, **change}.values()), text)


def test_rows_of_the_backward_workspaces():
    lib = _lib.lib()
    assert [lib.come_gated_backward_rows(t, f) for t, f in ((0, 5), (1, 2736), (64, 1 << 20), (65, 2736), (65, 5000), (1000, 262), (1000, 263), (6456, 2736), (1 << 30, 1 << 30))] == \
        [0, 2, 128, 130, 65, 2000, 1000, 6456, 1 << 30]


def test_status_word_names_the_product_kernels():
    """The header, the library's message and the kernels agree on the bits (19-21)."""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    assert "bits 19-21" in open(os.path.join(root, "include", "come_b200.h")).read()
    assert "kStatusMatmul = 0x380000u" in open(os.path.join(root, "come_b200", "csrc", "come_internal.cuh")).read()
    assert ctypes.sizeof(ctypes.c_uint32) == 4
