"""Products of 8-bit operands with a scale per block of 128, for the linear layers of the blocks.

A tensor in 8 bits is a :class:`BlockScaled`: float8 e4m3 numbers and float32 scales, value = number * scale.  Tokens
``[rows, C]`` have a scale per row and 128 columns, weights ``[features, C]`` one per 128 x 128 block.  Tokens come from
:func:`quantize_rows`, from :func:`come_b200.block.residual_rmsnorm` (the norm in front of a layer writes them directly) or from
:func:`block_scaled_gated_linear` (whose result is the next layer's operand); weights from :func:`quantize_weight`, once.

Forward only, like the attention of this package.  The arithmetic: every block of 128 is an exact product of 8-bit numbers summed in
float32 on the tensor cores, scaled by the two scales of the block and added to a float32 sum.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from ._torch_util import dtype_code, on_device, ptr, require_cuda, stream_ptr

__all__ = ["BLOCK", "BlockScaled", "quantize_rows", "quantize_weight", "block_scaled_linear", "block_scaled_gated_linear",
           "BlockScaledLinear", "BlockScaledGatedMlp"]

BLOCK = 128
ACTIVATIONS = {"silu": _lib.COME_ACT_SILU, "gelu": _lib.COME_ACT_GELU}


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


class BlockScaled(NamedTuple):
    """``data [rows, C]`` float8_e4m3fn, rows at multiples of 16 bytes; ``scale`` float32, ``[rows, ceil(C / 128)]`` for tokens or
    ``[ceil(rows / 128), ceil(C / 128)]`` for a weight."""
    data: torch.Tensor
    scale: torch.Tensor

    @property
    def shape(self):
        return self.data.shape

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the tensor stands for (plain tensor code; for tests and for looking at them)."""
        rows, cols = self.data.shape
        scale = self.scale if self.scale.shape[0] == rows else self.scale.repeat_interleave(BLOCK, 0)[:rows]
        return (self.data.float() * scale.repeat_interleave(BLOCK, 1)[:, :cols]).to(dtype)


def empty_rows(rows: int, cols: int, device) -> BlockScaled:
    """Uninitialised tokens in 8 bits: rows padded to whole 16 bytes, scales with the rows next to each other (the order in which a
    product's threads read them)."""
    data = torch.empty((rows, -(-cols // 16) * 16), dtype=torch.float8_e4m3fn, device=device)[:, :cols]
    return BlockScaled(data, torch.empty((_blocks(cols), rows), dtype=torch.float32, device=device).t())


def _matrix(x: torch.Tensor, name: str) -> torch.Tensor:
    require_cuda(x, name)
    if x.dim() != 2:
        raise ValueError(f"{name} must be a [rows, C] tensor, got {tuple(x.shape)}")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name}: the 8-bit quantisers are inference only (no autograd)")
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def quantize_rows(x: torch.Tensor) -> BlockScaled:
    """Rows ``[rows, C]`` (float32, float16 or bfloat16) in 8 bits with a scale per row and 128 columns (``come_quantize_rows``)."""
    x = _matrix(x, "x")
    code, dev = dtype_code(x.dtype, "x"), x.device
    rows, cols = x.shape
    out = empty_rows(rows, cols, dev)
    with on_device(dev):
        _lib.check(_lib.lib().come_quantize_rows(x.data_ptr(), code, rows, cols, x.stride(0), out.data.data_ptr(), out.data.stride(0),
                                                 out.scale.data_ptr(), *out.scale.stride(), stream_ptr(dev)))
    return out


def quantize_weight(w: torch.Tensor) -> BlockScaled:
    """A weight ``[features, C]`` in 8 bits with a scale per 128 x 128 block (``come_quantize_weight``)."""
    w = _matrix(w.detach(), "w")
    code, dev = dtype_code(w.dtype, "w"), w.device
    rows, cols = w.shape
    data = torch.empty((rows, -(-cols // 16) * 16), dtype=torch.float8_e4m3fn, device=dev)[:, :cols]
    scale = torch.empty((_blocks(rows), _blocks(cols)), dtype=torch.float32, device=dev)
    with on_device(dev):
        _lib.check(_lib.lib().come_quantize_weight(w.data_ptr(), code, rows, cols, w.stride(0), data.data_ptr(), data.stride(0),
                                                   scale.data_ptr(), scale.stride(0), stream_ptr(dev)))
    return BlockScaled(data, scale)


def _check_operand(t: BlockScaled, name: str, rows_per_scale: int, cols: Optional[int], device) -> None:
    data, scale = t
    if data.dtype != torch.float8_e4m3fn or scale.dtype != torch.float32:
        raise RuntimeError(f"{name}: needs float8_e4m3fn numbers and float32 scales, got {data.dtype} and {scale.dtype}")
    if not data.is_cuda or data.device != device or scale.device != device:
        raise RuntimeError(f"{name} must be on CUDA, on the device of x")
    if data.dim() != 2 or data.shape[1] == 0 or (cols is not None and data.shape[1] != cols):
        raise ValueError(f"{name} must be [rows, {'C' if cols is None else cols}], got {tuple(data.shape)}")
    rows, width = data.shape
    want = (rows if rows_per_scale == 1 else -(-rows // BLOCK), -(-width // BLOCK))
    if tuple(scale.shape) != want:
        raise ValueError(f"{name}: scales must be {list(want)}, got {list(scale.shape)}")
    if rows and (data.stride(1) != 1 or data.stride(0) % 16 or data.stride(0) < width or data.data_ptr() % 16):
        raise ValueError(f"{name}: rows must start at multiples of 16 bytes and be contiguous (strides {data.stride()})")
    if rows_per_scale != 1 and scale.shape[1] > 1 and scale.stride(1) != 1:
        raise ValueError(f"{name}: the scales of a weight must have contiguous rows")


def _check_bias(bias: Optional[torch.Tensor], name: str, features: int, device) -> None:
    if bias is None:
        return
    if bias.dtype != torch.float32 or tuple(bias.shape) != (features,) or bias.device != device or not bias.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 [{features}] on {device}, got {bias.dtype} {tuple(bias.shape)} on {bias.device}")


def block_scaled_linear(x: BlockScaled, weight: BlockScaled, bias: Optional[torch.Tensor] = None,
                        out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x @ weight.T + bias`` of 8-bit operands (``come_matmul_e4m3``): ``x [T, C]`` with a scale per row and 128 columns, ``weight
    [N, C]`` with one per 128 x 128 block, ``bias [N]`` float32.  Returns ``[T, N]`` in float32, float16 or bfloat16."""
    dev = x.data.device
    _check_operand(x, "x", 1, None, dev)
    tokens, cols = x.data.shape
    _check_operand(weight, "weight", BLOCK, cols, dev)
    features = weight.data.shape[0]
    _check_bias(bias, "bias", features, dev)
    code = dtype_code(out_dtype, "out_dtype")
    out = torch.empty((tokens, features), dtype=out_dtype, device=dev)
    xs, ws = x.scale, weight.scale
    with on_device(dev):
        _lib.check(_lib.lib().come_matmul_e4m3(x.data.data_ptr(), x.data.stride(0), xs.data_ptr(), xs.stride(0), xs.stride(1),
                                               weight.data.data_ptr(), weight.data.stride(0), ws.data_ptr(), ws.stride(0), ptr(bias),
                                               tokens, features, cols, out.data_ptr(), features, code, stream_ptr(dev)))
    return out


def block_scaled_gated_linear(x: BlockScaled, gate: BlockScaled, up: BlockScaled, gate_bias: Optional[torch.Tensor] = None,
                              up_bias: Optional[torch.Tensor] = None, activation: str = "silu",
                              out_dtype: Optional[torch.dtype] = None):
    """``act(x @ gate.T + gate_bias) * (x @ up.T + up_bias)`` of 8-bit operands in one kernel (``come_gated_matmul_e4m3``).
    ``activation``: "silu" or "gelu" (the exact one).  Returns ``[T, F]`` in ``out_dtype`` (float16 or bfloat16) or, by default, in
    8 bits (:class:`BlockScaled`): the operand of the down projection, quantised from the float32 values."""
    dev = x.data.device
    _check_operand(x, "x", 1, None, dev)
    tokens, cols = x.data.shape
    _check_operand(gate, "gate", BLOCK, cols, dev)
    features = gate.data.shape[0]
    _check_operand(up, "up", BLOCK, cols, dev)
    if up.data.shape[0] != features:
        raise ValueError(f"gate and up must have the same features, got {features} and {up.data.shape[0]}")
    _check_bias(gate_bias, "gate_bias", features, dev)
    _check_bias(up_bias, "up_bias", features, dev)
    act = activation_code(activation)
    if out_dtype is None:
        out = empty_rows(tokens, features, dev)
        where = (out.data.data_ptr(), out.data.stride(0), _lib.COME_E4M3, out.scale.data_ptr(), out.scale.stride(0), out.scale.stride(1))
    else:
        if out_dtype not in (torch.float16, torch.bfloat16):
            raise RuntimeError(f"out_dtype: unsupported dtype {out_dtype}; expected float16, bfloat16 or None (8 bits)")
        out = torch.empty((tokens, features), dtype=out_dtype, device=dev)
        where = (out.data_ptr(), features, dtype_code(out_dtype), None, 0, 0)
    xs, gs, us = x.scale, gate.scale, up.scale
    with on_device(dev):
        _lib.check(_lib.lib().come_gated_matmul_e4m3(
            x.data.data_ptr(), x.data.stride(0), xs.data_ptr(), xs.stride(0), xs.stride(1), gate.data.data_ptr(), gate.data.stride(0),
            gs.data_ptr(), gs.stride(0), up.data.data_ptr(), up.data.stride(0), us.data_ptr(), us.stride(0), ptr(gate_bias), ptr(up_bias),
            act, tokens, features, cols, *where, stream_ptr(dev)))
    return out


def activation_code(activation: str) -> int:
    try:
        return ACTIVATIONS[activation]
    except KeyError:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}") from None


class _QuantizedWeights(torch.nn.Module):
    """Holds weights in 8 bits as buffers."""

    def _hold(self, name: str, weight: torch.Tensor, bias: Optional[torch.Tensor]) -> None:
        w = quantize_weight(weight)
        self.register_buffer(name, w.data)
        self.register_buffer(name + "_scale", w.scale)
        self.register_buffer(name + "_bias", None if bias is None else bias.detach().float().contiguous())

    def _weight(self, name: str) -> BlockScaled:
        return BlockScaled(getattr(self, name), getattr(self, name + "_scale"))


class BlockScaledLinear(_QuantizedWeights):
    """An ``nn.Linear`` with its weight in 8 bits.  Takes tokens ``[..., C]`` in 16 or 32 bits (quantised on the way) and returns
    their dtype, or a :class:`BlockScaled` and returns ``out_dtype``."""

    def __init__(self, linear: torch.nn.Linear, out_dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.out_dtype = out_dtype
        self._hold("weight", linear.weight, linear.bias)

    def forward(self, x):
        if isinstance(x, BlockScaled):
            return block_scaled_linear(x, self._weight("weight"), self.weight_bias, self.out_dtype)
        flat = x.reshape(-1, x.shape[-1])
        out = block_scaled_linear(quantize_rows(flat), self._weight("weight"), self.weight_bias, x.dtype)
        return out.view(*x.shape[:-1], out.shape[-1])


class BlockScaledGatedMlp(_QuantizedWeights):
    """A :class:`come_b200.feed_forward.GatedMlp` with its weights in 8 bits: two kernels, the gated projections (whose result leaves
    in 8 bits) and the down projection.  Takes tokens ``[..., C]`` in 16 or 32 bits, or the 8-bit rows that
    :func:`come_b200.block.residual_rmsnorm` writes (then the result is ``out_dtype``)."""

    def __init__(self, mlp: torch.nn.Module, out_dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.activation, self.out_dtype = mlp.activation, out_dtype
        activation_code(self.activation)
        hidden = mlp.w3.in_features
        bias = mlp.w12.bias
        self._hold("gate", mlp.w12.weight[:hidden], None if bias is None else bias[:hidden])
        self._hold("up", mlp.w12.weight[hidden:], None if bias is None else bias[hidden:])
        self._hold("down", mlp.w3.weight, mlp.w3.bias)

    def forward(self, x):
        if isinstance(x, BlockScaled):
            return self._forward(x, self.out_dtype)
        return self._forward(quantize_rows(x.reshape(-1, x.shape[-1])), x.dtype).view(*x.shape[:-1], -1)

    def _forward(self, x: BlockScaled, out_dtype: torch.dtype) -> torch.Tensor:
        h = block_scaled_gated_linear(x, self._weight("gate"), self._weight("up"), self.gate_bias, self.up_bias, self.activation)
        return block_scaled_linear(h, self._weight("down"), self.down_bias, out_dtype)
