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
from ._torch_util import dtype_code, has_tangent, on_device, require_cuda, stream_ptr

__all__ = ["BLOCK", "BlockScaled", "quantize_rows", "quantize_weight", "block_scaled_linear", "block_scaled_gated_linear",
           "BlockScaledLinear", "BlockScaledGatedMlp", "to_block_scaled"]

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
    # (empty_strided: the cheapest of torch's allocating calls, which are half of a small launch's host time)
    return BlockScaled(torch.empty_strided((rows, cols), ((cols + 15) & ~15, 1), dtype=torch.float8_e4m3fn, device=device),
                       torch.empty_strided((rows, (cols + 127) >> 7), (1, rows or 1), dtype=torch.float32, device=device))


def _matrix(x: torch.Tensor, name: str) -> torch.Tensor:
    require_cuda(x, name)
    if x.dim() != 2:
        raise ValueError(f"{name} must be a [rows, C] tensor, got {tuple(x.shape)}")
    if (x.requires_grad and torch.is_grad_enabled()) or has_tangent(x):
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


def _tokens(t: BlockScaled):
    """(pointer, row stride, scale pointer, its two strides), rows, columns of checked tokens."""
    data, scale = t
    if data.dim() == 2 and scale.dim() == 2 and data.is_cuda:
        rows, cols = data.shape
        row, col = data.stride()
        if (data.dtype is torch.float8_e4m3fn and scale.dtype is torch.float32 and cols > 0 and scale.shape == (rows, (cols + 127) >> 7)
                and data.get_device() == scale.get_device() and ((col == 1 and row % 16 == 0 and row >= cols and data.data_ptr() % 16 == 0) or rows == 0)):
            return (data.data_ptr(), row, scale.data_ptr(), *scale.stride()), rows, cols
    raise _operand_error(t, "x", True, None, None)


def _weight(t: BlockScaled, name: str, cols: int, index: int):
    """(pointer, row stride, scale pointer, its row stride), rows of a checked weight."""
    data, scale = t
    if data.dim() == 2 and scale.dim() == 2 and data.is_cuda:
        rows, width = data.shape
        row, col = data.stride()
        s_row, s_block = scale.stride()
        if (data.dtype is torch.float8_e4m3fn and scale.dtype is torch.float32 and width == cols
                and scale.shape == ((rows + 127) >> 7, (cols + 127) >> 7) and (s_block == 1 or cols <= BLOCK)
                and data.get_device() == index and scale.get_device() == index
                and ((col == 1 and row % 16 == 0 and row >= cols and data.data_ptr() % 16 == 0) or rows == 0)):
            return (data.data_ptr(), row, scale.data_ptr(), s_row), rows
    raise _operand_error(t, name, False, cols, index)


def _operand_error(t: BlockScaled, name: str, tokens: bool, cols: Optional[int], index: Optional[int]) -> Exception:
    data, scale = t
    if data.dtype != torch.float8_e4m3fn or scale.dtype != torch.float32:
        return RuntimeError(f"{name}: needs float8_e4m3fn numbers and float32 scales, got {data.dtype} and {scale.dtype}")
    if not data.is_cuda or not scale.is_cuda or data.get_device() != scale.get_device() or (index is not None and data.get_device() != index):
        return RuntimeError(f"{name} must be on CUDA, its numbers and scales on the device of x")
    if data.dim() != 2 or data.shape[1] == 0 or (cols is not None and data.shape[1] != cols):
        return ValueError(f"{name} must be [rows, {'C' if cols is None else cols}], got {tuple(data.shape)}")
    rows, width = data.shape
    want = [rows if tokens else -(-rows // BLOCK), -(-width // BLOCK)]
    if list(scale.shape) != want:
        return ValueError(f"{name}: scales must be {want}, got {list(scale.shape)}")
    if data.stride(1) != 1 or data.stride(0) % 16 or data.stride(0) < width or data.data_ptr() % 16:
        return ValueError(f"{name}: rows must start at multiples of 16 bytes and be contiguous (strides {data.stride()})")
    return ValueError(f"{name}: the scales of a weight must have contiguous rows (strides {scale.stride()})")


def _bias_ptr(bias: Optional[torch.Tensor], name: str, features: int, index: int):
    if bias is None:
        return None
    if bias.dtype is not torch.float32 or bias.shape != (features,) or bias.get_device() != index or not bias.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 [{features}] on the device of x, got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
    return bias.data_ptr()


def block_scaled_linear(x: BlockScaled, weight: BlockScaled, bias: Optional[torch.Tensor] = None,
                        out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x @ weight.T + bias`` of 8-bit operands (``come_matmul_e4m3``): ``x [T, C]`` with a scale per row and 128 columns, ``weight
    [N, C]`` with one per 128 x 128 block, ``bias [N]`` float32.  Returns ``[T, N]`` in float32, float16 or bfloat16."""
    x_args, tokens, cols = _tokens(x)
    index, dev = x.data.get_device(), x.data.device
    w_args, features = _weight(weight, "weight", cols, index)
    bias_ptr = _bias_ptr(bias, "bias", features, index)
    code = dtype_code(out_dtype, "out_dtype")
    out = torch.empty_strided((tokens, features), (features or 1, 1), dtype=out_dtype, device=dev)
    with on_device(dev):
        _lib.check(_lib.lib().come_matmul_e4m3(*x_args, *w_args, bias_ptr, tokens, features, cols, out.data_ptr(), features, code, stream_ptr(dev)))
    return out


def block_scaled_gated_linear(x: BlockScaled, gate: BlockScaled, up: BlockScaled, gate_bias: Optional[torch.Tensor] = None,
                              up_bias: Optional[torch.Tensor] = None, activation: str = "silu",
                              out_dtype: Optional[torch.dtype] = None):
    """``act(x @ gate.T + gate_bias) * (x @ up.T + up_bias)`` of 8-bit operands in one kernel (``come_gated_matmul_e4m3``).
    ``activation``: "silu" or "gelu" (the exact one).  Returns ``[T, F]`` in ``out_dtype`` (float16 or bfloat16) or, by default, in
    8 bits (:class:`BlockScaled`): the operand of the down projection, quantised from the float32 values."""
    x_args, tokens, cols = _tokens(x)
    index, dev = x.data.get_device(), x.data.device
    g_args, features = _weight(gate, "gate", cols, index)
    u_args, up_features = _weight(up, "up", cols, index)
    if up_features != features:
        raise ValueError(f"gate and up must have the same features, got {features} and {up_features}")
    gb, ub = _bias_ptr(gate_bias, "gate_bias", features, index), _bias_ptr(up_bias, "up_bias", features, index)
    act = activation_code(activation)
    if out_dtype is None:
        out = empty_rows(tokens, features, dev)
        where = (out.data.data_ptr(), out.data.stride(0), _lib.COME_E4M3, out.scale.data_ptr(), *out.scale.stride())
    else:
        if out_dtype not in (torch.float16, torch.bfloat16):
            raise RuntimeError(f"out_dtype: unsupported dtype {out_dtype}; expected float16, bfloat16 or None (8 bits)")
        out = torch.empty_strided((tokens, features), (features or 1, 1), dtype=out_dtype, device=dev)
        where = (out.data_ptr(), features, dtype_code(out_dtype), None, 0, 0)
    with on_device(dev):
        _lib.check(_lib.lib().come_gated_matmul_e4m3(*x_args, *g_args, *u_args, gb, ub, act, tokens, features, cols, *where, stream_ptr(dev)))
    return out


def activation_code(activation: str) -> int:
    try:
        return ACTIVATIONS[activation]
    except KeyError:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}") from None


class _QuantizedWeights(torch.nn.Module):
    """Holds weights in 8 bits as buffers.  They follow the module to another device, not to another dtype: ``module.to(bfloat16)``
    leaves numbers, scales and biases what they are.  The numbers' buffer is as wide as its rows are apart (whole 16 bytes, zeros behind
    the last column): copies to another device and state dicts keep columns, not strides."""

    def __init__(self):
        super().__init__()
        self._columns = {}

    def _apply(self, fn, recurse=True):
        kept = {name: b for name, b in self._buffers.items() if b is not None}
        super()._apply(fn, recurse)
        for name, old in kept.items():
            new = self._buffers[name]
            if new.dtype != old.dtype:
                self._buffers[name] = old.to(new.device)
        return self

    def _hold(self, name: str, weight: torch.Tensor, bias: Optional[torch.Tensor]) -> None:
        w = quantize_weight(weight)
        rows, cols = w.shape
        held = torch.zeros((rows, w.data.stride(0)), dtype=torch.uint8, device=w.data.device)
        held[:, :cols] = w.data.view(torch.uint8)
        self._columns[name] = cols
        self.register_buffer(name, held.view(torch.float8_e4m3fn))
        self.register_buffer(name + "_scale", w.scale)
        self.register_buffer(name + "_bias", None if bias is None else bias.detach().float().contiguous())

    def _weight(self, name: str) -> BlockScaled:
        data, cols = getattr(self, name), self._columns[name]
        return BlockScaled(data if data.shape[1] == cols else data[:, :cols], getattr(self, name + "_scale"))


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
    in 8 bits) and the down projection.  Takes tokens ``[..., C]`` in 16 or 32 bits and returns their dtype, or the 8-bit rows that
    :func:`come_b200.block.residual_rmsnorm` writes and returns ``out_dtype`` (that of the call, else the module's)."""

    def __init__(self, mlp: torch.nn.Module, out_dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.activation, self.out_dtype = mlp.activation, out_dtype
        activation_code(self.activation)
        hidden = mlp.w3.in_features
        bias = mlp.w12.bias
        self._hold("gate", mlp.w12.weight[:hidden], None if bias is None else bias[:hidden])
        self._hold("up", mlp.w12.weight[hidden:], None if bias is None else bias[hidden:])
        self._hold("down", mlp.w3.weight, mlp.w3.bias)

    def forward(self, x, out_dtype: Optional[torch.dtype] = None):
        if isinstance(x, BlockScaled):
            return self._forward(x, self.out_dtype if out_dtype is None else out_dtype)
        out = self._forward(quantize_rows(x.reshape(-1, x.shape[-1])), x.dtype if out_dtype is None else out_dtype)
        return out.view(*x.shape[:-1], out.shape[-1])

    def _forward(self, x: BlockScaled, out_dtype: torch.dtype) -> torch.Tensor:
        h = block_scaled_gated_linear(x, self._weight("gate"), self._weight("up"), self.gate_bias, self.up_bias, self.activation)
        return block_scaled_linear(h, self._weight("down"), self.down_bias, out_dtype)


def to_block_scaled(module: torch.nn.Module, out_dtype: torch.dtype = torch.bfloat16) -> torch.nn.Module:
    """Replaces every gated MLP inside ``module`` (on its CUDA device) by its 8-bit form, in place and in every place where it stands;
    returns ``module``, or the 8-bit form of ``module`` when it is a gated MLP itself.  A module without one is refused: other MLPs keep
    their 16-bit linear layers."""
    from .feed_forward import GatedMlp
    if isinstance(module, GatedMlp):
        return BlockScaledGatedMlp(module, out_dtype).train(module.training)
    made = {}  # one for every module, however many places it stands in
    for parent in list(module.modules()):
        for name, child in list(parent._modules.items()):
            if isinstance(child, GatedMlp):
                if child not in made:
                    made[child] = BlockScaledGatedMlp(child, out_dtype).train(child.training)
                setattr(parent, name, made[child])
    if not made and not any(isinstance(m, BlockScaledGatedMlp) for m in module.modules()):
        raise ValueError(f"{type(module).__name__} has no gated MLP (come_b200.feed_forward.GatedMlp) to convert")
    return module
