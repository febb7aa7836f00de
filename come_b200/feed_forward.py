"""The gated feed-forward block: ``act(x Wg^T + bg) * (x Wu^T + bu)`` in one kernel, with its backward pass.

:func:`gated_linear` is the operator, :class:`GatedMlp` the module of a block (``block.mlp``), with the parameter layout of the gated
MLPs of visual transformers: ``w12`` holds both projections, the gate's rows first, ``w3`` the projection back.

A training step keeps only its inputs: the backward pass computes the projections again, in float32, and with them their gradients
(one kernel of ``come_gated_matmul_backward_in_range``), then ``dx = dg Wg + du Wu`` and ``dW = dg^T x`` / ``du^T x``.  ``dg`` and ``du`` are rounded to the
tokens' type once, as operands of these products (for few tokens, whose sums do not average that out, in two parts); saved 16-bit
projections would add their own rounding to every gradient.  In float16 they are held times a power of two where the largest ``|dh|``
is below 1/2 or from 2^10 on, so that neither a mean over many elements nor a scaled loss takes them out of the type's range.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._torch_util import dtype_code, has_tangent, on_device, ptr, require_cuda, stream_ptr
from .block_scaled import activation_code

__all__ = ["gated_linear", "GatedMlp"]


def _operand(t: torch.Tensor):
    """``t [rows, C]`` as the tensor cores can read it, rows that are contiguous and start at multiples of 16 bytes (copied if not):
    (tensor, pointer, row stride)."""
    row, col = t.stride()
    at = t.data_ptr()
    if col == 1 and row % 8 == 0 and row >= t.shape[1] and at % 16 == 0:
        return t, at, row
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), t.shape[1]


def _padded(rows: int, cols: int, like: torch.Tensor) -> torch.Tensor:
    return torch.empty_strided((rows, cols), ((cols + 7) & ~7, 1), dtype=like.dtype, device=like.device)


def _forward(x, w_gate, w_up, b_gate, b_up, act):
    tokens, cols = x.shape
    features, dev = w_gate.shape[0], x.device
    xo, x_at, x_row = _operand(x)  # the tensors are held until the launch is queued
    wg, g_at, g_row = _operand(w_gate)
    wu, u_at, u_row = _operand(w_up)
    out = torch.empty_strided((tokens, features), (features or 1, 1), dtype=x.dtype, device=dev)
    with on_device(dev):
        _lib.check(_lib.lib().come_gated_matmul(x_at, x_row, g_at, g_row, u_at, u_row, None if b_gate is None else b_gate.data_ptr(),
                                                None if b_up is None else b_up.data_ptr(), dtype_code(x.dtype), act, tokens, features, cols,
                                                out.data_ptr(), features, stream_ptr(dev)))
    return out


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        out = _forward(x, w_gate, w_up, b_gate, b_up, act)
        ctx.act = act
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, b_gate, b_up = ctx.saved_tensors
        need = ctx.needs_input_grad
        tokens, cols = x.shape
        features, dev = w_gate.shape[0], x.device

        def empty(wanted: bool, *shape):
            if not wanted:
                return None
            if tokens == 0 or features == 0:
                return torch.zeros(shape, dtype=x.dtype, device=dev)
            return torch.empty_strided(shape, (shape[-1], 1)[-len(shape):], dtype=x.dtype, device=dev)

        dx, dwg, dwu = empty(need[0], tokens, cols), empty(need[1], features, cols), empty(need[2], features, cols)
        dbg, dbu = empty(need[3], features), empty(need[4], features)
        if tokens == 0 or features == 0:
            return dx, dwg, dwu, dbg, dbu, None
        xo, x_at, x_row = _operand(x)  # the tensors are held until the launches are queued
        wg, g_at, g_row = _operand(w_gate)
        wu, u_at, u_row = _operand(w_up)
        if dh.stride(1) != 1:
            dh = dh.contiguous()
        lib = _lib.lib()
        d_rows = lib.come_gated_backward_rows(tokens, features)
        dg, du = _padded(d_rows + 1, features, x), _padded(d_rows, features, x)
        largest = dg.data_ptr() + 2 * d_rows * dg.stride(0)  # the float of workspace: in a row behind the last
        with on_device(dev):
            _lib.check(lib.come_gated_matmul_backward_in_range(
                x_at, x_row, g_at, g_row, u_at, u_row, ptr(b_gate), ptr(b_up), dtype_code(x.dtype), ctx.act,
                tokens, features, cols, dh.data_ptr(), dh.stride(0), dg.data_ptr(), du.data_ptr(), dg.stride(0), ptr(dx), cols, ptr(dwg), ptr(dwu), cols,
                ptr(dbg), ptr(dbu), largest, stream_ptr(dev)))
        return dx, dwg, dwu, dbg, dbu, None


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: Optional[torch.Tensor] = None,
                 b_up: Optional[torch.Tensor] = None, activation: str = "silu") -> torch.Tensor:
    """``act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)`` in one kernel, differentiable once in every tensor (in reverse mode).

    ``x [..., C]`` float16 or bfloat16, ``w_gate`` / ``w_up [F, C]`` and ``b_gate`` / ``b_up [F]`` in its dtype; ``C`` a multiple of 8.
    ``activation``: "silu" or "gelu" (the exact one).  Sums in float32, the result rounded once.  Rows that are not contiguous or do
    not start at multiples of 16 bytes are copied first.  Under autocast tensors in float32, or of several types, are cast to its type first."""
    require_cuda(x, "x")
    act = activation_code(activation)
    if torch.is_autocast_enabled("cuda"):
        x, w_gate, w_up, b_gate, b_up = _autocast(x, w_gate, w_up, b_gate, b_up)
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"x: unsupported dtype {x.dtype}; expected float16 or bfloat16")
    cols = x.shape[-1] if x.dim() else 0
    if w_gate.dim() != 2 or w_gate.shape[1] != cols or w_up.shape != w_gate.shape:
        raise ValueError(f"w_gate and w_up must be [F, {cols}], got {tuple(w_gate.shape)} and {tuple(w_up.shape)}")
    if cols == 0 or cols % 8 != 0:
        raise NotImplementedError(f"gated_linear needs a channel count that is a multiple of 8, got {cols}")
    dtype, index, features = x.dtype, x.get_device(), w_gate.shape[0]
    grad = x.requires_grad or w_gate.requires_grad or w_up.requires_grad
    if w_gate.dtype is not dtype or w_gate.get_device() != index:
        raise _mismatch("w_gate", w_gate, [features, cols], x)
    if w_up.dtype is not dtype or w_up.get_device() != index:
        raise _mismatch("w_up", w_up, [features, cols], x)
    if b_gate is not None:
        if b_gate.dtype is not dtype or b_gate.get_device() != index or b_gate.shape != (features,):
            raise _mismatch("b_gate", b_gate, [features], x)
        grad = grad or b_gate.requires_grad
        b_gate = b_gate.contiguous()
    if b_up is not None:
        if b_up.dtype is not dtype or b_up.get_device() != index or b_up.shape != (features,):
            raise _mismatch("b_up", b_up, [features], x)
        grad = grad or b_up.requires_grad
        b_up = b_up.contiguous()
    if has_tangent(x, w_gate, w_up, b_gate, b_up):
        raise RuntimeError("gated_linear has a backward pass, but no forward-mode derivative")
    apply = _GatedLinear.apply if grad and torch.is_grad_enabled() else _forward
    if x.dim() == 2:
        return apply(x, w_gate, w_up, b_gate, b_up, act)
    return apply(x.reshape(-1, cols), w_gate, w_up, b_gate, b_up, act).view(*x.shape[:-1], features)


def _autocast(*tensors):
    """The tensors as a linear layer takes them under autocast, unless they already have one 16-bit type."""
    have = {t.dtype for t in tensors if t is not None}
    if len(have) == 1 and have <= {torch.float16, torch.bfloat16}:
        return tensors
    dtype = torch.get_autocast_dtype("cuda")
    return tuple(t.to(dtype) if t is not None and t.dtype in (torch.float32, torch.float16, torch.bfloat16) else t for t in tensors)


def _mismatch(name: str, t: torch.Tensor, shape, x: torch.Tensor) -> Exception:
    return ValueError(f"{name} must be {shape} {x.dtype} on {x.device}, got {list(t.shape)} {t.dtype} on {t.device}")


class GatedMlp(torch.nn.Module):
    """``w3(act(gate) * up)`` with ``gate, up = w12(x).chunk(2)``: the gated MLP of a block.  The two projections, the activation and the
    product are one kernel; ``w3`` stays a PyTorch GEMM like the other linear layers of the blocks.  float16 and bfloat16, ``dim`` a multiple
    of 8, or float32 under autocast; float32 streams without it take the 8-bit form,
    :class:`come_b200.block_scaled.BlockScaledGatedMlp`."""

    def __init__(self, dim: int, hidden: int, bias: bool = True, activation: str = "silu"):
        super().__init__()
        activation_code(activation)
        self.activation = activation
        self.w12 = torch.nn.Linear(dim, 2 * hidden, bias=bias)
        self.w3 = torch.nn.Linear(hidden, dim, bias=bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        w_gate, w_up = self.w12.weight.chunk(2)
        b_gate, b_up = (None, None) if self.w12.bias is None else self.w12.bias.chunk(2)
        return self.w3(gated_linear(x, w_gate, w_up, b_gate, b_up, self.activation))
