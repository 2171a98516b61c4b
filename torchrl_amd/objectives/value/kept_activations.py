"""Activations kept for the backward pass in 8 bits.

A critic's or actor's linear layers keep their inputs until the backward pass; over a rollout of many steps those activations, not the
weights, fill the memory.  :func:`quantize_activation` keeps them at one byte an element and one more every 32 (half of bfloat16's, a
quarter of float32's); :func:`checkpointed_linear` / :class:`CheckpointedLinear` is the layer whose weight gradient is computed from them
directly, in matrix instructions that read the bytes: the wide activations never come back to memory.  The output and the gradient of the input
are those of an ordinary linear layer; only the weight gradient sees the rounding (half a step of 2^-6 of the block's largest
magnitude, less than one at the very top).  A layer of one output has a kernel of its own, so that its output has the same bits whether a
gradient is wanted or not.  The format and the kernels are behind ``trl_act_*`` of include/trl_value.h.

The reference has no counterpart.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch
from torch import nn, Tensor
from torch.autograd.function import once_differentiable

from torchrl_amd import _extension
from torchrl_amd.objectives.value import functional as F
from torchrl_amd.objectives.value.functional import _host_done, _native, _ptr

__all__ = ["QuantizedActivation", "quantize_activation", "checkpointed_linear", "CheckpointedLinear"]

BLOCK = 32  # features that share a step
HEAD_FEATURES = 65536  # kHeadFeatures of csrc/host_policy.cpp
_DT = {torch.float32: 0, torch.bfloat16: 2, torch.float16: 3}


def _check(x: Tensor, name: str):
    if not isinstance(x, Tensor):
        raise TypeError(f"{name} must be a tensor")
    if x.dtype not in _DT:
        raise NotImplementedError(f"torchrl_amd 8-bit activations support float32, bfloat16 and float16, got {x.dtype}")


def _check_device(x: Tensor):
    if x.device.type != "cuda":
        raise RuntimeError(f"torchrl_amd 8-bit activations run on MI355X (HIP, device type 'cuda') tensors only; got a tensor on {x.device}.")


def _rows(x: Tensor) -> Tensor:
    """``x`` as (N, D) with last stride 1."""
    x = x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


@dataclass
class QuantizedActivation:
    """``codes`` (int8, last dim filled up to whole blocks) and ``exponents`` (uint8, one a block: a step is ``2 ** (exponent - 127)``) of a
    tensor of ``shape`` and ``dtype``."""

    codes: Tensor
    exponents: Tensor
    shape: torch.Size
    dtype: torch.dtype

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> Tensor:
        """The values that the bytes stand for (exact in the tensor's own dtype and in bfloat16)."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _DT:
            raise NotImplementedError(f"torchrl_amd 8-bit activations support float32, bfloat16 and float16, got {dtype}")
        codes, exponents, lead, D = self.codes, self.exponents, tuple(self.shape[:-1]), self.shape[-1]
        blocks = (D + BLOCK - 1) // BLOCK
        if tuple(codes.shape) != (*lead, blocks * BLOCK) or tuple(exponents.shape) != (*lead, blocks) or codes.dtype != torch.int8 or \
                exponents.dtype != torch.uint8 or codes.device != exponents.device:
            raise RuntimeError(f"QuantizedActivation: codes {tuple(codes.shape)} {codes.dtype} and exponents {tuple(exponents.shape)} {exponents.dtype} "
                               f"do not hold a tensor of shape {tuple(self.shape)}")
        compiling = torch.compiler.is_compiling()
        host = None if compiling else F._HOST if F._HOST_TRIED else F._host_module()
        if host is not None:
            out = host.dequantize(codes, exponents, D, _DT[dtype])
            if out is not None:
                return _host_done(out)
        if compiling or F._recorded():
            from torchrl_amd.objectives.value import _ops
            return _ops.dequantize_activation_op(codes, exponents, D, dtype)
        _check_device(codes)
        out = torch.empty(self.shape, dtype=dtype, device=codes.device)
        if out.numel():
            codes, exponents = codes.contiguous(), exponents.contiguous()
            _native("trl_act_dequantize", out.device, _DT[dtype], codes.data_ptr(), exponents.data_ptr(), out.numel() // D, D, out.data_ptr())
        return out


def quantize_activation(x: Tensor) -> QuantizedActivation:
    """Keeps ``x`` ``[*B, D]`` (float32, bfloat16 or float16) in 8 bits: blocks of 32 features share a power of two, 2^-6 of the one at or below
    the block's largest magnitude; codes are rounded to nearest even and held to 127.  Blocks with a NaN or an infinity stand for NaN."""
    compiling = torch.compiler.is_compiling()
    host = None if compiling else F._HOST if F._HOST_TRIED else F._host_module()
    if host is not None:
        got = host.quantize(x)
        if got is not None:
            return QuantizedActivation(*_host_done(got), x.shape, x.dtype)
    if compiling or F._recorded():
        from torchrl_amd.objectives.value import _ops
        return QuantizedActivation(*_ops.quantize_activation_op(x), x.shape, x.dtype)
    _check(x, "x")
    if x.ndim < 1 or x.shape[-1] == 0:
        raise RuntimeError(f"quantize_activation needs a feature dim, got shape {tuple(x.shape)}")
    _check_device(x)
    codes, exponents = _empty_kept(x)
    if x.numel():
        rows = _rows(x.detach())
        _native("trl_act_quantize", x.device, _DT[x.dtype], rows.data_ptr(), rows.stride(0), rows.shape[0], x.shape[-1], codes.data_ptr(),
              exponents.data_ptr())
    return QuantizedActivation(codes, exponents, x.shape, x.dtype)


def _empty_kept(x: Tensor):
    blocks = (x.shape[-1] + BLOCK - 1) // BLOCK
    return (torch.empty(*x.shape[:-1], blocks * BLOCK, dtype=torch.int8, device=x.device),
            torch.empty(*x.shape[:-1], blocks, dtype=torch.uint8, device=x.device))


def _linear(x: Tensor, weight: Tensor, bias: Optional[Tensor]) -> Tensor:
    """The library's product.  With batch dims it is a view, and a Function's (or a no_grad block's) views may not be written in place later."""
    y = torch.nn.functional.linear(x, weight, bias)
    return torch.ops.aten._unsafe_view(y, y.shape) if y._is_view() else y


def _is_head(x: Tensor, weight: Tensor) -> bool:
    """Whether the layer runs in one pass of its own over x (host_policy.cpp has the measurements of the rule)."""
    return weight.shape[0] == 1 and weight.shape[1] <= HEAD_FEATURES and x.numel() > 0


def _linear_and_kept(x: Tensor, weight: Tensor, bias: Optional[Tensor], keep: bool):
    """(x W^T + b, codes, exponents), the latter None unless ``keep``: y has the same bits either way."""
    if not _is_head(x, weight):
        y = _linear(x, weight, bias)
        if not keep:
            return y, None, None
        kept = quantize_activation(x)
        return y, kept.codes, kept.exponents
    codes, exponents = _empty_kept(x) if keep else (None, None)
    y = torch.empty(*x.shape[:-1], 1, dtype=x.dtype, device=x.device)
    rows, w = _rows(x.detach()), weight.detach().contiguous()
    _native("trl_act_head_fwd", x.device, _DT[x.dtype], rows.data_ptr(), rows.stride(0), rows.shape[0], x.shape[-1], w.data_ptr(), _ptr(bias),
          _ptr(codes), _ptr(exponents), y.data_ptr())
    return y, codes, exponents


def _weight_grad(dy: Tensor, codes: Optional[Tensor], exponents: Optional[Tensor], D: int, want_db: bool, weight: Optional[Tensor] = None):
    """(dy^T x^, column sums of dy or None) of (N, O) gradients and a kept (N, D) activation; without one (D == 0) the sums alone.
    With the ``weight`` of a layer of one output (dw, db, dy weight)."""
    dy = dy if dy.stride(1) == 1 or dy.shape[1] == 1 else dy.contiguous()
    N, O = dy.shape
    dt = _DT[dy.dtype]
    if D:  # may come from a saved-tensor hook
        blocks = (D + BLOCK - 1) // BLOCK
        codes, exponents = codes.reshape(N, blocks * BLOCK).contiguous(), exponents.reshape(N, blocks).contiguous()
        F._check_kept((codes, exponents), ((torch.int8, (N, blocks * BLOCK), dy.device), (torch.uint8, (N, blocks), dy.device)))
    dw = torch.empty(O, D, dtype=dy.dtype, device=dy.device) if D else None
    db = torch.empty(O, dtype=dy.dtype, device=dy.device) if want_db else None
    need = _extension.get_lib().trl_act_weight_grad_workspace_bytes(dt, N, O, D)
    ws = torch.empty(need, dtype=torch.uint8, device=dy.device) if need else None
    if weight is not None:
        F._check_kept((weight,), ((dy.dtype, (1, D), dy.device),))
        w, dx = weight.detach().contiguous(), torch.empty(N, D, dtype=dy.dtype, device=dy.device)
        _native("trl_act_head_bwd", dy.device, dt, dy.data_ptr(), dy.stride(0), _ptr(codes), _ptr(exponents), N, D, w.data_ptr(), _ptr(dw), _ptr(db),
              _ptr(dx), _ptr(ws), need)
        return dw, db, dx
    _native("trl_act_weight_grad", dy.device, dt, dy.data_ptr(), dy.stride(0), _ptr(codes), _ptr(exponents), N, O, D, _ptr(dw), _ptr(db), _ptr(ws), need)
    return dw, db


class _CheckpointedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        y, codes, exponents = _linear_and_kept(x, weight, bias, ctx.needs_input_grad[1])
        ctx.save_for_backward(codes, exponents, weight if ctx.needs_input_grad[0] else None)
        ctx.features = x.shape[-1]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        codes, exponents, weight = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad
        dx = dw = db = None
        dy = grad.reshape(math.prod(grad.shape[:-1]), grad.shape[-1])
        if need_x and need_w and weight.shape[0] == 1:
            dw, db, dx = _weight_grad(dy, codes, exponents, ctx.features, need_b, weight)
            return dx.view(*grad.shape[:-1], ctx.features), dw, db
        if need_x:
            dx = (dy @ weight).view(*grad.shape[:-1], ctx.features)
        if need_w:
            dw, db = _weight_grad(dy, codes, exponents, ctx.features, need_b)
        elif need_b:
            _, db = _weight_grad(dy, None, None, 0, True)
        return dx, dw, db


def checkpointed_linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None) -> Tensor:
    """``torch.nn.functional.linear(x, weight, bias)`` that keeps ``x`` in 8 bits for the weight gradient (see the module's docstring).

    ``x`` ``[*B, D]``, ``weight`` ``[O, D]`` and ``bias`` ``[O]`` share one dtype (float32, bfloat16 or float16) and device; under autocast they
    are cast to its dtype.  Without a gradient to ``weight`` nothing is kept."""
    autocast, compiling = torch.is_autocast_enabled("cuda"), torch.compiler.is_compiling()
    if not autocast and not compiling:
        host = F._HOST if F._HOST_TRIED else F._host_module()
        if host is not None:  # checks, launches and the autograd node in one C++ hop (csrc/host_policy.cpp)
            got = host.checkpointed_linear(x, weight, bias)
            if got is not None:
                return _host_done(got)
    if autocast and all(isinstance(t, Tensor) for t in (x, weight)):
        dt = torch.get_autocast_dtype("cuda")
        x, weight, bias = x.to(dt), weight.to(dt), None if bias is None else bias.to(dt)
    if compiling or F._recorded():
        from torchrl_amd.objectives.value import _ops
        return _ops.checkpointed_linear(x, weight, bias)
    checkpointed_linear_check(x, weight, bias)
    if not F._needs_grad(x, weight, bias):
        return _linear_and_kept(x, weight, bias, False)[0]
    return _CheckpointedLinear.apply(x, weight, bias)


def checkpointed_linear_check(x: Tensor, weight: Tensor, bias: Optional[Tensor]) -> None:
    """Raises for arguments that :func:`checkpointed_linear` does not take."""
    for t, name in ((x, "x"), (weight, "weight"), (bias, "bias")):
        if t is not None or name != "bias":
            _check(t, name)
    if weight.ndim != 2 or x.ndim < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise RuntimeError(f"checkpointed_linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise RuntimeError(f"checkpointed_linear: bias must have shape {(weight.shape[0],)}, got {tuple(bias.shape)}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise RuntimeError(f"checkpointed_linear: {name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}")
    _check_device(x)


class CheckpointedLinear(nn.Linear):
    """``torch.nn.Linear`` on :func:`checkpointed_linear`: value and policy heads, and the hidden layers of actors and critics."""

    def forward(self, x: Tensor) -> Tensor:
        return checkpointed_linear(x, self.weight, self.bias)
