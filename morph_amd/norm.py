"""Layer norm over the last dimension, and its gradients.

    y = (x - mean) / sqrt(var + eps) * weight + bias

for x [..., cols] (FP32, FP16 or BF16; statistics and sums FP32), weight and bias [cols] of x's type or
FP32, or None.  Kernels: csrc/norm.hip.

    y = layer_norm(x, weight, bias)                        # serving
    y, saved = layer_norm_forward(x, weight, bias)         # training
    dx, dweight, dbias = layer_norm_backward(dy, saved)
    y = layer_normalization(x, weight, bias)               # the same under autograd
"""
import ctypes

import torch

from ._lib import NormArgs, check, lib, stage_calls
from .layers import (address, as_rows, current_stream, dtype_code, first_order, native, require_gpu, requires_grad,
                     row_stride, running_on)

FLOATS = (torch.float32, torch.float16, torch.bfloat16)


class SavedNorm:
    """What a forward kept for its backward: its input (which may not change before it) and each row's
    FP32 mean and 1 / sqrt(var + eps), [2, rows]."""

    __slots__ = ("x", "weight", "bias", "stats", "eps")

    def __init__(self, x, weight, bias, stats, eps):
        self.x, self.weight, self.bias, self.stats, self.eps = x, weight, bias, stats, eps


def check_weights(x, cols, **weights):
    """The weights' type: each is [cols] of x's type or FP32, all of one."""
    dtype = None
    for name, w in weights.items():
        if w is not None:
            require_gpu(w, name, (x.dtype, torch.float32), (cols,), x.device)
            if dtype not in (None, w.dtype):
                raise TypeError(f"{' and '.join(weights)} must have one type")
            dtype = w.dtype
    return torch.float32 if dtype is None else dtype


def whole(t):
    """t contiguous (a copy if it is not), None kept."""
    return t.detach().contiguous() if t is not None else None


def _check(x, weight, bias, eps):
    require_gpu(x, "x", FLOATS)
    if x.dim() == 0:
        raise ValueError("x must have at least one dimension")
    if not (isinstance(eps, (int, float)) and 0 <= eps < float("inf")):
        raise ValueError(f"eps must be a number from 0 on, got {eps}")
    return check_weights(x, x.shape[-1], weight=weight, bias=bias)


def _args(rows, weight, bias, eps, dtype):
    return NormArgs(address(rows), address(weight), address(bias), rows.shape[0], rows.shape[1], row_stride(rows), eps,
                    dtype_code(dtype))


def _rows(t):
    """t as as_rows has it, an empty one too."""
    return as_rows(t.detach()) if t.numel() else t.detach().reshape(t.shape[:-1].numel(), t.shape[-1])


def _forward(x, weight, bias, eps, train, stream):
    if stream is None and type(eps) is float:
        made = stage_calls().norm_forward(x, weight, bias, eps, train)
        if made is not None:
            if not train:
                return native(made), None
            y, stats = native(made)
            return y, SavedNorm(x.detach(), *(w.detach() if w is not None else None for w in (weight, bias)), stats, eps)
    dtype = _check(x, weight, bias, eps)
    with running_on(x.device, stream, (x, weight, bias)):
        rows, weight, bias = _rows(x), whole(weight), whole(bias)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        stats = torch.empty((2, rows.shape[0]), dtype=torch.float32, device=x.device) if train else None
        check(lib().morph_norm_forward(ctypes.byref(_args(rows, weight, bias, eps, dtype)), dtype_code(x.dtype),
                                       address(y), address(stats), current_stream()))
        return y, SavedNorm(rows.view(x.shape) if rows.is_contiguous() else x.detach(), weight, bias, stats, eps)


def layer_norm(x, weight=None, bias=None, eps=1e-5, stream=None):
    """The norm of x along its last dimension."""
    return _forward(x, weight, bias, eps, False, stream)[0]


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, stream=None):
    """(y, saved): layer_norm, with what the backward needs."""
    return _forward(x, weight, bias, eps, True, stream)


def layer_norm_backward(dy, saved, stream=None):
    """(dx, dweight, dbias): the gradients of x, and of weight and bias in their type (None without one)."""
    if not isinstance(saved, SavedNorm):
        raise TypeError("saved must come from layer_norm_forward")
    x, weight, bias = saved.x, saved.weight, saved.bias
    if stream is None and type(saved.eps) is float:
        made = stage_calls().norm_backward(dy, x, weight, bias, saved.stats, saved.eps)
        if made is not None:
            return native(made)
    require_gpu(dy, "dy", (x.dtype,), x.shape, x.device)
    with running_on(x.device, stream, (dy, x, weight, bias, saved.stats)):
        rows, dys = _rows(x), _rows(dy)
        weights = [w for w in (weight, bias) if w is not None]
        dtype = weights[0].dtype if weights else torch.float32
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dweight = torch.empty_like(weight) if weight is not None else None
        dbias = torch.empty_like(bias) if bias is not None else None
        size = lib().morph_norm_workspace_bytes(*rows.shape) if weights else 0
        workspace = torch.empty(size, dtype=torch.uint8, device=x.device)
        check(lib().morph_norm_backward(ctypes.byref(_args(rows, weight, bias, saved.eps, dtype)), dtype_code(x.dtype),
                                        address(saved.stats), address(dys), row_stride(dys), address(dx),
                                        address(dweight), address(dbias), address(workspace), size, current_stream()))
        return dx, dweight, dbias


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, saved = layer_norm_forward(x, weight, bias, eps)
        # what was kept is autograd's to hold and release; the inputs for its guard against changes in place
        ctx.save_for_backward(x, weight, bias, saved.x, saved.weight, saved.bias, saved.stats)
        ctx.eps = eps
        return y

    @staticmethod
    def backward(ctx, dy):
        saved = SavedNorm(*ctx.saved_tensors[3:], ctx.eps)
        return *first_order("layer_normalization", layer_norm_backward(dy, saved)), None


def layer_normalization(x, weight=None, bias=None, eps=1e-5):
    """layer_norm under autograd: differentiable once in x, weight and bias."""
    if requires_grad("layer_normalization", x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm(x, weight, bias, eps)
