"""What the layer operators' wrappers share: checks of tensors, the stream a call runs on, and the
order of their derivatives."""
import contextlib
import ctypes

import torch
from torch.autograd import forward_ad

from ._lib import check, dtype_code

HALF = (torch.float16, torch.bfloat16)
GROUP = 32  # values of a row that share a scale in the 8-bit form (MORPH_ACT_GROUP)


def require_gpu(t, name, dtypes=None, shape=None, device=None):
    """t, checked: a GPU tensor of one of `dtypes`, of `shape` and on `device` where given."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must live on the GPU (got {t.device}); morph_amd has no CPU path")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


def as_rows(t):
    """t as [rows, cols] with its last dimension contiguous and one row stride: a view where
    there is one, else a copy."""
    if t.dim() == 2:
        rows = t
    else:
        try:
            rows = t.view(-1, t.shape[-1])
        except RuntimeError:
            rows = t.reshape(-1, t.shape[-1])
    if rows.shape[1] > 1 and rows.stride(1) != 1 or rows.shape[0] > 1 and rows.stride(0) < rows.shape[1]:
        rows = rows.contiguous()
    return rows


def row_stride(rows):
    """The leading dimension of as_rows' result (of one row: its length)."""
    return rows.stride(0) if rows.shape[0] > 1 else max(1, rows.shape[1])


@contextlib.contextmanager
def _elsewhere(device, stream, inputs):
    with torch.cuda.device(device), torch.cuda.stream(stream):
        for t in inputs:
            if t is not None:
                t.record_stream(torch.cuda.current_stream())
        yield


def running_on(device, stream, inputs=()):
    """A context whose current device and stream are the call's, so that what it allocates
    belongs to that stream.  Inputs are kept alive for the work queued there; their
    contents are the caller's to order, as for any stream."""
    if stream is not None and stream.device != device:
        raise ValueError(f"stream is on {stream.device}, expected {device}")
    if stream is None and device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return _elsewhere(device, stream, inputs if stream is not None else ())


def requires_grad(name, *tensors):
    """Whether a call under autograd has to keep something for its backward.  Tangents of forward mode
    are refused: the kernels would drop them."""
    tensors = [t for t in tensors if isinstance(t, torch.Tensor)]  # the operator refuses what is none
    if any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative (an input is a dual tensor)")
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors)


class _FirstOrder(torch.autograd.Function):
    @staticmethod
    def forward(ctx, name, anchor, *grads):
        ctx.name = name
        # aliases: inputs handed through would count as views of each other and refuse changes in place
        return tuple(g.detach() if g is not None else None for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.name} can be differentiated once: its gradients have no backward of their own")


def first_order(name, grads):
    """The gradients that a backward returns.  Under create_graph=True they would count as constants, and
    their own derivatives would be missing from a sum without an error: there they raise where they
    are differentiated.  (torch's once_differentiable does so only where the gradient that comes in
    requires one: not for the gradient of y.sum().)"""
    if not torch.is_grad_enabled():
        return grads
    return _FirstOrder.apply(name, torch.empty(0, requires_grad=True), *grads)


def native(result):
    """A result of LayerCalls (hostlayers.cpp); raises where it is a status of the library."""
    if type(result) is int:
        check(result)
    return result


def address(t):
    return t.data_ptr() if t is not None else None


def current_stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

