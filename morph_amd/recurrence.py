"""A gated linear recurrence over sequences and by single steps.

    a_t = sigmoid(f_t),   s_t = a_t s_(t-1) + (1 - a_t) v_t,   y_t = s_t silu(z_t)

for f, v, z [batch, steps, dim] (FP32, FP16 or BF16), every channel on its own; without z,
y_t = s_t.  The state is FP32 [batch, dim].  f = -inf forgets a finite one exactly (a packed
document begins), +inf passes it on unchanged (padding).  Kernels: csrc/scan.hip.

    y, state = gated_scan(f, v, z, state)                  # a prompt, then token by token
    y, state, saved = gated_scan_forward(f, v, z, state)   # training
    df, dv, dz, dstate = gated_scan_backward(dy, saved, dlast)
    y, state = gated_recurrence(f, v, z, state)            # the same under autograd
"""
import ctypes

import torch

from ._lib import SCAN_SPAN, ScanArgs, check, layer_calls, lib
from .layers import address, current_stream, dtype_code, first_order, native, require_gpu, requires_grad, running_on

FLOATS = (torch.float32, torch.float16, torch.bfloat16)


class SavedScan:
    """What a forward kept for its backward: its inputs, and the FP32 state that every
    SCAN_SPAN steps begin with.  The inputs may not change before the backward."""

    __slots__ = ("f", "v", "z", "state", "states")

    def __init__(self, f, v, z, state, states):
        self.f, self.v, self.z, self.state, self.states = f, v, z, state, states


def _channels_last(t):
    """t with its last dimension contiguous (a copy if it is not); other strides are free."""
    t = t.detach()
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _check(f, v, z, state):
    require_gpu(f, "f", FLOATS)
    if f.dim() != 3:
        raise ValueError(f"f must be [batch, steps, dim], got {tuple(f.shape)}")
    require_gpu(v, "v", (f.dtype,), f.shape, f.device)
    if z is not None:
        require_gpu(z, "z", (f.dtype,), f.shape, f.device)
    if state is not None:
        require_gpu(state, "state", (torch.float32,), (f.shape[0], f.shape[2]), f.device)


def _args(f, v, z, state):
    batch, steps, dim = f.shape
    zb, zs = (z.stride(0), z.stride(1)) if z is not None else (0, 0)
    return ScanArgs(address(f), address(v), address(z), address(state), batch, steps, dim,
                    f.stride(0), f.stride(1), v.stride(0), v.stride(1), zb, zs)


def _workspace(f, backward):
    size = lib().morph_scan_workspace_bytes(*f.shape, dtype_code(f.dtype), backward)
    return (torch.empty(size, dtype=torch.uint8, device=f.device) if size else None), size


def _forward(f, v, z, state, train, stream):
    if stream is None:
        made = layer_calls().scan_forward(f, v, z, state, train)
        if made is not None:
            if not train:
                return native(made)
            y, last, states = native(made)
            return y, last, SavedScan(f.detach(), v.detach(), z.detach() if z is not None else None,
                                      state.detach() if state is not None else None, states)
    _check(f, v, z, state)
    with running_on(f.device, stream, (f, v, z, state)):
        f, v = _channels_last(f), _channels_last(v)
        z = _channels_last(z) if z is not None else None
        state = state.detach().contiguous() if state is not None else None
        batch, steps, dim = f.shape
        y = torch.empty((batch, steps, dim), dtype=f.dtype, device=f.device)
        last = torch.empty((batch, dim), dtype=torch.float32, device=f.device)
        states = None
        if train:
            states = torch.empty((batch, -(-steps // SCAN_SPAN), dim), dtype=torch.float32, device=f.device)
        workspace, size = _workspace(f, 0)
        check(lib().morph_scan_forward(ctypes.byref(_args(f, v, z, state)), dtype_code(f.dtype), address(y),
                                       address(last), address(states), address(workspace), size,
                                       current_stream()))
        return y, last, SavedScan(f, v, z, state, states)


def gated_scan(f, v, z=None, state=None, stream=None):
    """(y, state behind the last step); state: the one before the first (None: zeros)."""
    return _forward(f, v, z, state, False, stream)[:2]


def gated_scan_forward(f, v, z=None, state=None, stream=None):
    """(y, last state, saved): gated_scan, with what the backward needs."""
    return _forward(f, v, z, state, True, stream)


def gated_scan_backward(dy, saved, dlast=None, stream=None):
    """(df, dv, dz, dstate): gradients of f, v, z (None without z) and of the first state, from
    those of y and of the last state (None: zeros)."""
    if not isinstance(saved, SavedScan):
        raise TypeError("saved must come from gated_scan_forward")
    f, v, z = saved.f, saved.v, saved.z
    if stream is None:
        made = layer_calls().scan_backward(dy, f, v, z, saved.state, saved.states, dlast)
        if made is not None:
            return native(made)
    require_gpu(dy, "dy", (f.dtype,), f.shape, f.device)
    if dlast is not None:
        require_gpu(dlast, "dlast", (torch.float32,), (f.shape[0], f.shape[2]), f.device)
    with running_on(f.device, stream, (dy, f, v, z, saved.state, saved.states, dlast)):
        dy = _channels_last(dy)
        dlast = dlast.detach().contiguous() if dlast is not None else None
        df, dv = (torch.empty(f.shape, dtype=f.dtype, device=f.device) for _ in range(2))
        dz = torch.empty(f.shape, dtype=f.dtype, device=f.device) if z is not None else None
        dstate = torch.empty((f.shape[0], f.shape[2]), dtype=torch.float32, device=f.device)
        workspace, size = _workspace(f, 1)
        check(lib().morph_scan_backward(ctypes.byref(_args(f, v, z, saved.state)), dtype_code(f.dtype),
                                        address(saved.states), address(dy), dy.stride(0), dy.stride(1),
                                        address(dlast), address(df), address(dv), address(dz),
                                        address(dstate), address(workspace), size, current_stream()))
        return df, dv, dz, dstate


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, f, v, z, state):
        y, last, saved = gated_scan_forward(f, v, z, state)
        # what was kept is autograd's to hold and release; the inputs for its guard against changes in place
        ctx.save_for_backward(f, v, z, state, *(getattr(saved, name) for name in SavedScan.__slots__))
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        saved = SavedScan(*ctx.saved_tensors[4:])
        if dy is None:
            dy = torch.zeros_like(saved.f)
        df, dv, dz, dstate = gated_scan_backward(dy, saved, dlast)
        return first_order("gated_recurrence", (df, dv, dz, dstate if saved.state is not None else None))


def gated_recurrence(f, v, z=None, state=None):
    """gated_scan under autograd: (y, last state), differentiable once in f, v, z and state."""
    if requires_grad("gated_recurrence", f, v, z, state):
        return _GatedScan.apply(f, v, z, state)
    return gated_scan(f, v, z, state)
