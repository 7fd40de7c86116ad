"""The selective state space mixer: a short causal convolution and the selective scan, over sequences and by
single steps.

    u_t = silu(bias + sum_k weight_k x_(t-taps+1+k))                       causal_conv
    d_t = softplus(dt_t + dt_bias), h_t = exp(d_t A) h_(t-1) + d_t x_t B_t,
    y_t = (sum_n C_t h_t + skip x_t) silu(z_t)                             selective_scan

x, dt, z [batch, steps, dim] and B, C [batch, steps, states] are FP32, FP16 or BF16; A [dim, states] (negative, so
that states fade), skip and dt_bias [dim] and the states [batch, dim, states] are FP32, up to 64 states a
channel.  weight [dim, taps] and bias [dim] have x's type or FP32, taps 2 to 4; the convolution's state is its
last inputs, [batch, taps - 1, dim].  dt = -inf passes a state on unchanged (padding, with x, B and C finite).  A
positive A is taken while exp(A times the sum of d over the steps) stays finite.  Kernels: csrc/conv.hip, csrc/ssm.hip.

    u, inputs = causal_conv(x, weight, bias, inputs)                       # a prompt, then token by token
    y, state = selective_scan(u, dt, A, B, C, skip, z, dt_bias, state)
    u, inputs, saved = causal_conv_forward(x, weight, bias, inputs)        # training
    dx, dweight, dbias, dinputs = causal_conv_backward(du, saved, dlast)
    y, state, saved = selective_scan_forward(u, dt, A, B, C, skip, z, dt_bias, state)
    dx, ddt, dA, dB, dC, dskip, dz, ddt_bias, dstate = selective_scan_backward(dy, saved, dlast)
    causal_convolution(..), selective_state_space(..)                      # the same under autograd
"""
import ctypes

import torch

from ._lib import (CONV_MAX_TAPS, SSM_MAX_STATES, SSM_MAX_STEP, SSM_SPAN, ConvArgs, SsmArgs, SsmGrads, check, lib,
                   stage_calls)
from .layers import address, current_stream, dtype_code, first_order, native, require_gpu, requires_grad, running_on
from .norm import FLOATS, whole


def _channels_last(t):
    """t with its last dimension contiguous (a copy if it is not); other strides are free.  None kept."""
    if t is None:
        return None
    t = t.detach()
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _sequence(t, name):
    require_gpu(t, name, FLOATS)
    if t.dim() != 3:
        raise ValueError(f"{name} must be [batch, steps, dim], got {tuple(t.shape)}")


def _empty(shape, dtype, device):
    return torch.empty(shape, dtype=dtype, device=device)


# ---- the convolution ---------------------------------------------------------
class SavedConv:
    """What a forward kept for its backward: its inputs, which may not change before it."""

    __slots__ = ("x", "weight", "bias", "state")

    def __init__(self, x, weight, bias, state):
        self.x, self.weight, self.bias, self.state = x, weight, bias, state


def _check_conv(x, weight, bias, state):
    _sequence(x, "x")
    batch, _, dim = x.shape
    require_gpu(weight, "weight", (x.dtype, torch.float32), None, x.device)
    if weight.dim() != 2 or weight.shape[0] != dim or not 2 <= weight.shape[1] <= CONV_MAX_TAPS:
        raise ValueError(f"weight must be [{dim}, 2 to {CONV_MAX_TAPS}], got {tuple(weight.shape)}")
    if bias is not None:
        require_gpu(bias, "bias", (weight.dtype,), (dim,), x.device)
    if state is not None:
        require_gpu(state, "state", (x.dtype,), (batch, weight.shape[1] - 1, dim), x.device)


def _conv_args(x, weight, bias, state):
    return ConvArgs(address(x), address(state), address(weight), address(bias), *x.shape, x.stride(0), x.stride(1),
                    weight.shape[1], dtype_code(weight.dtype))


def _bare(*tensors):
    return (t.detach() if t is not None else None for t in tensors)


def _conv(x, weight, bias, state, train, stream):
    if stream is None:
        made = stage_calls().conv_forward(x, weight, bias, state)
        if made is not None:
            u, last = native(made)
            return u, last, SavedConv(*_bare(x, weight, bias, state)) if train else None
    _check_conv(x, weight, bias, state)
    with running_on(x.device, stream, (x, weight, bias, state)):
        x, weight, bias, state = _channels_last(x), whole(weight), whole(bias), whole(state)
        u = _empty(x.shape, x.dtype, x.device)
        last = _empty((x.shape[0], weight.shape[1] - 1, x.shape[2]), x.dtype, x.device)
        check(lib().morph_conv_forward(ctypes.byref(_conv_args(x, weight, bias, state)), dtype_code(x.dtype),
                                       address(u), address(last), current_stream()))
        return u, last, SavedConv(x, weight, bias, state)


def causal_conv(x, weight, bias=None, state=None, stream=None):
    """(u, the last taps - 1 inputs); state: those before the first step (None: zeros)."""
    return _conv(x, weight, bias, state, False, stream)[:2]


def causal_conv_forward(x, weight, bias=None, state=None, stream=None):
    """(u, inputs, saved): causal_conv, with what the backward needs."""
    return _conv(x, weight, bias, state, True, stream)


def causal_conv_backward(du, saved, dlast=None, stream=None):
    """(dx, dweight, dbias, dstate): gradients of x, weight, bias (None without one) and the inputs before the
    first step, from those of u and of the last inputs (None: zeros)."""
    if not isinstance(saved, SavedConv):
        raise TypeError("saved must come from causal_conv_forward")
    x, weight, bias, state = saved.x, saved.weight, saved.bias, saved.state
    if stream is None:
        made = stage_calls().conv_backward(du, x, weight, bias, state, dlast)
        if made is not None:
            return native(made)
    require_gpu(du, "du", (x.dtype,), x.shape, x.device)
    batch, steps, dim, taps = *x.shape, weight.shape[1]
    if dlast is not None:
        require_gpu(dlast, "dlast", (x.dtype,), (batch, taps - 1, dim), x.device)
    with running_on(x.device, stream, (du, x, weight, bias, state, dlast)):
        du, dlast = _channels_last(du), whole(dlast)
        dx, dweight = _empty(x.shape, x.dtype, x.device), torch.empty_like(weight)
        dbias = torch.empty_like(bias) if bias is not None else None
        dstate = _empty((batch, taps - 1, dim), x.dtype, x.device)
        size = lib().morph_conv_workspace_bytes(batch, steps, dim, taps)
        workspace = _empty(size, torch.uint8, x.device)
        check(lib().morph_conv_backward(ctypes.byref(_conv_args(x, weight, bias, state)), dtype_code(x.dtype),
                                        address(du), du.stride(0), du.stride(1), address(dlast), address(dx),
                                        address(dweight), address(dbias), address(dstate), address(workspace), size,
                                        current_stream()))
        return dx, dweight, dbias, dstate


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state):
        u, last, saved = causal_conv_forward(x, weight, bias, state)
        ctx.save_for_backward(x, weight, bias, state, *(getattr(saved, name) for name in SavedConv.__slots__))
        ctx.set_materialize_grads(False)
        return u, last

    @staticmethod
    def backward(ctx, du, dlast):
        saved = SavedConv(*ctx.saved_tensors[4:])
        if du is None:
            du = torch.zeros_like(saved.x)
        dx, dweight, dbias, dstate = causal_conv_backward(du, saved, dlast)
        return first_order("causal_convolution", (dx, dweight, dbias, dstate if saved.state is not None else None))


def causal_convolution(x, weight, bias=None, state=None):
    """causal_conv under autograd: (u, last inputs), differentiable once in x, weight, bias and state."""
    if requires_grad("causal_convolution", x, weight, bias, state):
        return _CausalConv.apply(x, weight, bias, state)
    return causal_conv(x, weight, bias, state)


# ---- the scan ------------------------------------------------------------------
class SavedSelective:
    """What a forward kept for its backward: its inputs, which may not change before it, and the FP32 states that
    every SSM_SPAN steps begin with."""

    __slots__ = ("x", "dt", "A", "B", "C", "skip", "z", "dt_bias", "state", "states")

    def __init__(self, x, dt, A, B, C, skip, z, dt_bias, state, states):
        self.x, self.dt, self.A, self.B, self.C = x, dt, A, B, C
        self.skip, self.z, self.dt_bias, self.state, self.states = skip, z, dt_bias, state, states


def _check_scan(x, dt, A, B, C, skip, z, dt_bias, state):
    _sequence(x, "x")
    batch, steps, dim = x.shape
    require_gpu(dt, "dt", (x.dtype,), x.shape, x.device)
    require_gpu(A, "A", (torch.float32,), None, x.device)
    if A.dim() != 2 or A.shape[0] != dim or not 1 <= A.shape[1] <= SSM_MAX_STATES:
        raise ValueError(f"A must be [{dim}, 1 to {SSM_MAX_STATES}], got {tuple(A.shape)}")
    for name, t in (("B", B), ("C", C)):
        require_gpu(t, name, (x.dtype,), (batch, steps, A.shape[1]), x.device)
    if z is not None:
        require_gpu(z, "z", (x.dtype,), x.shape, x.device)
    for name, t in (("skip", skip), ("dt_bias", dt_bias)):
        if t is not None:
            require_gpu(t, name, (torch.float32,), (dim,), x.device)
    if state is not None:
        require_gpu(state, "state", (torch.float32,), (batch, dim, A.shape[1]), x.device)


def _step(t):
    """From step to step; of one step it does not matter."""
    return t.stride(1) if t.shape[1] > 1 else 0


def _scan_args(x, dt, A, B, C, skip, z, dt_bias, state):
    strides = [s for t in (x, dt, z, B, C) for s in ((t.stride(0), _step(t)) if t is not None else (0, 0))]
    return SsmArgs(*(address(t) for t in (x, dt, z, B, C, A, skip, dt_bias, state)), *x.shape, *strides, A.shape[1], 0)


def _workspace(x, A, backward):
    size = lib().morph_ssm_workspace_bytes(*x.shape, A.shape[1], backward)
    return (_empty(size, torch.uint8, x.device) if size else None), size


def _rows_of(t):
    """_channels_last, with steps as near to each other as the kernels count (a copy if they are not)."""
    t = _channels_last(t)
    return t if t is None or _step(t) <= SSM_MAX_STEP else t.contiguous()


def _scan(inputs, train, stream):
    if stream is None:
        made = stage_calls().ssm_forward(inputs, train)
        if made is not None:
            if not train:
                return native(made)
            y, last, states = native(made)
            return y, last, SavedSelective(*_bare(*inputs), states)
    x, dt, A, B, C, skip, z, dt_bias, state = inputs
    _check_scan(*inputs)
    with running_on(x.device, stream, inputs):
        x, dt, B, C, z = (_rows_of(t) for t in (x, dt, B, C, z))
        A, skip, dt_bias, state = (whole(t) for t in (A, skip, dt_bias, state))
        batch, steps, dim = x.shape
        y = _empty(x.shape, x.dtype, x.device)
        last = _empty((batch, dim, A.shape[1]), torch.float32, x.device)
        states = _empty((batch, -(-steps // SSM_SPAN), dim, A.shape[1]), torch.float32, x.device) if train else None
        inputs = x, dt, A, B, C, skip, z, dt_bias, state
        workspace, size = _workspace(x, A, 0)
        check(lib().morph_ssm_forward(ctypes.byref(_scan_args(*inputs)), dtype_code(x.dtype), address(y), address(last),
                                      address(states), address(workspace), size, current_stream()))
        return y, last, SavedSelective(*inputs, states)


def selective_scan(x, dt, A, B, C, skip=None, z=None, dt_bias=None, state=None, stream=None):
    """(y, state behind the last step); state: the one before the first (None: zeros)."""
    return _scan((x, dt, A, B, C, skip, z, dt_bias, state), False, stream)[:2]


def selective_scan_forward(x, dt, A, B, C, skip=None, z=None, dt_bias=None, state=None, stream=None):
    """(y, last state, saved): selective_scan, with what the backward needs."""
    return _scan((x, dt, A, B, C, skip, z, dt_bias, state), True, stream)


def selective_scan_backward(dy, saved, dlast=None, stream=None):
    """(dx, ddt, dA, dB, dC, dskip, dz, ddt_bias, dstate): the gradients of selective_scan's arguments in their
    order (None for skip, z and dt_bias where there was none), from those of y and of the last state (None:
    zeros)."""
    if not isinstance(saved, SavedSelective):
        raise TypeError("saved must come from selective_scan_forward")
    inputs = tuple(getattr(saved, name) for name in SavedSelective.__slots__[:-1])
    if stream is None:
        made = stage_calls().ssm_backward(dy, inputs, saved.states, dlast)
        if made is not None:
            return native(made)
    x, dt, A, B, C, skip, z, dt_bias, state = inputs
    require_gpu(dy, "dy", (x.dtype,), x.shape, x.device)
    batch, steps, dim = x.shape
    if dlast is not None:
        require_gpu(dlast, "dlast", (torch.float32,), (batch, dim, A.shape[1]), x.device)
    with running_on(x.device, stream, (dy, *inputs, saved.states, dlast)):
        dy, dlast = _rows_of(dy), whole(dlast)

        def like(t):
            return _empty(t.shape, t.dtype, t.device) if t is not None else None

        dx, ddt, dA, dB, dC, dskip, dz, ddt_bias = (like(t) for t in inputs[:-1])
        dstate = _empty((batch, dim, A.shape[1]), torch.float32, x.device)
        grads = SsmGrads(*(address(t) for t in (dx, ddt, dz, dB, dC, dA, dskip, ddt_bias, dstate)))
        workspace, size = _workspace(x, A, 1)
        check(lib().morph_ssm_backward(ctypes.byref(_scan_args(*inputs)), dtype_code(x.dtype), address(saved.states),
                                       address(dy), dy.stride(0), _step(dy), address(dlast), ctypes.byref(grads),
                                       address(workspace), size, current_stream()))
        return dx, ddt, dA, dB, dC, dskip, dz, ddt_bias, dstate


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *inputs):
        y, last, saved = selective_scan_forward(*inputs)
        ctx.save_for_backward(*inputs, *(getattr(saved, name) for name in SavedSelective.__slots__))
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        saved = SavedSelective(*ctx.saved_tensors[9:])
        if dy is None:
            dy = torch.zeros_like(saved.x)
        *grads, dstate = selective_scan_backward(dy, saved, dlast)
        return first_order("selective_state_space", (*grads, dstate if saved.state is not None else None))


def selective_state_space(x, dt, A, B, C, skip=None, z=None, dt_bias=None, state=None):
    """selective_scan under autograd: (y, last state), differentiable once in every argument."""
    inputs = x, dt, A, B, C, skip, z, dt_bias, state
    if requires_grad("selective_state_space", *inputs):
        return _SelectiveScan.apply(*inputs)
    return selective_scan(*inputs)
