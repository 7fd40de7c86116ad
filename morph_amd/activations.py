"""Activation checkpoints in 8 bits: what a stage keeps between its forward and its backward.

The streamed engine keeps one boundary activation per stage and micro-batch from the forward to
the replayed backward (disk.py:365-396), on the device or on the host.  pack_activation holds
one in 33/64 of its 16 bits: E4M3 codes with a power-of-two scale per 32 consecutive values of a
row (csrc/act8.hip), relative error 2^-4 at most within 2^14 of a group's largest value.  The topmost
values of a type (FP16's from 63488 on) are nearest to a code beyond its range; back in that type they are
its largest value.
gated_ffn_forward(keep="fp8") keeps its own activations the same way.

A value that is not finite is held as NaN and comes back as NaN: in a step under a dynamic loss
scale it reaches the gradients, and the detector skips the step.
"""
import torch

from ._lib import ACT_SATURATE, check, layer_calls, lib
from .layers import (GROUP, address, as_rows, current_stream, dtype_code, native, require_gpu, row_stride,
                     running_on)

FLOATS = (torch.float32, torch.float16, torch.bfloat16)


class PackedActivation:
    """codes: uint8 [rows, 32 G] (zeros behind the last value), exponents: uint8 [rows, G] with
    G = ceil(cols / 32); the value of a code is E4M3(code) * 2^(exponent - 127).  shape and
    dtype are those of the activation.  to() moves it, also between host and device."""

    __slots__ = ("codes", "exponents", "shape", "dtype")

    def __init__(self, codes, exponents, shape, dtype):
        self.codes, self.exponents = codes, exponents
        self.shape, self.dtype = shape if type(shape) is torch.Size else torch.Size(shape), dtype

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self):
        return self.codes.numel() + self.exponents.numel()

    def to(self, device, non_blocking=False):
        return PackedActivation(self.codes.to(device, non_blocking=non_blocking),
                                self.exponents.to(device, non_blocking=non_blocking),
                                self.shape, self.dtype)


def pack_activation(x, stream=None):
    """The 8-bit form of x ([..., cols], FP32, FP16 or BF16), scaled in groups along its last
    dimension."""
    if stream is None:
        made = layer_calls().pack(x)
        if made is not None:
            codes, exponents = native(made)
            return PackedActivation(codes, exponents, x.shape, x.dtype)
    require_gpu(x, "x", FLOATS)
    if x.dim() == 0:
        raise ValueError("x must have at least one dimension")
    with running_on(x.device, stream, (x,)):
        cols = x.shape[-1]
        rows = x.numel() // cols if cols else 0
        groups = -(-cols // GROUP)
        codes = torch.empty((rows, groups * GROUP), dtype=torch.uint8, device=x.device)
        exponents = torch.empty((rows, groups), dtype=torch.uint8, device=x.device)
        if rows:
            flat = as_rows(x.detach())
            check(lib().morph_act_pack(address(flat), dtype_code(x.dtype), rows, cols, row_stride(flat),
                                       address(codes), address(exponents), current_stream()))
        return PackedActivation(codes, exponents, x.shape, x.dtype)


def unpack_activation(packed, dtype=None, stream=None):
    """The activation that `packed` stands for, contiguous: in its own dtype, where what was finite comes
    back finite, or converted to `dtype` as a cast converts it (beyond that type's range: infinite)."""
    if not isinstance(packed, PackedActivation):
        raise TypeError("packed must be a PackedActivation")
    saturate = ACT_SATURATE if dtype is None else 0
    dtype = packed.dtype if dtype is None else dtype
    if dtype not in FLOATS:
        raise TypeError(f"unsupported dtype {dtype}; expected float32, float16 or bfloat16")
    if stream is None:
        out = layer_calls().unpack(packed.codes, packed.exponents, packed.shape, dtype_code(dtype) | saturate)
        if out is not None:
            return native(out)
    cols = packed.shape[-1]
    rows = packed.shape.numel() // cols if cols else 0
    groups = -(-cols // GROUP)
    codes = require_gpu(packed.codes, "codes", (torch.uint8,), (rows, groups * GROUP))
    exponents = require_gpu(packed.exponents, "exponents", (torch.uint8,), (rows, groups), codes.device)
    if not (codes.is_contiguous() and exponents.is_contiguous()):
        raise ValueError("codes and exponents must be contiguous")
    with running_on(codes.device, stream, (codes, exponents)):
        out = torch.empty(packed.shape, dtype=dtype, device=codes.device)
        if rows:
            check(lib().morph_act_unpack(address(codes), address(exponents), rows, cols, address(out),
                                         dtype_code(dtype) | saturate, cols, current_stream()))
        return out
