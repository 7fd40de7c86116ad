"""The gated feed-forward block of a stage (SwiGLU: gate, up, down), forward and backward.

    h = silu(x @ gate.T) * (x @ up.T),    y = h @ down.T

with the weights as the streamed engine holds them, gate and up [ff, d], down [d, ff], in FP16
or BF16 (the compute copies that FusedAdamW exports).  The kernels (csrc/ffn.hip) accumulate in
FP32 and carry the gate in the products' epilogues.

    y = gated_ffn(x, gate, up, down)                              # serving: from one token on
    y, saved = gated_ffn_forward(x, gate, up, down, keep="fp8")   # training
    dx, dgate, dup, ddown = gated_ffn_backward(dy, saved, gate, up, down)
    y = gated_feed_forward(x, gate, up, down, keep="fp8")         # the same under autograd

The weight gradients have the weights' type and shape, as StageGradients.accumulate takes them.
GatedFFN is the block as a module whose parameters carry the engine's names (gate.weight, ...).
"""
import ctypes

import torch

from ._lib import FfnBlock, FfnSaved, check, layer_calls, lib
from .activations import PackedActivation
from .layers import (GROUP, HALF, address, as_rows, current_stream, dtype_code, first_order, native,
                     require_gpu, requires_grad, row_stride, running_on)

KEEP = {"none": 0, "full": 1, "fp8": 2}


class SavedFFN:
    """What a forward kept for its backward.  keep "full": x itself and both projections in
    FP32 (gate, up: [rows, 32 G], zero behind ff); "fp8": x, gate and up as PackedActivation."""

    __slots__ = ("keep", "x", "projections", "packed", "shape", "ff", "dtype")

    def __init__(self, keep, x, projections, packed, shape, ff, dtype):
        self.keep, self.shape, self.ff, self.dtype = keep, shape, ff, dtype
        self.x, self.projections, self.packed = x, projections, packed  # of one kind or the other

    @property
    def gate(self):
        return self.packed[1] if self.keep == "fp8" else self.projections[0]

    @property
    def up(self):
        return self.packed[2] if self.keep == "fp8" else self.projections[1]

    @classmethod
    def of(cls, tensors, keep, shape, ff, dtype):
        """From tensors() and the rest."""
        if keep == "fp8":
            packed = _packings(tensors, shape, tensors[0].shape[0], ff, dtype)
            return cls(keep, packed[0], None, packed, shape, ff, dtype)
        return cls(keep, *tensors, None, shape, ff, dtype)

    def tensors(self):
        if self.keep == "fp8":
            return tuple(t for p in self.packed for t in (p.codes, p.exponents))
        return self.x, self.projections

    @property
    def device(self):
        return self.tensors()[1].device

    @property
    def nbytes(self):
        """Bytes held beyond x, or with "fp8" in all (x need not be kept beside it)."""
        if self.keep == "fp8":
            return sum(p.nbytes for p in self.packed)
        return 4 * self.projections.numel()


def _check_keep(keep):
    if keep not in ("full", "fp8"):
        raise ValueError('keep must be "full" or "fp8"')


def _weights(x, gate, up, down):
    """ff of the weights, which are checked against x."""
    require_gpu(x, "x", HALF)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("x must be [..., d] with d >= 1")
    d, device = x.shape[-1], x.device
    require_gpu(gate, "gate", (x.dtype,), None, device)
    if gate.dim() != 2 or gate.shape[1] != d or gate.shape[0] == 0:
        raise ValueError(f"gate has shape {tuple(gate.shape)}, expected [ff, {d}] with ff >= 1")
    ff = gate.shape[0]
    require_gpu(up, "up", (x.dtype,), (ff, d), device)
    require_gpu(down, "down", (x.dtype,), (d, ff), device)
    return ff


def _block(x, gate, up, down, rows, d, ff):
    return FfnBlock(address(x), address(gate), address(up), address(down), rows, d, ff,
                    row_stride(x) if x is not None else d, row_stride(gate), row_stride(up), row_stride(down))


def _descriptor(saved):
    if saved.keep == "full":
        return FfnSaved(KEEP["full"], 0, address(saved.gate), address(saved.up), None, None, None, None)
    x, gate, up = saved.packed
    return FfnSaved(KEEP["fp8"], 0, address(gate.codes), address(up.codes), address(gate.exponents),
                    address(up.exponents), address(x.codes), address(x.exponents))


def _packings(tensors, shape, rows, ff, dtype):
    """x, gate and up from their codes and exponents."""
    return tuple(PackedActivation(tensors[2 * i], tensors[2 * i + 1], s, dtype)
                 for i, s in enumerate((shape, (rows, ff), (rows, ff))))


def _forward(x, gate, up, down, keep, stream):
    if stream is None:
        made = layer_calls().ffn_forward(x, gate, up, down, KEEP[keep])
        if made is not None:
            made = native(made)
            if keep == "none":
                return made, None
            y, kept = made
            ff = gate.shape[0]
            if keep == "full":
                kept = x.detach().view(-1, x.shape[-1]), kept[0]
            return y, SavedFFN.of(kept, keep, x.shape, ff, x.dtype)
    ff = _weights(x, gate, up, down)
    d, device, dtype = x.shape[-1], x.device, x.dtype
    rows = x.numel() // d
    with running_on(device, stream, (x, gate, up, down)):
        flat, gate, up, down = (as_rows(t.detach()) for t in (x, gate, up, down))
        y = torch.empty(x.shape, dtype=dtype, device=device)
        saved = None
        if keep == "full":
            wide = -(-ff // GROUP) * GROUP
            projections = torch.empty((2, rows, wide), dtype=torch.float32, device=device)
            saved = SavedFFN.of((flat, projections), keep, x.shape, ff, dtype)
        elif keep == "fp8":
            codes = [torch.empty((rows, -(-n // GROUP) * size), dtype=torch.uint8, device=device)
                     for n in (d, ff, ff) for size in (GROUP, 1)]
            saved = SavedFFN.of(codes, keep, x.shape, ff, dtype)
        if rows:
            L = lib()
            size = L.morph_ffn_workspace_bytes(rows, d, ff, KEEP[keep], 0)
            workspace = torch.empty(size, dtype=torch.uint8, device=device)
            check(L.morph_ffn_forward(ctypes.byref(_block(flat, gate, up, down, rows, d, ff)), dtype_code(dtype),
                                      ctypes.byref(_descriptor(saved)) if saved is not None else None,
                                      address(y), d, address(workspace), size, current_stream()))
        return y, saved


def gated_ffn(x, gate, up, down, stream=None):
    """y [..., d] of x [..., d]; nothing is kept for a backward."""
    return _forward(x, gate, up, down, "none", stream)[0]


def gated_ffn_forward(x, gate, up, down, keep="full", stream=None):
    """(y, saved).  keep "full" holds the projections in FP32, so the gradients carry only the
    roundings of the matrix instructions' 16-bit operands (8 ff bytes a row, and x by reference:
    it may not change before the backward); "fp8" holds x and both projections in 8 bits, about
    d + 2 ff bytes a row, and the backward takes them for x and the projections."""
    _check_keep(keep)
    return _forward(x, gate, up, down, keep, stream)


def gated_ffn_backward(dy, saved, gate, up, down, stream=None):
    """(dx, dgate, dup, ddown) from the gradient of y and what the forward kept."""
    if not isinstance(saved, SavedFFN):
        raise TypeError("saved must come from gated_ffn_forward")
    device = saved.device
    require_gpu(dy, "dy", (saved.dtype,), saved.shape, device)
    if stream is None and isinstance(gate, torch.Tensor) and gate.shape[:1] == (saved.ff,):
        made = layer_calls().ffn_backward(dy, saved.tensors(), gate, up, down, KEEP[saved.keep])
        if made is not None:
            return native(made)
    ff = _weights(dy, gate, up, down)
    if ff != saved.ff:
        raise ValueError(f"the weights have {ff} hidden units, the forward had {saved.ff}")
    d, dtype = dy.shape[-1], dy.dtype
    rows = dy.numel() // d
    with running_on(device, stream, (dy, gate, up, down, *saved.tensors())):
        flat, gate, up, down = (as_rows(t.detach()) for t in (dy, gate, up, down))
        dx = torch.empty(saved.shape, dtype=dtype, device=device)
        dgate, dup = (torch.empty((ff, d), dtype=dtype, device=device) for _ in range(2))
        ddown = torch.empty((d, ff), dtype=dtype, device=device)
        L = lib()
        size = L.morph_ffn_workspace_bytes(rows, d, ff, KEEP[saved.keep], 1)
        workspace = torch.empty(size, dtype=torch.uint8, device=device)
        block = _block(saved.x if saved.keep == "full" else None, gate, up, down, rows, d, ff)
        check(L.morph_ffn_backward(ctypes.byref(block), dtype_code(dtype), ctypes.byref(_descriptor(saved)),
                                   address(flat), row_stride(flat), address(dx), address(dgate), address(dup),
                                   address(ddown), address(workspace), size, current_stream()))
        return dx, dgate, dup, ddown


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, up, down, keep):
        y, saved = gated_ffn_forward(x, gate, up, down, keep)
        # what was kept is autograd's to hold and release; x for its guard against changes in place
        ctx.save_for_backward(gate, up, down, x if keep == "full" else None, *saved.tensors())
        ctx.kept = keep, saved.shape, saved.ff, saved.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        gate, up, down, _, *tensors = ctx.saved_tensors
        grads = gated_ffn_backward(dy, SavedFFN.of(tensors, *ctx.kept), gate, up, down)
        return *first_order("gated_feed_forward", grads), None


def gated_feed_forward(x, gate, up, down, keep="full"):
    """gated_ffn under autograd: y, differentiable once in x and the weights.  keep: as
    gated_ffn_forward's."""
    _check_keep(keep)
    if requires_grad("gated_feed_forward", x, gate, up, down):
        return _GatedFFN.apply(x, gate, up, down, keep)
    return gated_ffn(x, gate, up, down)


class GatedFFN(torch.nn.Module):
    """The block as a module: gate, up and down as bias-free Linear layers, so a state dict has
    gate.weight, up.weight and down.weight.  keep: as gated_ffn_forward's."""

    def __init__(self, d, ff, keep="full", device=None, dtype=torch.float16):
        super().__init__()
        _check_keep(keep)
        self.gate = torch.nn.Linear(d, ff, bias=False, device=device, dtype=dtype)
        self.up = torch.nn.Linear(d, ff, bias=False, device=device, dtype=dtype)
        self.down = torch.nn.Linear(ff, d, bias=False, device=device, dtype=dtype)
        self.keep = keep

    def forward(self, x):
        return gated_feed_forward(x, self.gate.weight, self.up.weight, self.down.weight, self.keep)
