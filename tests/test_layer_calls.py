"""What the layer operators' wrappers do before and around their launches, with the launches taken
out, on the CPU."""
import contextlib
import ctypes
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from morph_amd import _lib, activations, ffn, layers, recurrence
from test_abi import no_gpu_visible


class _Library:
    """Entry points that launch nothing and succeed; workspaces of no bytes."""

    def __getattr__(self, name):
        return lambda *args: 0


class _NoNativePath:
    def __getattr__(self, name):
        return lambda *args: None


class _Copies(TorchDispatchMode):
    """Notes for every copy of a tensor whether it was made on the call's stream."""

    def __init__(self, place):
        super().__init__()
        self.place, self.made = place, []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.overloadpacket in (torch.ops.aten.clone, torch.ops.aten.copy_, torch.ops.aten._to_copy):
            self.made.append(self.place["entered"])
        return func(*args, **(kwargs or {}))


@pytest.fixture
def wrappers(monkeypatch):
    """The wrappers on CPU tensors: {"entered": whether the call's stream is current, "inputs": the
    storages that were kept alive for it}."""
    place = {"entered": False, "inputs": set()}

    @contextlib.contextmanager
    def running_on(device, stream, inputs=()):
        place["inputs"] |= {t.untyped_storage().data_ptr() for t in inputs if t is not None}
        place["entered"] = True
        yield
        place["entered"] = False

    def require(t, name, dtypes=None, shape=None, device=None):
        assert shape is None or tuple(t.shape) == tuple(shape)
        return t
    for module in (activations, ffn, recurrence):
        monkeypatch.setattr(module, "running_on", running_on)
        monkeypatch.setattr(module, "require_gpu", require)
        monkeypatch.setattr(module, "lib", _Library)
        monkeypatch.setattr(module, "layer_calls", _NoNativePath)
        monkeypatch.setattr(module, "current_stream", lambda: None)
    return place


def _ffn_inputs(rows=5, d=16, ff=24):
    half = torch.float16
    x, dy = torch.zeros(d, rows, dtype=half).t(), torch.zeros(1, d, dtype=half).expand(rows, d)
    return x, dy, [torch.zeros(d, ff, dtype=half).t(), torch.zeros(1, d, dtype=half).expand(ff, d),
                   torch.zeros(ff, d, dtype=half).t()]


@pytest.mark.parametrize("keep", ["full", "fp8"])
def test_ffn_copies_its_operands_on_the_calls_stream(wrappers, keep):
    """Views that are no rows are copied; a copy made on the stream that is current outside the call
    would not be ordered with the kernels that read it, nor with what wrote the view."""
    x, dy, weights = _ffn_inputs()
    for call in (lambda: ffn.gated_ffn(x, *weights, stream=object()),
                 lambda: ffn.gated_ffn_forward(x, *weights, keep=keep, stream=object())):
        wrappers["inputs"].clear()
        with _Copies(wrappers) as copies:
            call()
        assert copies.made == [True] * 4
        assert {t.untyped_storage().data_ptr() for t in (x, *weights)} <= wrappers["inputs"]
    _, saved = ffn.gated_ffn_forward(x, *weights, keep=keep, stream=object())
    wrappers["inputs"].clear()
    with _Copies(wrappers) as copies:
        ffn.gated_ffn_backward(dy, saved, *weights, stream=object())
    assert copies.made == [True] * 4
    assert {t.untyped_storage().data_ptr() for t in (dy, *weights)} <= wrappers["inputs"]


def test_other_operators_copy_on_the_calls_stream(wrappers):
    x = torch.zeros(16, 5).t()
    with _Copies(wrappers) as copies:
        activations.pack_activation(x, stream=object())
    assert copies.made == [True]
    f = torch.zeros(2, 16, 5).transpose(1, 2)
    state = torch.zeros(16, 2).t()
    with _Copies(wrappers) as copies:
        _, _, saved = recurrence.gated_scan_forward(f, f, f, state, stream=object())
    assert copies.made == [True] * 4
    with _Copies(wrappers) as copies:
        recurrence.gated_scan_backward(f, saved, state, stream=object())
    assert copies.made == [True] * 2


@no_gpu_visible
def test_saturate_is_unpacks_alone():
    """MORPH_ACT_SATURATE goes with a dtype that there is, and with the unpack."""
    header = (Path(__file__).resolve().parents[1] / "include" / "morph_layers.h").read_text()
    assert f"#define MORPH_ACT_SATURATE {_lib.ACT_SATURATE:#x}\n" in header
    p = ctypes.c_void_p(0x10000)
    for dtype in (-1, 3, _lib.ACT_SATURATE | 3, 0x200):
        assert _lib.lib().morph_act_unpack(p, p, 1, 1, p, dtype, 1, None) == -2
    assert _lib.lib().morph_act_unpack(p, p, 0, 1, p, _lib.ACT_SATURATE | 1, 1, None) == 0
    assert _lib.lib().morph_act_pack(p, _lib.ACT_SATURATE | 1, 1, 1, 1, p, p, None) == -2


def test_a_stream_of_another_device_is_refused():
    """Launched there, the kernels would read this device's memory from the other one."""
    there = SimpleNamespace(device=torch.device("cuda", 1))
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        layers.running_on(torch.device("cuda", 0), there)
    layers.running_on(torch.device("cuda", 1), there)


@no_gpu_visible
def test_grids_past_the_launch_limit_are_refused():
    """A launch has fewer than 2^32 threads along a dimension: more are MORPH_ERANGE, with nothing enqueued,
    not a launch that fails behind another one (a recurrence's first kernel clears its workspace)."""
    lib, p = _lib.lib(), ctypes.c_void_p(0x10000)
    for dtype in (0, 1, 2):
        for rows in (1 << 34, (1 << 32) + 1):  # 2^24 workgroups and more of 256 groups
            assert lib.morph_act_pack(p, dtype, rows, 1, 1, p, p, None) == -4
            assert lib.morph_act_unpack(p, p, rows, 1, p, dtype, 1, None) == -4
        for batch, steps, dim in ((65535, 16640, 8), (65535, 1 << 20, 1), (1, 1 << 31, 130), (4096, 1 << 19, 64)):
            args = _lib.ScanArgs(0x10000, 0x10000, 0x10000, None, batch, steps, dim, *[steps * dim, dim] * 3)
            assert lib.morph_scan_forward(ctypes.byref(args), dtype, p, p, p, p, 1 << 50, None) == -4
            assert lib.morph_scan_backward(ctypes.byref(args), dtype, p, p, steps * dim, dim, None, p, p, p, p, p,
                                           1 << 50, None) == -4


def test_gradients_under_create_graph_take_changes_in_place():
    """They are scaled and clipped as others are, share the kernels' memory, and still raise."""
    given = torch.ones(3), None, torch.ones(2)
    grads = layers.first_order("operator", given)
    assert grads[1] is None and grads[0].data_ptr() == given[0].data_ptr()
    with torch.no_grad():
        grads[0].mul_(2)
    scaled = grads[2].mul_(3)
    assert (given[0] == 2).all() and (given[2] == 3).all()
    for g in (grads[0], scaled):
        with pytest.raises(RuntimeError, match="operator can be differentiated once"):
            g.sum().backward()
    with torch.no_grad():
        assert layers.first_order("operator", given) is given
