"""What the state space operators refuse, and what their wrappers do around the launches, on the CPU."""
import contextlib
import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from morph_amd import _lib, norm, selective
from test_abi import no_gpu_visible
from test_layer_calls import _Copies, _Library, _NoNativePath

ROOT = Path(__file__).resolve().parents[1]
P = 0x10000  # never allocated: only where no GPU is visible, and nothing is launched
EINVAL, EDTYPE, ERANGE, EWORKSPACE = -1, -2, -4, -5


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a host C compiler")
def test_struct_layouts_match_the_headers(tmp_path):
    pairs = [("NormArgs", "morph_norm"), ("ConvArgs", "morph_conv"), ("SsmArgs", "morph_ssm"),
             ("SsmGrads", "morph_ssm_grads"), ("MomentValues", "morph_moment_values")]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "morph_state_space.h"', "int main(void) {"]
    for cls, name in pairs:
        lines.append(f'  printf("{cls} size %zu\\n", sizeof({name}));')
        for field, _ in getattr(_lib, cls)._fields_:
            lines.append(f'  printf("{cls} {field} %zu\\n", offsetof({name}, {field}));')
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-I", str(ROOT / "include"), "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")],
                   check=True)
    for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines():
        cls, field, value = line.split()
        struct = getattr(_lib, cls)
        assert (ctypes.sizeof(struct) if field == "size" else getattr(struct, field).offset) == int(value), (cls, field)


def test_constants_match_the_headers():
    text = "".join((ROOT / "include" / h).read_text() for h in ("morph_state_space.h", "morph_optim.h"))
    for name, value in (("MORPH_SSM_SPAN", _lib.SSM_SPAN), ("MORPH_SSM_MAX_STATES", _lib.SSM_MAX_STATES),
                        ("MORPH_CONV_MAX_TAPS", _lib.CONV_MAX_TAPS), ("MORPH_MOMENT_GROUP", _lib.MOMENT_GROUP)):
        assert re.search(rf"#define {name} {value}\b", text), name


@no_gpu_visible
def test_norm_refuses_before_any_launch():
    lib, p = _lib.lib(), ctypes.c_void_p(P)

    def args(rows=4, cols=8, ld=8, eps=1e-5, wdtype=0, x=P):
        return ctypes.byref(_lib.NormArgs(x, P, P, rows, cols, ld, eps, wdtype))

    def forward(a, dtype=1, y=p):
        return lib.morph_norm_forward(a, dtype, y, None, None)

    def backward(a, dtype=1, stats=p, dy=p, ld=8, ws=p, size=1 << 40):
        return lib.morph_norm_backward(a, dtype, stats, dy, ld, p, p, p, ws, size, None)
    for call in (forward, backward):
        assert call(args(), dtype=7) == EDTYPE and call(args(wdtype=2)) == EDTYPE
        assert call(None) == EINVAL and call(args(rows=-1)) == EINVAL and call(args(cols=-1)) == EINVAL
        assert call(args(eps=-1.0)) == EINVAL and call(args(eps=float("nan"))) == EINVAL
        assert call(args(ld=7)) == EINVAL and call(args(x=None)) == EINVAL
    assert forward(args(), y=None) == EINVAL and forward(args(rows=0)) == 0 and forward(args(cols=0)) == 0
    assert backward(args(), stats=None) == EINVAL and backward(args(), dy=None) == EINVAL and backward(args(), ld=7) == EINVAL
    need = lib.morph_norm_workspace_bytes(4, 8)
    assert backward(args(), size=need - 1) == EWORKSPACE and backward(args(), ws=None) == EWORKSPACE
    assert backward(args(cols=1 << 33, ld=1 << 33), ld=1 << 33, size=1 << 60) == ERANGE


@no_gpu_visible
def test_conv_refuses_before_any_launch():
    lib, p = _lib.lib(), ctypes.c_void_p(P)

    def args(batch=2, steps=5, dim=8, taps=4, wdtype=0, x=P, w=P):
        return ctypes.byref(_lib.ConvArgs(x, P, w, P, batch, steps, dim, steps * dim, dim, taps, wdtype))

    def forward(a, dtype=1, y=p, after=p):
        return lib.morph_conv_forward(a, dtype, y, after, None)

    def backward(a, dtype=1, dy=p, dw=p, ws=p, size=1 << 40):
        return lib.morph_conv_backward(a, dtype, dy, 40, 8, p, p, dw, p, p, ws, size, None)
    for call in (forward, backward):
        assert call(args(), dtype=-1) == EDTYPE and call(args(wdtype=2)) == EDTYPE and call(None) == EINVAL
        assert call(args(taps=1)) == ERANGE and call(args(taps=5)) == ERANGE and call(args(steps=-1)) == EINVAL
        assert call(args(x=None)) == EINVAL and call(args(w=None)) == EINVAL
    assert forward(args(), y=None) == EINVAL and forward(args(), after=None) == EINVAL
    assert forward(args(batch=1 << 20, steps=1 << 30)) == ERANGE and forward(args(batch=0)) == 0
    assert backward(args(), dy=None) == EINVAL and backward(args(), dw=None) == EINVAL
    assert backward(args(), size=lib.morph_conv_workspace_bytes(2, 5, 8, 4) - 1) == EWORKSPACE
    assert backward(args(), ws=None) == EWORKSPACE


@no_gpu_visible
def test_scan_refuses_before_any_launch():
    lib, p = _lib.lib(), ctypes.c_void_p(P)

    def args(batch=2, steps=5, dim=8, n=16, x=P, A=P, B=P, reserved=0):
        return ctypes.byref(_lib.SsmArgs(x, P, P, B, P, A, P, P, P, batch, steps, dim, *[steps * dim, dim] * 3,
                                         *[steps * n, n] * 2, n, reserved))
    full = [P] * 9

    def forward(a, dtype=1, y=p, last=p, ws=p, size=1 << 60):
        return lib.morph_ssm_forward(a, dtype, y, last, p, ws, size, None)

    def backward(a, dtype=1, kept=p, dy=p, grads=full, ws=p, size=1 << 60):
        grads = ctypes.byref(_lib.SsmGrads(*grads)) if grads else None
        return lib.morph_ssm_backward(a, dtype, kept, dy, 40, 8, p, grads, ws, size, None)
    for call in (forward, backward):
        assert call(args(), dtype=3) == EDTYPE and call(None) == EINVAL and call(args(reserved=1)) == EINVAL
        assert call(args(n=0)) == ERANGE and call(args(n=65)) == ERANGE and call(args(dim=-1)) == EINVAL
        assert call(args(x=None)) == EINVAL and call(args(A=None)) == EINVAL and call(args(B=None)) == EINVAL
        assert call(args(batch=1 << 20, dim=1 << 20, steps=1 << 20)) == ERANGE
    assert forward(args(), y=None) == EINVAL and forward(args(), last=None) == EINVAL and forward(args(batch=0)) == 0
    assert forward(args(batch=1 << 20, dim=1 << 10)) == ERANGE  # 2^26 workgroups of 512
    assert backward(args(), kept=None) == EINVAL and backward(args(), dy=None) == EINVAL
    assert backward(args(), grads=None) == EINVAL
    for k in range(8):  # all but dfirst
        assert backward(args(), grads=[None if i == k else P for i in range(9)]) == EINVAL, k
    assert backward(args(), size=lib.morph_ssm_workspace_bytes(2, 5, 8, 16, 1) - 1) == EWORKSPACE
    assert lib.morph_ssm_workspace_bytes(2, 5, 8, 16, 0) == 0 < lib.morph_ssm_workspace_bytes(1, 1000, 64, 16, 0)
    assert forward(args(1, 1000, 64), size=lib.morph_ssm_workspace_bytes(1, 1000, 64, 16, 0) - 1) == EWORKSPACE
    assert forward(args(1, 1000, 64), ws=None) == EWORKSPACE
    assert forward(args(dim=(1 << 25) + 1)) == ERANGE and forward(args(steps=(1 << 31) - 1, dim=1)) == ERANGE
    assert backward(args(), ws=None) == EWORKSPACE


@no_gpu_visible
def test_moments_refuse_before_any_launch():
    lib = _lib.lib()
    t = (_lib.MomentValues * 1)(_lib.MomentValues(P, P, P, P, 64))
    call = lib.morph_moment_decode
    assert call(t, 1, 9, None) == EDTYPE and call(t, -1, 0, None) == EINVAL and call(None, 1, 0, None) == EINVAL
    for k in range(4):
        bad = [P] * 4
        bad[k] = None
        assert call((_lib.MomentValues * 1)(_lib.MomentValues(*bad, 64)), 1, 0, None) == EINVAL
    assert call((_lib.MomentValues * 1)(_lib.MomentValues(P + 2, P, P, P, 64)), 1, 0, None) == EINVAL
    assert call((_lib.MomentValues * 1)(_lib.MomentValues(P, P, P, P, (1 << 30) + 1)), 1, 0, None) == ERANGE
    assert call(t, 0, 0, None) == 0
    hp, sched = _lib.AdamwHP(), _lib.AdamwSched(0.1, P, P, 5)
    state = ctypes.c_void_p(P)

    def step(m=P, n=64):
        d = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(P, P, m, P, None, n, 0, 0))
        return [lib.morph_adamw8_multi_dev(d, 1, 1, -1, ctypes.byref(hp), ctypes.byref(sched), 1, state, state, 0, None, None, None),
                lib.morph_adamw8_table_dev(state, d, 1, 1, -1, ctypes.byref(hp), ctypes.byref(sched), 1, state, state, 0, None,
                                           None, None)]
    assert step(m=P + 1) == [EINVAL] * 2 and step(n=(1 << 30) + 1) == [ERANGE] * 2 and step(m=None)[0] == EINVAL


def test_wrappers_refuse_what_is_not_theirs():
    x = torch.zeros(2, 5, 8)
    for call in (lambda: norm.layer_norm(x), lambda: selective.causal_conv(x, torch.zeros(8, 4)),
                 lambda: selective.selective_scan(x, x, torch.zeros(8, 16), x, x)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    for call in (lambda: norm.layer_norm(3), lambda: selective.causal_conv(None, None),
                 lambda: selective.selective_scan([], x, x, x, x)):
        with pytest.raises(TypeError, match="must be a tensor"):
            call()
    for call in (lambda: norm.layer_norm_backward(x, x), lambda: selective.causal_conv_backward(x, x),
                 lambda: selective.selective_scan_backward(x, x)):
        with pytest.raises(TypeError, match="must come from"):
            call()


@pytest.fixture
def wrappers(monkeypatch):
    """The wrappers on CPU tensors, without launches: see test_layer_calls."""
    place = {"entered": False, "inputs": set()}

    @contextlib.contextmanager
    def running_on(device, stream, inputs=()):
        place["inputs"] |= {t.untyped_storage().data_ptr() for t in inputs if t is not None}
        place["entered"] = True
        yield
        place["entered"] = False

    def require(t, name, dtypes=None, shape=None, device=None):
        if dtypes is not None and t.dtype not in dtypes:
            raise TypeError(name)
        if shape is not None and tuple(t.shape) != tuple(shape):
            raise ValueError(name)
        return t
    for module in (norm, selective):
        monkeypatch.setattr(module, "running_on", running_on)
        monkeypatch.setattr(module, "require_gpu", require)
        monkeypatch.setattr(module, "lib", _Library)
        monkeypatch.setattr(module, "current_stream", lambda: None)
        monkeypatch.setattr(module, "stage_calls", _NoNativePath)
    return place


def test_copies_are_made_on_the_calls_stream(wrappers):
    x, w = torch.zeros(8, 6).t(), torch.zeros(16)[::2]
    with _Copies(wrappers) as copies:
        _, saved = norm.layer_norm_forward(x, w, w, stream=object())
        norm.layer_norm_backward(x, saved, stream=object())
    assert copies.made and all(copies.made)
    assert {x.untyped_storage().data_ptr(), w.untyped_storage().data_ptr()} <= wrappers["inputs"]
    x, taps, state = torch.zeros(2, 8, 5).transpose(1, 2), torch.zeros(4, 8).t(), torch.zeros(2, 8, 3).transpose(1, 2)
    with _Copies(wrappers) as copies:
        _, _, saved = selective.causal_conv_forward(x, taps, w, state, stream=object())
        selective.causal_conv_backward(x, saved, state, stream=object())
    assert len(copies.made) >= 5 and all(copies.made)
    B, first = torch.zeros(2, 4, 5).transpose(1, 2), torch.zeros(2, 4, 8).transpose(1, 2)
    with _Copies(wrappers) as copies:
        _, _, saved = selective.selective_scan_forward(x, x, taps, B, B, w, x, w, first, stream=object())
        selective.selective_scan_backward(x, saved, first, stream=object())
    assert len(copies.made) >= 9 and all(copies.made)


def test_wrappers_refuse_shapes_and_types(wrappers):
    x, half = torch.zeros(2, 5, 8), torch.zeros(2, 5, 8).half()
    A, B = torch.zeros(8, 16), torch.zeros(2, 5, 16)
    good = dict(x=x, dt=x, A=A, B=B, C=B)
    selective.selective_scan(**good)
    for name, bad in (("x", x[0]), ("dt", x[:, :4]), ("A", A[:, :0]), ("A", torch.zeros(8, 65)), ("A", torch.zeros(7, 16)),
                      ("B", B[..., :15]), ("C", B[:1]), ("z", x[:1]), ("skip", A[0]), ("dt_bias", A[0]),
                      ("state", torch.zeros(2, 8, 15))):
        with pytest.raises(ValueError):
            selective.selective_scan(**{**good, name: bad})
    for name, bad in (("dt", half), ("A", A.half()), ("B", B.half()), ("z", half), ("skip", torch.zeros(8).half()),
                      ("state", torch.zeros(2, 8, 16).half())):
        with pytest.raises(TypeError):
            selective.selective_scan(**{**good, name: bad})
    w = torch.zeros(8, 4)
    for bad in (w[:7], w[:, :1], torch.zeros(8, 5), w[0]):
        with pytest.raises(ValueError):
            selective.causal_conv(x, bad)
    with pytest.raises(ValueError):
        selective.causal_conv(x, w, state=torch.zeros(2, 4, 8))
    with pytest.raises(TypeError):
        selective.causal_conv(half, w, torch.zeros(8).half())
    with pytest.raises(ValueError, match="eps"):
        norm.layer_norm(x, eps=-1)
    with pytest.raises(TypeError, match="one type"):
        norm.layer_norm(half, torch.zeros(8), torch.zeros(8).half())
    with pytest.raises(ValueError):
        norm.layer_norm(x, torch.zeros(7))
    with pytest.raises(ValueError, match="at least one dimension"):
        norm.layer_norm(torch.zeros(()))
