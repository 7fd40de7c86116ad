"""The float64 references of the layer operators against differences of themselves and torch
(CPU), and the C entry points' refusals."""
import ctypes

import numpy as np
import pytest
import torch

import layer_reference as R
from test_abi import no_gpu_visible


def test_e4m3_table_equals_torch():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    ours = R.e4m3_values()
    assert np.array_equal(np.isnan(codes), np.isnan(ours))
    assert np.array_equal(codes[~np.isnan(codes)], ours[~np.isnan(ours)])


def test_pack_reference_rounds_to_nearest():
    x = torch.randn(40, 70, generator=torch.Generator().manual_seed(0)) * torch.exp(torch.arange(70) / 9 - 4)
    codes, exps = R.pack(x)
    torch_codes = (torch.nn.functional.pad(x, (0, 26)) * torch.exp2(127 - torch.from_numpy(exps).float())
                   .repeat_interleave(32, 1)).to(torch.float8_e4m3fn).view(torch.uint8)
    assert np.array_equal(codes, torch_codes.numpy())
    full = torch.nn.functional.pad(x, (0, 26)).view(40, 3, 32).abs().amax(-1)
    scale = torch.exp2(torch.from_numpy(exps).float() - 127)
    assert (full <= 448 * scale).all() and (full > 224 * scale).all()


def test_ffn_reference_gradients():
    gen = torch.Generator().manual_seed(1)
    ts = [torch.randn(s, generator=gen, dtype=torch.float64).requires_grad_() for s in ((5, 6), (7, 6), (7, 6), (6, 7))]
    dy = torch.randn(5, 6, generator=gen, dtype=torch.float64)
    g, u, h, y = R.ffn(*ts)
    y.backward(dy)
    with torch.no_grad():
        ref = R.ffn_backward(dy, ts[0], g, u, *ts[1:])
    for t, name in zip(ts, ("dx", "dgate", "dup", "ddown")):
        torch.testing.assert_close(t.grad, ref[name], rtol=1e-10, atol=1e-12)


@pytest.mark.parametrize("gate", [True, False])
def test_scan_reference_gradients(gate):
    gen = torch.Generator().manual_seed(1)
    f, v, z = (torch.randn(2, 9, 3, generator=gen, dtype=torch.float64).requires_grad_() for _ in range(3))
    s0 = torch.randn(2, 3, generator=gen, dtype=torch.float64).requires_grad_()
    dy, dl = torch.randn(2, 9, 3, generator=gen, dtype=torch.float64), torch.randn(2, 3, generator=gen, dtype=torch.float64)
    y, last, _ = R.scan(f, v, z if gate else None, s0)
    torch.autograd.backward([y, last], [dy, dl])
    with torch.no_grad():
        grads = R.scan_backward(f, v, z if gate else None, s0, dy, dl)
    for t, g in zip((f, v, z, s0), grads):
        if g is not None:
            torch.testing.assert_close(t.grad, g, rtol=1e-10, atol=1e-12)


@no_gpu_visible
def test_entry_points_refuse_before_any_launch():
    from morph_amd import _lib
    lib = _lib.lib()
    p, odd = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10001)
    pack = lambda src, dtype, rows, cols, ld, codes=p, exps=p: lib.morph_act_pack(
        src, dtype, rows, cols, ld, codes, exps, None)
    assert pack(p, 7, 1, 1, 1) == -2
    assert pack(p, 1, -1, 1, 1) == -1 and pack(p, 1, 1, 8, 7) == -1 and pack(None, 1, 1, 1, 1) == -1
    assert pack(p, 1, 1, 1, 1, codes=None) == -1 and pack(p, 1, 1, 1, 1, codes=odd) == -1
    assert pack(odd, 1, 1, 1, 1) == -1 and pack(p, 1, 2, 1, 1 << 62) == -4
    assert pack(p, 1, 1 << 40, 32, 32) == -4
    assert pack(None, 1, 0, 5, 5) == 0 and pack(None, 1, 5, 0, 0) == 0
    assert lib.morph_act_unpack(p, p, 1, 1, None, 1, 1, None) == -1
    assert lib.morph_act_unpack(p, p, 1, 1, p, 3, 1, None) == -2

    def block(**kw):
        f = dict(x=0x10000, gate=0x10000, up=0x10000, down=0x10000, rows=4, d=8, ff=16, x_ld=8, gate_ld=8,
                 up_ld=8, down_ld=16)
        return _lib.FfnBlock(*dict(f, **kw).values())

    def forward(dtype=1, saved=None, y=p, y_ld=8, ws=p, size=1 << 30, **kw):
        return lib.morph_ffn_forward(ctypes.byref(block(**kw)), dtype, ctypes.byref(saved) if saved else None, y,
                                     y_ld, ws, size, None)
    assert forward(dtype=0) == -2 and forward(dtype=9) == -2
    for kw in (dict(rows=-1), dict(d=0), dict(ff=0), dict(x=None), dict(gate=None), dict(up=None), dict(down=None),
               dict(x_ld=7), dict(gate_ld=7), dict(up_ld=7), dict(down_ld=15), dict(x=0x10001), dict(down=0x10001)):
        assert forward(**kw) == -1, kw
    assert forward(rows=1 << 40) == -4 and forward(d=1 << 40, x_ld=1 << 41, gate_ld=1 << 41, up_ld=1 << 41) == -4
    assert forward(x_ld=1 << 33) == -4
    assert forward(y=None) == -1 and forward(y_ld=7) == -1 and forward(y=odd) == -1
    assert forward(ws=None) == -5 and forward(size=4 * 32 * 2 - 1) == -5 and forward(ws=ctypes.c_void_p(0x10008)) == -5
    assert forward(rows=0, x=None, y=None, ws=None) == 0
    assert lib.morph_ffn_workspace_bytes(4, 8, 16, 0, 0) == 4 * 32 * 2
    saved = lambda keep, **kw: _lib.FfnSaved(*dict(dict(keep=keep, reserved=0, gate=0x10000, up=0x10000, ge=0x10000,
                                                        ue=0x10000, xc=0x10000, xe=0x10000), **kw).values())
    assert forward(saved=saved(3)) == -1 and forward(saved=saved(-1)) == -1
    assert forward(saved=saved(1, gate=None)) == -1 and forward(saved=saved(1, up=0x10008)) == -1
    for name in ("ge", "ue", "xc", "xe"):
        assert forward(saved=saved(2, **{name: None})) == -1

    def backward(dtype=1, keep=1, dy=p, dy_ld=8, outs=(p, p, p, p), ws=p, size=1 << 30, **kw):
        return lib.morph_ffn_backward(ctypes.byref(block(**kw)), dtype, ctypes.byref(saved(keep)), dy, dy_ld, *outs,
                                      ws, size, None)
    assert backward(keep=0) == -1 and backward(dy=None) == -1 and backward(dy_ld=7) == -1 and backward(dtype=0) == -2
    for i in range(4):
        assert backward(outs=[None if j == i else p for j in range(4)]) == -1
        assert backward(outs=[odd if j == i else p for j in range(4)]) == -1
    assert backward(ws=None) == -5 and backward(size=16) == -5
    assert lib.morph_ffn_backward(ctypes.byref(block()), 1, None, p, 8, p, p, p, p, p, 1 << 30, None) == -1

    scan = lambda **kw: _lib.ScanArgs(*dict(dict(f=0x10000, v=0x10000, z=0x10000, s0=0x10000, batch=2, steps=3, dim=4,
                                                 fb=12, fs=4, vb=12, vs=4, zb=12, zs=4), **kw).values())
    run = lambda a, dtype=0, y=p: lib.morph_scan_forward(ctypes.byref(a), dtype, y, p, None, p, 1 << 30, None)
    assert run(scan(), dtype=5) == -2 and run(scan(batch=-1)) == -1 and run(scan(steps=-1)) == -1
    assert run(scan(f=None)) == -1 and run(scan(v=None)) == -1 and run(scan(), y=None) == -1
    assert run(scan(batch=1 << 20)) == -4 and run(scan(dim=1 << 40)) == -4 and run(scan(steps=1 << 50)) == -4
    assert lib.morph_scan_forward(None, 0, p, p, None, p, 1 << 30, None) == -1
    assert run(scan(batch=0, f=None, v=None), y=None) == 0
    back = lambda a, states=p, dy=p, df=p, dv=p, dz=p: lib.morph_scan_backward(
        ctypes.byref(a), 0, states, dy, 12, 4, None, df, dv, dz, p, p, 1 << 30, None)
    for kw in (dict(states=None), dict(dy=None), dict(df=None), dict(dv=None), dict(dz=None)):
        assert back(scan(), **kw) == -1, kw


@pytest.mark.parametrize("cls,ctype", [("FfnBlock", "morph_ffn"), ("FfnSaved", "morph_ffn_saved"),
                                       ("ScanArgs", "morph_scan")])
def test_layer_struct_layouts_match_the_header(tmp_path, cls, ctype):
    import shutil
    import subprocess
    from pathlib import Path

    from morph_amd import _lib
    if shutil.which("gcc") is None:
        pytest.skip("needs a host C compiler")
    struct = getattr(_lib, cls)
    fields = [name for name, *_ in struct._fields_]
    source = ['#include <stdio.h>', '#include <stddef.h>', '#include "morph_layers.h"', 'int main(void) {',
              f'printf("%zu\\n", sizeof({ctype}));', *(f'printf("%zu\\n", offsetof({ctype}, {n}));' for n in fields),
              'printf("%d %d\\n", MORPH_SCAN_SPAN, MORPH_ACT_GROUP);', 'return 0; }']
    (tmp_path / "layout.c").write_text("\n".join(source))
    root = Path(__file__).resolve().parents[1]
    subprocess.run(["gcc", "-std=c11", "-I", str(root / "include"), "-o", str(tmp_path / "layout"),
                    str(tmp_path / "layout.c")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out[:-2]] == [ctypes.sizeof(struct), *(getattr(struct, n).offset for n in fields)]
    assert [int(v) for v in out[-2:]] == [_lib.SCAN_SPAN, 32]


@no_gpu_visible
def test_wrappers_refuse_host_tensors():
    """A CPU tensor raises the wrappers' own error, with or without a GPU in the machine."""
    from morph_amd.activations import pack_activation
    from morph_amd.ffn import gated_ffn
    from morph_amd.recurrence import gated_scan
    x = torch.zeros(4, 8, dtype=torch.float16)
    for call in (lambda: pack_activation(x), lambda: gated_ffn(x, x, x, x.t()), lambda: gated_scan(x[None], x[None])):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError):
        pack_activation(None)
