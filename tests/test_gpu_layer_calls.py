"""Calls of the layer operators as users make them: on another stream, under autograd, at the ends
of a type's range, and with what they refuse."""
import math

import pytest
import torch
from torch.autograd import forward_ad

import layer_reference as R
from morph_amd.activations import pack_activation, unpack_activation
from morph_amd.ffn import gated_feed_forward, gated_ffn, gated_ffn_backward, gated_ffn_forward
from morph_amd.recurrence import gated_recurrence, gated_scan, gated_scan_backward, gated_scan_forward

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def normal(gen, *shape, scale=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen) * scale + mean).to(dtype)


@pytest.mark.parametrize("keep", ["full", "fp8"])
def test_ffn_views_written_on_the_calls_stream(keep):
    """Weights that are no rows (transposed, expanded), written on the call's stream behind other work:
    the copies that the kernels read are made in that stream's order, not in the current one's."""
    gen = torch.Generator().manual_seed(21)
    rows, d, ff, dtype = 130, 96, 160, torch.bfloat16
    x, dy = (normal(gen, rows, d, dtype=dtype).to(DEV) for _ in range(2))
    sources = [normal(gen, d, ff, scale=d ** -.5, dtype=dtype).to(DEV), normal(gen, 1, d, scale=d ** -.5, dtype=dtype).to(DEV),
               normal(gen, ff, d, scale=ff ** -.5, dtype=dtype).to(DEV)]

    def views(gate, up, down):
        return gate.t(), up.expand(ff, d), down.t()
    copies = [w.contiguous() for w in views(*sources)]
    y, saved = gated_ffn_forward(x, *copies, keep=keep)
    grads = gated_ffn_backward(dy, saved, *copies)
    work = torch.randn(4096, 4096, device=DEV)
    side = torch.cuda.Stream()
    for _ in range(3):
        written = [torch.zeros_like(s) for s in sources]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(4):
                work @ work
            for w, s in zip(written, sources):
                w.copy_(s)
        got, kept = gated_ffn_forward(x, *views(*written), keep=keep, stream=side)
        served = gated_ffn(x, *views(*written), stream=side)
        with torch.cuda.stream(side):  # written anew between the calls
            for w in written:
                w.zero_()
            for _ in range(4):
                work @ work
            for w, s in zip(written, sources):
                w.copy_(s)
        back = gated_ffn_backward(dy, kept, *views(*written), stream=side)
        side.synchronize()
        assert torch.equal(got, y) and torch.equal(served, gated_ffn(x, *copies))
        assert all(torch.equal(a, b) for a, b in zip(back, grads))


# ---- the top of a type's range in 8 bits ----------------------------------------
def _top_values(dtype, gen, rows, cols):
    """Values of the type's last two binades, either sign, some that are not finite; a row that holds its
    largest value only, and one far below."""
    x = (torch.rand(rows, cols, generator=gen, dtype=torch.float64) * .75 + .25) * torch.finfo(dtype).max
    x[torch.rand(rows, cols, generator=gen) < .5] *= -1
    x = x.to(dtype)
    bad = torch.rand(rows, cols, generator=gen)
    for k, value in enumerate((math.nan, math.inf, -math.inf)):
        x[(bad > .01 * k) & (bad < .01 * (k + 1))] = value
    x[0], x[-1] = torch.finfo(dtype).max, 1.0
    return x


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(3, 40), (7, 64), (5, 37), (20000, 1024), (20001, 1021)])
def test_unpacked_in_its_own_type_the_finite_stays_finite(dtype, rows, cols):
    x = _top_values(dtype, torch.Generator().manual_seed(rows), rows, cols).to(DEV)
    packed = pack_activation(x)
    out = unpack_activation(packed)
    assert torch.equal(out.isfinite(), x.isfinite()) and torch.equal(out.isnan(), ~x.isfinite())
    fine = x.isfinite()
    assert ((out - x).abs()[fine] <= x.abs()[fine] / 16).all()
    assert (out[0] == torch.finfo(dtype).max).all() and (out[-1] == 1).all()
    assert torch.equal(unpack_activation(packed, stream=torch.cuda.current_stream()).nan_to_num(7.0), out.nan_to_num(7.0))
    # another type asked for: a cast, and what lies beyond its range is infinite
    wide = unpack_activation(packed, torch.float16)
    assert torch.isinf(wide[0]).all()
    if dtype == torch.float16:
        assert (unpack_activation(packed, torch.float32)[0] == 65536).all()


@pytest.mark.parametrize("rows", [5, 300])
def test_ffn_kept_in_8_bits_takes_the_top_of_fp16(rows):
    """x near 65504, kept in 8 bits: finite gradients, those of the formula on x saturated."""
    gen = torch.Generator().manual_seed(23)
    d, ff, dtype = 72, 104, torch.float16
    x = normal(gen, rows, d, dtype=dtype)
    x[2, 3], x[3, 50], x[1, 71] = 65504, -63488, 64000
    weights = [normal(gen, ff, d, scale=2.0 ** -14, dtype=dtype), normal(gen, ff, d, scale=2.0 ** -14, dtype=dtype),
               normal(gen, d, ff, scale=ff ** -.5, dtype=dtype)]
    dy = normal(gen, rows, d, scale=2.0 ** -7, dtype=dtype)
    dev = [w.to(DEV) for w in weights]
    y, saved = gated_ffn_forward(x.to(DEV), *dev, keep="fp8")
    dx, dgate, dup, ddown = gated_ffn_backward(dy.to(DEV), saved, *dev)
    assert all(t.isfinite().all() for t in (y, dx, dgate, dup, ddown))
    xk, g, u = (R.unpack(p.codes, p.exponents, p.shape[-1]) for p in (saved.x, saved.gate, saved.up))
    assert xk.abs().max() == 65536
    ref = R.ffn_backward(dy.double(), xk.clamp(-65504, 65504), g, u, *(w.double() for w in weights))
    R.assert_product(dgate, ref["dg"].T, xk.clamp(-65504, 65504), dtype, "dgate")
    R.assert_product(dup, ref["du"].T, xk.clamp(-65504, 65504), dtype, "dup")


# ---- derivatives ------------------------------------------------------------------
def _differentiable(kind):
    """An operator as a function of tensors, and the tensors."""
    gen = torch.Generator().manual_seed(29)
    if kind in ("full", "fp8"):
        tensors = [normal(gen, 5, 64, dtype=torch.bfloat16), normal(gen, 96, 64, scale=.1, dtype=torch.bfloat16),
                   normal(gen, 96, 64, scale=.1, dtype=torch.bfloat16), normal(gen, 64, 96, scale=.1, dtype=torch.bfloat16)]
        return lambda *t: gated_feed_forward(*t, keep=kind), [t.to(DEV) for t in tensors]
    f, v, z = (normal(gen, 2, 150, 40, mean=m).to(DEV) for m in (2.0, 0.0, 0.0))
    if kind == "scan":
        return lambda f, v: gated_recurrence(f, v)[0], [f, v]
    return lambda f, v, z, s: torch.cat([t.flatten() for t in gated_recurrence(f, v, z, s)]), [f, v, z, normal(gen, 2, 40).to(DEV)]


@pytest.mark.parametrize("loss", [lambda y: y.float().sum(), lambda y: y.float().square().sum()])
@pytest.mark.parametrize("kind", ["full", "fp8", "scan", "scan_gated"])
def test_second_derivatives_raise(kind, loss):
    """A gradient penalty, in every input: an error, not the penalty's missing share; the first
    derivatives under create_graph are the ordinary ones."""
    run, tensors = _differentiable(kind)
    for i in range(len(tensors)):
        leaves = [t.detach().requires_grad_(i == k) for k, t in enumerate(tensors)]
        plain, = torch.autograd.grad(loss(run(*leaves)), leaves[i])
        assert not plain.requires_grad
        grad, = torch.autograd.grad(loss(run(*leaves)), leaves[i], create_graph=True)
        assert torch.equal(grad.detach(), plain) and grad.requires_grad
        with pytest.raises(RuntimeError, match="differentiated once"):
            (grad.float().square().sum() + leaves[i].float().square().sum()).backward()
    leaves = [t.detach().requires_grad_() for t in tensors]
    loss(run(*leaves)).backward(create_graph=True)
    grads = [t.grad.detach() for t in leaves]
    for t in leaves:
        t.grad = None
    loss(run(*leaves)).backward()
    assert all(torch.equal(a, t.grad) for a, t in zip(grads, leaves))


@pytest.mark.parametrize("kind", ["full", "fp8", "scan", "scan_gated"])
def test_forward_mode_raises(kind):
    """Tangents (dual tensors, torch.func.jvp), in every input and with gradients on or off: an error, not a
    result without its tangent; tensors without one are computed as ever."""
    run, tensors = _differentiable(kind)
    plain = run(*tensors)
    for i in range(len(tensors)):
        for leaf in (False, True):
            with forward_ad.dual_level():
                duals = [t.detach().requires_grad_(leaf) for t in tensors]
                assert torch.equal(run(*duals), plain)
                duals[i] = forward_ad.make_dual(duals[i], torch.ones_like(duals[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    run(*duals)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    run(*duals)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(lambda t: run(*tensors[:i], t, *tensors[i + 1:]), (tensors[i],), (torch.ones_like(tensors[i]),))


# ---- refusals ---------------------------------------------------------------------
def test_scan_refuses_on_another_stream():
    """The documented errors with stream= too, whichever argument is wrong."""
    f, side = torch.zeros(2, 5, 64, device=DEV), torch.cuda.Stream()
    for args, error in (((f, "v"), TypeError), ((f, f.cpu()), ValueError), ((f, f, [1]), TypeError),
                        ((f, f, f.cpu()), ValueError), ((f, f, None, 1.0), TypeError),
                        ((f, f, None, f[:, 0].cpu()), ValueError), (([1], f), TypeError), ((f[0], f), ValueError)):
        for call in (gated_scan, gated_scan_forward):
            with pytest.raises(error):
                call(*args, stream=side)
    _, _, saved = gated_scan_forward(f, f)
    for args, error in (((f, saved, "dlast"), TypeError), ((f.cpu(), saved), ValueError), ((f, saved, f[:, 0].cpu()), ValueError)):
        with pytest.raises(error):
            gated_scan_backward(*args, stream=side)


def test_calls_under_autograd_refuse():
    """What is no tensor, and a keep that there is none, raise as in the calls without autograd."""
    x = torch.zeros(4, 64, dtype=torch.float16, device=DEV)
    gate, up, down = (torch.zeros(s, dtype=torch.float16, device=DEV) for s in ((96, 64), (96, 64), (64, 96)))
    for args in ((None, gate, up, down), (x, None, up, down), (x, gate, 3, down), (x, gate, up, [down])):
        with pytest.raises(TypeError):
            gated_feed_forward(*args)
        with pytest.raises(TypeError):
            gated_feed_forward(x.requires_grad_() if args[0] is not None else None, *args[1:])
    for leaf in (x, x.detach()):
        with pytest.raises(ValueError, match="keep"):
            gated_feed_forward(leaf, gate, up, down, keep="none")
    with torch.no_grad(), pytest.raises(ValueError, match="keep"):
        gated_feed_forward(x, gate, up, down, keep="bf16")
    f = torch.zeros(2, 5, 64, device=DEV)
    for args in ((f, "v"), (None, f), (f, f, 1), (f, f, None, [0])):
        with pytest.raises(TypeError):
            gated_recurrence(*args)


@pytest.mark.parametrize("kind", ["full", "fp8", "scan", "scan_gated"])
def test_backward_releases_what_was_kept(kind):
    """Behind a backward only inputs, outputs and gradients are held, as torch's own operators do, also
    while an output is kept; and what is kept passes through saved_tensors_hooks (offloading)."""
    run, tensors = _differentiable(kind)
    leaves = [torch.cat([t.detach()] * 200).requires_grad_() if i == 0 or kind.startswith("scan") else
              t.detach().requires_grad_() for i, t in enumerate(tensors)]
    before = torch.cuda.memory_allocated()
    out = run(*leaves)
    size = out.untyped_storage().nbytes()
    held = torch.cuda.memory_allocated() - before - size
    assert held > (1 << 16)
    grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
    del grads
    assert torch.cuda.memory_allocated() - before - size < held // 8
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, leaves, torch.ones_like(out))

    plain = torch.autograd.grad(run(*leaves), leaves, torch.ones_like(out))
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        out = run(*leaves)
    assert torch.cuda.memory_allocated() - before - size < held // 8
    for a, b in zip(torch.autograd.grad(out, leaves, torch.ones_like(out)), plain):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["full", "fp8", "scan", "scan_gated"])
def test_inputs_changed_before_the_backward_raise(kind):
    """Every input that the backward reads; of the block's x the 8-bit form has a copy."""
    run, tensors = _differentiable(kind)
    for i in range(len(tensors)):
        if kind.startswith("scan") and i == 3:
            continue  # the first state is read by the forward alone
        leaves = [t.clone().requires_grad_(k != i) for k, t in enumerate(tensors)]
        out = run(*leaves)
        leaves[i].add_(1)
        if kind == "fp8" and i == 0:
            out.float().sum().backward()
        else:
            with pytest.raises(RuntimeError, match="inplace operation"):
                out.float().sum().backward()
