"""Layer norm, causal convolution and selective scan on the GPU against float64."""
import math

import pytest
import torch

import state_space_reference as R
from morph_amd.norm import layer_norm, layer_norm_backward, layer_norm_forward, layer_normalization
from morph_amd.selective import (causal_conv, causal_conv_backward, causal_conv_forward, causal_convolution,
                                 selective_scan, selective_scan_backward, selective_scan_forward,
                                 selective_state_space)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def normal(gen, *shape, scale=1.0, mean=0.0, dtype=F32):
    return (torch.randn(*shape, generator=gen) * scale + mean).to(dtype)


def double(*tensors):
    return [t.double() if t is not None else None for t in tensors]


def on_gpu(*tensors):
    return [t.to(DEV) if t is not None else None for t in tensors]


def same(a, b):
    return all((x is None and y is None) or torch.equal(x, y) for x, y in zip(a, b))


# ---- layer norm ------------------------------------------------------------------
NORM_SIZES = [(1, 1), (3, 2), (5, 7), (4, 8), (2, 63), (9, 64), (3, 65), (7, 511), (2, 512), (5, 513), (333, 1021),
              (6, 1024), (5, 1025), (3, 2048), (4, 2049), (3, 4096), (2, 4100), (3, 8192), (2, 8193), (2, 16384),
              (3, 16390), (2, 40000), (2100, 72), (1500, 300)]


def check_norm(x, w, b, dy, eps):
    got = layer_norm_forward(x, w, b, eps)
    y, saved = got
    back = layer_norm_backward(dy, saved)
    assert torch.equal(y, layer_norm(x, w, b, eps))
    cpu = [t.cpu() if t is not None else None for t in (x, w, b, dy)]
    x64, w64, b64, dy64 = double(*cpu)
    x64, dy64 = (t.reshape(-1, t.shape[-1]) for t in (x64, dy64))
    wdtype = next((t.dtype for t in (w, b) if t is not None), F32)
    _, r, xh, ref = R.norm(x64, w64, b64, eps)
    refs = R.norm_backward(dy64, xh, r, w64)
    bounds = R.norm_bounds(x64, w64, b64, dy64, eps, x.dtype, wdtype)
    R.assert_within(y.reshape(ref.shape), ref, bounds[0], "y")
    R.assert_within(back[0].reshape(ref.shape), refs[0], bounds[1], "dx")
    for name, g, ref, bound, given in (("dweight", back[1], refs[1], bounds[2], w), ("dbias", back[2], refs[2], bounds[3], b)):
        assert (g is None) == (given is None)
        if g is not None:
            assert g.dtype == given.dtype
            R.assert_within(g, ref, bound, name)
    return y, back


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,cols", NORM_SIZES)
def test_norm(rows, cols, dtype):
    gen = torch.Generator().manual_seed(rows * 7 + cols)
    x, dy = normal(gen, rows, cols, mean=.3, dtype=dtype), normal(gen, rows, cols, dtype=dtype)
    wdtype = dtype if (rows + cols) % 2 else F32
    w, b = normal(gen, cols, scale=.3, mean=1, dtype=wdtype), normal(gen, cols, dtype=wdtype)
    check_norm(*on_gpu(x, w, b, dy), 1e-5)


@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_norm_without_weights(has_w, has_b):
    gen = torch.Generator().manual_seed(5)
    for rows, cols in ((5, 200), (3, 3000), (2, 17000)):
        w, b = normal(gen, cols) if has_w else None, normal(gen, cols) if has_b else None
        check_norm(*on_gpu(normal(gen, rows, cols, dtype=BF16), w, b, normal(gen, rows, cols, dtype=BF16)), 1e-3)


def test_norm_of_any_layout():
    """Rows of a wider tensor at an odd place, transposed ones, three dimensions, no rows, no columns, one constant row."""
    gen = torch.Generator().manual_seed(6)
    wide = normal(gen, 40, 700, dtype=F16).to(DEV)
    w, b = normal(gen, 333).to(DEV), normal(gen, 333).to(DEV)
    whole = check_norm(wide[:, 5:338].contiguous(), w, b, wide[:, 301:634].contiguous(), 1e-5)
    part = check_norm(wide[:, 5:338], w, b, wide[:, 301:634], 1e-5)
    assert torch.equal(whole[0], part[0]) and same(whole[1], part[1])
    check_norm(normal(gen, 333, 40, dtype=F16).to(DEV).t(), w, b, normal(gen, 333, 40, dtype=F16).to(DEV).t(), 1e-5)
    check_norm(normal(gen, 4, 5, 333, dtype=F16).to(DEV), w, b, normal(gen, 4, 5, 333, dtype=F16).to(DEV), 1e-5)
    for shape in ((0, 333), (2, 0, 333)):
        y, saved = layer_norm_forward(torch.empty(shape, device=DEV), w, b)
        dx, dw, db = layer_norm_backward(torch.empty(shape, device=DEV), saved)
        assert y.shape == dx.shape == torch.Size(shape) and not dw.any() and not db.any()
    y, saved = layer_norm_forward(torch.empty(4, 0, device=DEV))
    assert y.shape == (4, 0) and layer_norm_backward(y, saved)[0].shape == (4, 0)
    flat = layer_norm(torch.full((2, 333), 3.0, device=DEV), w, b)
    assert torch.equal(flat, b.expand(2, -1))


def test_norm_of_what_is_not_finite_stays_in_its_row():
    gen = torch.Generator().manual_seed(7)
    x, w, b = on_gpu(normal(gen, 5, 700, dtype=BF16), normal(gen, 700), normal(gen, 700))
    clean = layer_norm(x, w, b)
    x[1, 3], x[3, 699] = math.inf, math.nan
    got = layer_norm(x, w, b)
    assert got[[1, 3]].isnan().any(1).all() and torch.equal(got[[0, 2, 4]], clean[[0, 2, 4]])


def test_norm_of_long_and_many_rows():
    """A row stride and rows whose offsets pass 2^31 elements, and more rows than workgroups."""
    big = torch.empty(3, 1 << 30, dtype=F16, device=DEV)
    rows = big[:, -1000:]
    rows.copy_(torch.randn(3, 1000, device=DEV))
    assert torch.equal(layer_norm(rows), layer_norm(rows.contiguous()))
    del big
    x = torch.randn(1 << 21, 64, device=DEV)
    y = layer_norm(x)
    for part in (slice(0, 64), slice(-64, None)):
        assert torch.equal(y[part], layer_norm(x[part].contiguous()))


# ---- causal convolution ------------------------------------------------------------
def check_conv(x, w, b, state, dy, dlast):
    u, last, saved = causal_conv_forward(x, w, b, state)
    back = causal_conv_backward(dy, saved, dlast)
    x64, w64, b64, s64, dy64, dl64 = double(*(t.cpu() if t is not None else None for t in (x, w, b, state, dy, dlast)))
    _, y, after = R.conv(x64, w64, b64, s64)
    refs = R.conv_backward(dy64, x64, w64, b64, s64, dl64)
    bounds = R.conv_bounds(x64, w64, b64, s64, dy64, dl64, x.dtype, w.dtype)
    R.assert_within(u, y, bounds[0], "u")
    assert torch.equal(last.cpu().double(), after)
    for name, g, ref, bound in zip(("dx", "dweight", "dbias", "dstate"), back, refs, bounds[1:]):
        if name == "dbias" and b is None:
            assert g is None
        else:
            R.assert_within(g, ref, bound, name)
    return (u, last), back


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,steps,dim,taps", [
    (1, 1, 1, 2), (2, 1, 70, 4), (3, 2, 8, 4), (2, 3, 512, 3), (1, 15, 513, 4), (2, 16, 37, 2), (2, 31, 64, 4),
    (1, 33, 100, 4), (3, 64, 40, 3), (2, 65, 300, 4), (1, 129, 260, 4), (1, 700, 12, 4), (600, 3, 20, 4), (2, 1030, 130, 4)])
def test_conv(batch, steps, dim, taps, dtype):
    gen = torch.Generator().manual_seed(batch + steps * 3 + dim)
    wdtype = dtype if dim % 2 else F32
    check_conv(*on_gpu(normal(gen, batch, steps, dim, dtype=dtype), normal(gen, dim, taps, scale=.5, dtype=wdtype),
                       normal(gen, dim, dtype=wdtype), normal(gen, batch, taps - 1, dim, dtype=dtype),
                       normal(gen, batch, steps, dim, dtype=dtype), normal(gen, batch, taps - 1, dim, dtype=dtype)))


def test_conv_without_what_is_optional_and_of_any_layout():
    gen = torch.Generator().manual_seed(8)
    both = normal(gen, 2, 90, 203, dtype=BF16).to(DEV)
    w, dy = normal(gen, 100, 4).to(DEV), normal(gen, 2, 90, 203, dtype=BF16).to(DEV)
    check_conv(both[..., :100], w, None, None, dy[..., 3:103], None)
    part = check_conv(both[..., 103:], w, None, None, dy[..., :100], None)
    whole = check_conv(both[..., 103:].contiguous(), w, None, None, dy[..., :100].contiguous(), None)
    assert same(part[0] + part[1], whole[0] + whole[1])
    turned = normal(gen, 90, 100, 2, dtype=BF16).to(DEV).permute(2, 0, 1)
    check_conv(turned, w.t().contiguous().t(), None, None, dy[..., :100], None)


def test_conv_of_no_steps_and_no_sequences():
    w = torch.randn(6, 4, device=DEV)
    s, ds = torch.randn(2, 3, 6, device=DEV), torch.randn(2, 3, 6, device=DEV)
    u, last, saved = causal_conv_forward(torch.empty(2, 0, 6, device=DEV), w, None, s)
    dx, dw, _, dstate = causal_conv_backward(u, saved, ds)
    assert u.shape == (2, 0, 6) and torch.equal(last, s) and torch.equal(dstate, ds) and not dw.any()
    u, last, saved = causal_conv_forward(torch.empty(0, 5, 6, device=DEV), w)
    dx, dw, _, dstate = causal_conv_backward(u, saved)
    assert u.shape == dx.shape == (0, 5, 6) and not dw.any() and dstate.shape == (0, 3, 6)


@pytest.mark.parametrize("cuts", [(1, 2, 3, 4, 5, 6, 7), (40,), (16, 64), (63,)])
def test_conv_in_pieces_is_the_whole(cuts):
    gen = torch.Generator().manual_seed(9)
    x, w, b = on_gpu(normal(gen, 2, 80, 50, dtype=F16), normal(gen, 50, 4), normal(gen, 50))
    whole, last = causal_conv(x, w, b)
    state, out = None, []
    for a, z in zip((0, *cuts), (*cuts, 80)):
        u, state = causal_conv(x[:, a:z], w, b, state)
        out.append(u)
    assert torch.equal(torch.cat(out, 1), whole) and torch.equal(state, last)


# ---- selective scan --------------------------------------------------------------------
def scan_inputs(gen, batch, steps, dim, n, dtype, gate=True, skip=True, bias=True, first=True):
    return on_gpu(normal(gen, batch, steps, dim, dtype=dtype), normal(gen, batch, steps, dim, scale=.7, dtype=dtype),
                  -torch.exp(normal(gen, dim, n, scale=.7)), normal(gen, batch, steps, n, dtype=dtype),
                  normal(gen, batch, steps, n, dtype=dtype), normal(gen, dim) if skip else None,
                  normal(gen, batch, steps, dim, dtype=dtype) if gate else None,
                  normal(gen, dim, scale=.8, mean=-4) if bias else None,
                  normal(gen, batch, dim, n) if first else None)


NAMES = ("dx", "ddt", "dA", "dB", "dC", "dskip", "dz", "ddt_bias", "dstate")


def check_scan(inputs, dy, dlast):
    y, last, saved = selective_scan_forward(*inputs)
    back = selective_scan_backward(dy, saved, dlast)
    assert same(selective_scan(*inputs), (y, last))
    cpu = double(*(t.cpu() if t is not None else None for t in inputs))
    dy64, dl64 = double(*(t.cpu() if t is not None else None for t in (dy, dlast)))
    *_, states, _, ref = R.scan(*cpu)
    dtype = y.dtype
    R.assert_scan(y, ref, dtype, "y")
    R.assert_scan(last, states[-1], F32, "last")
    for name, g, r in zip(NAMES, back, R.scan_backward(dy64, dl64, *cpu)):
        if r is None:
            assert g is None, name
        else:
            R.assert_scan(g, r, g.dtype, name)
    return (y, last), back


SCAN_SIZES = [(1, 1, 1, 1), (2, 1, 20, 16), (3, 2, 16, 16), (2, 7, 33, 16), (1, 8, 17, 3), (2, 9, 70, 4), (2, 63, 40, 8),
              (2, 64, 16, 16), (1, 65, 48, 16), (3, 130, 21, 12), (1, 300, 30, 17), (2, 129, 9, 32), (1, 100, 7, 33),
              (2, 70, 10, 64), (1, 333, 64, 16), (2, 200, 65, 1), (40, 66, 18, 16)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,steps,dim,n", SCAN_SIZES)
def test_scan(batch, steps, dim, n, dtype):
    gen = torch.Generator().manual_seed(batch + 3 * steps + 5 * dim + n)
    inputs = scan_inputs(gen, batch, steps, dim, n, dtype)
    check_scan(inputs, *on_gpu(normal(gen, batch, steps, dim, dtype=dtype), normal(gen, batch, dim, n)))


@pytest.mark.parametrize("missing", ["gate", "skip", "bias", "first", "all"])
@pytest.mark.parametrize("steps", [1, 150])
def test_scan_without_what_is_optional(missing, steps):
    gen = torch.Generator().manual_seed(11)
    given = {name: missing not in (name, "all") for name in ("gate", "skip", "bias", "first")}
    inputs = scan_inputs(gen, 2, steps, 37, 16, BF16, **given)
    check_scan(inputs, normal(gen, 2, steps, 37, dtype=BF16).to(DEV), None)


def test_scan_of_views():
    """Slices of wider projections, at odd places, and transposed inputs: the same bits as their copies."""
    gen = torch.Generator().manual_seed(12)
    b, t, d, n = 2, 90, 35, 16
    x, dt, A, B, C, skip, z, bias, first = scan_inputs(gen, b, t, d, n, F16)
    dy = normal(gen, b, t, d, dtype=F16).to(DEV)
    wide = torch.cat([x, z, dt], 2)
    small = torch.cat([B[..., :1], B, C], 2)
    turned = C.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    late = dy.transpose(0, 1).contiguous().transpose(0, 1)
    views = [wide[..., :d], wide[..., 2 * d:], A.t().contiguous().t(), small[..., 1:n + 1], turned, skip,
             wide[..., d:2 * d], bias, first.transpose(1, 2).contiguous().transpose(1, 2)]
    y, last, saved = selective_scan_forward(x, dt, A, B, C, skip, z, bias, first)
    y2, last2, saved2 = selective_scan_forward(*views)
    assert same((y, last), (y2, last2))
    assert same(selective_scan_backward(dy, saved), selective_scan_backward(late, saved2))
    check_scan(views, late, None)


def test_scan_passes_padding_on():
    """dt = -inf: the state goes on unchanged, and the step's gradients are those of the skip and the gate alone."""
    gen = torch.Generator().manual_seed(13)
    x, dt, A, B, C, skip, z, bias, first = scan_inputs(gen, 2, 150, 20, 16, BF16)
    dt[0, 100:] = -math.inf
    dt[1, 30:70] = -math.inf
    dlast = normal(gen, 2, 20, 16).to(DEV)
    (y, last), back = check_scan([x, dt, A, B, C, skip, z, bias, first], normal(gen, 2, 150, 20, dtype=BF16).to(DEV), dlast)
    short = selective_scan(x[:1, :100], dt[:1, :100], A, B[:1, :100], C[:1, :100], skip, z[:1, :100], bias, first[:1])
    # the two are joined at other places, as in test_scan_in_pieces_is_the_whole
    R.assert_scan(last[:1], short[1].cpu(), F32, "last")
    for steps in (1, 40, 150):  # gates of 1 and inputs of 0, however they are joined
        nothing = torch.full_like(dt[:, :steps], -math.inf)
        _, same_state = selective_scan(x[:, :steps], nothing, A, B[:, :steps], C[:, :steps], skip, None, bias, first)
        assert torch.equal(same_state, first)
    assert not back[1][0, 100:].any() and not back[3][0, 100:].any()


def test_scan_forgets():
    """Steps long enough that every gate is 0: the state is the step's own."""
    gen = torch.Generator().manual_seed(14)
    x, dt, A, B, C, skip, z, bias, first = scan_inputs(gen, 1, 70, 20, 16, F32)
    A.fill_(-50.0)
    dt.fill_(30.0)
    _, last = selective_scan(x, dt, A, B, C, state=first * 1e20)
    assert torch.equal(last, (30 * x[:, -1])[..., None] * B[:, -1, None])


def test_scan_of_no_steps_and_no_sequences():
    gen = torch.Generator().manual_seed(15)
    inputs = scan_inputs(gen, 2, 0, 20, 16, F16)
    dlast = normal(gen, 2, 20, 16).to(DEV)
    y, last, saved = selective_scan_forward(*inputs)
    back = selective_scan_backward(y, saved, dlast)
    assert y.shape == (2, 0, 20) and torch.equal(last, inputs[-1]) and torch.equal(back[-1], dlast)
    assert not back[2].any() and not back[5].any() and not back[7].any() and back[3].shape == (2, 0, 16)
    inputs = scan_inputs(gen, 0, 5, 20, 16, F16)
    y, last, saved = selective_scan_forward(*inputs)
    back = selective_scan_backward(y, saved)
    assert y.shape == (0, 5, 20) and last.shape == (0, 20, 16) and not back[2].any()


@pytest.mark.parametrize("cuts", [(1, 2, 3, 4), (64,), (50, 51), (7, 100, 128)])
def test_scan_in_pieces_is_the_whole(cuts):
    """FP32 sums are joined at other places: a few units of 2^-24 of the results' size a step remembered."""
    gen = torch.Generator().manual_seed(16)
    x, dt, A, B, C, skip, z, bias, first = scan_inputs(gen, 2, 140, 40, 16, F32)
    whole, last = selective_scan(x, dt, A, B, C, skip, z, bias, first)
    state, out = first, []
    for a, e in zip((0, *cuts), (*cuts, 140)):
        y, state = selective_scan(x[:, a:e], dt[:, a:e], A, B[:, a:e], C[:, a:e], skip, z[:, a:e], bias, state)
        out.append(y)
    R.assert_scan(torch.cat(out, 1), whole.cpu(), F32, "y")
    R.assert_scan(state, last.cpu(), F32, "state")


# ---- calls -----------------------------------------------------------------------------
def operators(gen):
    """(forward and backward as one function of nothing, its inputs) of each operator."""
    x, w, b, dy = on_gpu(normal(gen, 300, 520, dtype=BF16), normal(gen, 520), normal(gen, 520), normal(gen, 300, 520, dtype=BF16))

    def norm(stream=None):
        y, saved = layer_norm_forward(x, w, b, stream=stream)
        return (y, *layer_norm_backward(dy, saved, stream=stream))
    cx, cw, cb, cs, cy = on_gpu(normal(gen, 2, 140, 90, dtype=F16), normal(gen, 90, 4), normal(gen, 90),
                                normal(gen, 2, 3, 90, dtype=F16), normal(gen, 2, 140, 90, dtype=F16))

    def conv(stream=None):
        u, last, saved = causal_conv_forward(cx, cw, cb, cs, stream=stream)
        return (u, last, *causal_conv_backward(cy, saved, cs, stream=stream))
    inputs = scan_inputs(gen, 2, 140, 90, 16, F16)
    sy = normal(gen, 2, 140, 90, dtype=F16).to(DEV)

    def scan(stream=None):
        y, last, saved = selective_scan_forward(*inputs, stream=stream)
        return (y, last, *selective_scan_backward(sy, saved, inputs[-1], stream=stream))
    one = [t[:, :1] if t.dim() == 3 and t.shape[1] == 140 else t for t in inputs]

    def token(stream=None):
        return (*causal_conv(cx[:, :1], cw, cb, cs, stream=stream), *selective_scan(*one, stream=stream))
    return dict(norm=(norm, [x, dy]), conv=(conv, [cx, cs, cy]), scan=(scan, [*inputs[:2], *inputs[3:5], sy]),
                token=(token, [cx, cs, *inputs[:2]]))


@pytest.mark.parametrize("kind", ["norm", "conv", "scan", "token"])
def test_calls_repeat_their_bits_on_any_stream_and_in_a_graph(kind):
    call, inputs = operators(torch.Generator().manual_seed(17))[kind]
    first = call()
    assert same(call(), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    there = call(stream=side)
    side.synchronize()
    assert same(there, first)
    with torch.cuda.stream(side):
        call()
        graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = call()
        with torch.cuda.graph(second, stream=side):
            other = call()
    for k in range(4):
        for t in inputs:
            t.copy_(t.roll(1, 0))
        expected = call()
        torch.cuda.synchronize()
        for t in (*out, *other):
            if t is not None:
                t.zero_()
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        assert same(out, expected) and same(other, expected), k


def autograd_cases(gen):
    x, w, b = on_gpu(normal(gen, 4, 30, 66, dtype=BF16), normal(gen, 66, dtype=BF16), normal(gen, 66, dtype=BF16))
    cx, cw, cb, cs = on_gpu(normal(gen, 2, 40, 30, dtype=F16), normal(gen, 30, 4), normal(gen, 30), normal(gen, 2, 3, 30, dtype=F16))
    return dict(norm=(lambda *a: (layer_normalization(*a),), [x, w, b], lambda *a: layer_norm_forward(*a)[1],
                      layer_norm_backward),
                conv=(causal_convolution, [cx, cw, cb, cs], lambda *a: causal_conv_forward(*a)[2], causal_conv_backward),
                scan=(selective_state_space, scan_inputs(gen, 2, 70, 20, 16, BF16),
                      lambda *a: selective_scan_forward(*a)[2], selective_scan_backward))


@pytest.mark.parametrize("kind", ["norm", "conv", "scan"])
def test_autograd(kind):
    gen = torch.Generator().manual_seed(18)
    f, tensors, forward, backward = autograd_cases(gen)[kind]
    plain = f(*tensors)
    assert not any(t.requires_grad for t in plain)
    leaves = [t.clone().requires_grad_() for t in tensors]
    outs = f(*leaves)
    assert same(outs, plain)
    ends = [normal(gen, *o.shape, dtype=o.dtype).to(DEV) for o in outs]
    torch.autograd.backward(outs, ends)
    for leaf, g in zip(leaves, backward(ends[0], forward(*tensors), *ends[1:])):
        assert torch.equal(leaf.grad, g)
    # the state alone, and y alone
    if len(outs) > 1:
        again = [t.clone().requires_grad_() for t in tensors]
        f(*again)[1].sum().backward()
        assert again[0].grad is not None and again[0].grad.isfinite().all()
    # second derivatives raise; so do inputs that were changed before the backward
    leaves = [t.clone().requires_grad_() for t in tensors]
    y = f(*leaves)[0]
    grad, = torch.autograd.grad(y.float().sum(), leaves[:1], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        grad.float().sum().backward()
    leaves = [t.clone().requires_grad_() for t in tensors]
    y = f(*leaves)[0]
    with torch.no_grad():
        leaves[0].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_stage_of_them_against_float64():
    """Norm, projection, convolution, projections, scan, projection, as a model runs them, in FP32: forward and all
    gradients by autograd against the same stage in float64; then the sequence token by token."""
    gen = torch.Generator().manual_seed(19)
    b, t, d, inner, n = 2, 50, 24, 40, 8
    x = normal(gen, b, t, d)
    params = [normal(gen, d, mean=1, scale=.2), normal(gen, d, scale=.2), normal(gen, 2 * inner, d, scale=d ** -.5),
              normal(gen, inner, 4, scale=.5), normal(gen, inner, scale=.2), normal(gen, 2 * n + inner, inner, scale=inner ** -.5),
              torch.log(torch.arange(1, n + 1).float()).expand(inner, n).contiguous(), normal(gen, inner),
              normal(gen, inner, mean=-3), normal(gen, d, inner, scale=inner ** -.5)]

    def stage(x, params, norm, conv, scan, states=(None, None)):
        w, c, into, taps, cb, mix, logA, skip, bias, out = params
        u, z = (norm(x, w, c) @ into.t()).split(inner, -1)
        u, inputs = conv(u, taps, cb, states[0])
        B, C, dt = (u @ mix.t()).split([n, n, inner], -1)
        y, state = scan(u, dt, -logA.exp(), B, C, skip, z, bias, states[1])
        return x + y @ out.t(), (inputs, state)

    def plain_conv(x, w, b, state):
        _, y, after = R.conv(x, w, b, state)
        return y, after

    leaves = [p.double().requires_grad_() for p in (x, *params)]
    ref, _ = stage(leaves[0], leaves[1:], lambda x, w, c: R.norm(x, w, c, 1e-5)[3], plain_conv,
                   plain_scan)
    end = normal(gen, b, t, d)
    ref.backward(end.double())
    mine = [p.to(DEV).requires_grad_() for p in (x, *params)]
    got, _ = stage(mine[0], mine[1:], layer_normalization, causal_convolution, selective_state_space)
    got.backward(end.to(DEV))
    R.assert_scan(got.detach(), ref.detach(), F32, "output")
    for k, (a, r) in enumerate(zip(mine, leaves)):
        R.assert_scan(a.grad, r.grad, F32, f"gradient {k}")
    with torch.no_grad():
        states, out = (None, None), []
        for i in range(t):
            y, states = stage(mine[0][:, i:i + 1], mine[1:], layer_norm, causal_conv, selective_scan, states)
            out.append(y)
    R.assert_scan(torch.cat(out, 1), ref.detach(), F32, "token by token")


def plain_scan(x, dt, A, B, C, skip, z, bias, first):
    """R.scan without writes in place, for autograd."""
    d = R.softplus(dt + bias)
    h = torch.zeros(x.shape[0], *A.shape, dtype=x.dtype) if first is None else first
    s = []
    for t in range(x.shape[1]):
        h = torch.exp(d[:, t, :, None] * A) * h + (d[:, t] * x[:, t])[..., None] * B[:, t, None]
        s.append((h * C[:, t, None]).sum(2))
    s = torch.stack(s, 1) + skip * x
    return s * z * torch.sigmoid(z), h


# ---- forms that sizes alone choose -----------------------------------------------------------
@pytest.mark.parametrize("rows,cols", [(3300, 1100), (1700, 2100), (1600, 8200)])
def test_norm_of_more_rows_than_workgroups(rows, cols):
    gen = torch.Generator().manual_seed(20)
    check_norm(*on_gpu(normal(gen, rows, cols, dtype=BF16), normal(gen, cols, mean=1), normal(gen, cols),
                       normal(gen, rows, cols, dtype=BF16)), 1e-5)


@pytest.mark.parametrize("batch,steps,dim,n", [
    (1, 700, 16, 16), (2, 600, 7, 5),     # more segments than are joined where they are needed
    (400, 140, 16, 16),                   # segments of several tiles
    (300, 1600, 5, 4), (100, 6000, 3, 17),  # of many, and not a multiple of the waves
    (520, 70, 10, 8),                     # sequences enough to stay whole
    (800, 3, 32, 16), (300, 34, 40, 16),  # two channel groups a workgroup backward; two and one
    (130, 40, 100, 64)])
def test_scan_forms(batch, steps, dim, n):
    gen = torch.Generator().manual_seed(21)
    inputs = scan_inputs(gen, batch, steps, dim, n, F32)
    check_scan(inputs, *on_gpu(normal(gen, batch, steps, dim), normal(gen, batch, dim, n)))


@pytest.mark.parametrize("batch,steps", [(1, 1), (1, 3), (2, 1), (2, 3)])
def test_scan_of_steps_that_lie_far_apart(batch, steps):
    """Steps farther apart than the kernels count: copies of them, and of one step its stride does not matter."""
    gen = torch.Generator().manual_seed(22)
    inputs = scan_inputs(gen, batch, steps, 21, 16, BF16)
    dy = normal(gen, batch, steps, 21, dtype=BF16).to(DEV)
    y, last, saved = selective_scan_forward(*inputs)
    far = torch.empty(batch, steps, (1 << 25) + 8, dtype=BF16, device=DEV)
    views = [inputs[0], inputs[1], inputs[3], inputs[4], inputs[6], dy]
    places, at = [], 0
    for t in views:
        far[..., at:at + t.shape[2]] = t
        places.append(far[..., at:at + t.shape[2]])
        at += t.shape[2]
    x2, dt2, B2, C2, z2, dy2 = places
    for stream in (None, torch.cuda.current_stream()):
        y2, last2, saved2 = selective_scan_forward(x2, dt2, inputs[2], B2, C2, inputs[5], z2, *inputs[7:], stream=stream)
        assert same((y, last), (y2, last2))
        assert same(selective_scan_backward(dy, saved), selective_scan_backward(dy2, saved2, stream=stream))


def test_scan_of_inputs_that_are_shared():
    """One state, one B and C for all sequences, one step length for all steps: expanded views, and their gradients."""
    gen = torch.Generator().manual_seed(23)
    x, dt, A, B, C, skip, z, bias, first = scan_inputs(gen, 3, 50, 20, 16, F32)
    shared = [x, dt[:, :1], A, B[:1], C[:1], skip, z, bias, first[:1]]
    sizes = [None, (3, 50, 20), None, (3, 50, 16), (3, 50, 16), None, None, None, (3, 20, 16)]
    end = normal(gen, 3, 50, 20)

    def run(leaves, f, end):
        wide = [t if size is None else t.expand(size) for t, size in zip(leaves, sizes)]
        return torch.autograd.grad(f(*wide)[0], leaves, end)
    refs = run([t.cpu().double().requires_grad_() for t in shared], plain_scan, end.double())
    for k, (g, r) in enumerate(zip(run([t.clone().requires_grad_() for t in shared], selective_state_space, end.to(DEV)), refs)):
        R.assert_scan(g, r, F32, f"gradient {k}")


@pytest.mark.parametrize("kind", ["norm", "conv", "scan"])
def test_autograd_in_a_graph(kind):
    """Forward and backward of leaves of the capture's own, replayed between eager work."""
    gen = torch.Generator().manual_seed(24)
    f, tensors, _, _ = autograd_cases(gen)[kind]
    ends = [normal(gen, *o.shape, dtype=o.dtype).to(DEV) for o in f(*tensors)]

    def run():
        leaves = [t.detach().requires_grad_() for t in tensors]
        outs = f(*leaves)
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, ends))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = run()
    side.synchronize()
    for k in range(3):
        for t in tensors[:2]:
            t.copy_(t.roll(1, 0))
        expected = run()
        torch.cuda.synchronize()
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, expected), k


@pytest.mark.parametrize("kind", ["norm", "conv", "scan"])
def test_two_streams_at_once(kind):
    call, _ = operators(torch.Generator().manual_seed(25))[kind]
    first = call()
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(call())
    torch.cuda.synchronize()
    assert all(same(r, first) for r in results)
