"""The layer operators against float64 (tests/layer_reference.py), at the sizes, strides and
values where they can go wrong, and what they refuse."""
import math

import pytest
import torch

import layer_reference as R
from morph_amd.activations import PackedActivation, pack_activation, unpack_activation
from morph_amd.ffn import GatedFFN, gated_ffn, gated_ffn_backward, gated_ffn_forward
from morph_amd.recurrence import gated_recurrence, gated_scan, gated_scan_backward, gated_scan_forward

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HALF = [torch.float16, torch.bfloat16]
FLOATS = [torch.float32, *HALF]


def normal(gen, *shape, scale=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen) * scale + mean).to(dtype)


# ---- activations -------------------------------------------------------------
def _packed_equals(x, dev_x=None):
    packed = pack_activation(x.to(DEV) if dev_x is None else dev_x)
    codes, exps = R.pack(x.reshape(-1, x.shape[-1]))
    assert torch.equal(packed.exponents.cpu(), torch.from_numpy(exps))
    assert torch.equal(packed.codes.cpu(), torch.from_numpy(codes))
    for dtype in FLOATS:
        out = unpack_activation(packed, dtype)
        assert out.shape == x.shape and out.dtype == dtype
        ref = R.unpack(packed.codes, packed.exponents, x.shape[-1]).reshape(x.shape).to(dtype)
        assert torch.equal(out.cpu().nan_to_num(7.0, 1e30, -1e30), ref.nan_to_num(7.0, 1e30, -1e30))
        assert torch.equal(out.cpu().isnan(), ref.isnan())
    return packed


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 3, 200), (257, 96), (64, 1024), (7, 8)])
def test_pack_equals_the_definition(dtype, shape):
    gen = torch.Generator().manual_seed(sum(shape))
    x = normal(gen, *shape) * torch.exp(2 * normal(gen, shape[-1]))
    _packed_equals(x.to(dtype))


@pytest.mark.parametrize("dtype", FLOATS)
def test_pack_at_the_ends_of_the_range(dtype):
    """Zeros and their signs, subnormals, the type's largest values, ties, powers of two and
    1.75 of them (where the exponent steps), and groups that hold what is not finite."""
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = [torch.zeros(40), torch.full((40,), -0.0), torch.full((40,), top), torch.full((40,), tiny),
            torch.full((40,), tiny * 2.0 ** -4 if dtype != torch.float32 else 2.0 ** -149)]
    for k in range(-14, 15):
        for m in (1.0, 1.75, 1.7578125, 1.9921875):
            rows.append(m * 2.0 ** k * torch.tensor([1.0, -0.53125, 0.0625, 0.03125] * 10))
    rows.append(torch.arange(40) / 16 + 1)  # ties between codes
    for bad in (math.nan, math.inf, -math.inf):
        row = torch.linspace(-3, 3, 40)
        row[5] = row[37] = bad
        rows.append(row)
        rows.append(torch.full((40,), bad))
    _packed_equals(torch.stack(rows).to(dtype))


@pytest.mark.parametrize("dtype", FLOATS)
def test_pack_of_views(dtype):
    """Rows of a wider tensor, an offset that no 16-byte access fits, transposed and expanded
    views: the same codes as of a copy."""
    gen = torch.Generator().manual_seed(3)
    base = normal(gen, 20, 130, dtype=dtype)
    dev = base.to(DEV)
    for view in (lambda t: t[:, :96], lambda t: t[:, 1:98], lambda t: t[::2, 3:], lambda t: t.t(),
                 lambda t: t[:1].expand(6, 130), lambda t: t.view(4, 5, 130)[:, 1:4]):
        _packed_equals(view(base).contiguous(), view(dev))


def test_pack_moves_to_the_host_and_back():
    x = normal(torch.Generator().manual_seed(1), 33, 70, dtype=torch.bfloat16).to(DEV)
    packed = pack_activation(x)
    back = packed.to("cpu").to(DEV)
    assert packed.nbytes == 33 * (96 + 3)
    assert torch.equal(unpack_activation(back), unpack_activation(packed))


def test_pack_of_nothing():
    for shape in ((0, 64), (4, 0), (0,)):
        packed = pack_activation(torch.empty(shape, dtype=torch.float16, device=DEV))
        assert unpack_activation(packed).shape == shape


def test_pack_refuses():
    x = torch.zeros(4, 64, device=DEV)
    with pytest.raises(ValueError):
        pack_activation(x.cpu())
    with pytest.raises(TypeError):
        pack_activation(x.double())
    with pytest.raises(ValueError):
        pack_activation(x[0, 0])
    p = pack_activation(x)
    with pytest.raises(TypeError):
        unpack_activation(p, torch.int32)
    with pytest.raises(TypeError):
        unpack_activation(x)
    with pytest.raises(ValueError):
        unpack_activation(PackedActivation(p.codes, p.exponents, (5, 64), torch.float32))
    with pytest.raises(ValueError):
        unpack_activation(p.to("cpu"))


# ---- the feed-forward block --------------------------------------------------
SHAPES = [  # rows, d, ff: one row to several tiles, whole and ragged, widths that fit nothing
    (1, 8, 8), (1, 64, 128), (1, 200, 535), (2, 33, 7), (5, 96, 200), (16, 128, 256), (17, 256, 96),
    (33, 264, 520), (64, 64, 64), (65, 72, 136), (100, 129, 257), (129, 320, 192), (130, 512, 384),
    (257, 200, 712), (300, 384, 1000), (513, 136, 264)]


def _weights(gen, d, ff, dtype):
    return (normal(gen, ff, d, scale=d ** -.5, dtype=dtype), normal(gen, ff, d, scale=d ** -.5, dtype=dtype),
            normal(gen, d, ff, scale=ff ** -.5, dtype=dtype))


def _check_forward(y, x, weights, dtype, what):
    x, gate, up, down = (t.double().cpu() for t in (x, *weights))
    h = R.ffn(x, gate, up, down)[2]
    R.assert_product(y.reshape(-1, y.shape[-1]), h, down.T, dtype, what)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,d,ff", SHAPES)
def test_ffn_forward(dtype, rows, d, ff):
    gen = torch.Generator().manual_seed(rows + d + ff)
    x, weights = normal(gen, rows, d, dtype=dtype), _weights(gen, d, ff, dtype)
    y = gated_ffn(x.to(DEV), *(w.to(DEV) for w in weights))
    _check_forward(y, x, weights, dtype, "y")


def _check_backward(grads, dy, x, g, u, weights, dtype):
    gate, up, down = (w.double().cpu() for w in weights)
    dy, x = dy.double().cpu(), x.double().cpu()
    ref = R.ffn_backward(dy, x, g, u, gate, up, down)
    dx, dgate, dup, ddown = grads
    both = torch.cat([ref["dg"], ref["du"]], 1)
    R.assert_product(dx.reshape(-1, dx.shape[-1]), both, torch.cat([gate, up]), dtype, "dx")
    R.assert_product(dgate, ref["dg"].T, x, dtype, "dgate")
    R.assert_product(dup, ref["du"].T, x, dtype, "dup")
    R.assert_product(ddown, dy.T, ref["h"], dtype, "ddown")


def _kept(saved, rows, ff):
    """(x, g, u) that the backward stands on, in float64."""
    if saved.keep == "full":
        for t in (saved.gate, saved.up):
            assert (t[:, ff:] == 0).all()
        return saved.x.double().cpu(), saved.gate[:, :ff].double().cpu(), saved.up[:, :ff].double().cpu()
    return tuple(R.unpack(p.codes, p.exponents, p.shape[-1]) for p in (saved.x, saved.gate, saved.up))


@pytest.mark.parametrize("keep", ["full", "fp8"])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,d,ff", SHAPES)
def test_ffn_training_step(dtype, rows, d, ff, keep):
    """Forward, what is kept, and the four gradients (those by the formula on what was kept)."""
    gen = torch.Generator().manual_seed(rows + d + ff)
    x, weights = normal(gen, rows, d, dtype=dtype), _weights(gen, d, ff, dtype)
    dy = normal(gen, rows, d, dtype=dtype)
    dev = [w.to(DEV) for w in weights]
    y, saved = gated_ffn_forward(x.to(DEV), *dev, keep=keep)
    _check_forward(y, x, weights, dtype, "y")
    xk, g, u = _kept(saved, rows, ff)
    exact = R.ffn(x.double(), *(w.double() for w in weights))
    for name, got, ref, left, right in (("g", g, exact[0], x.double(), weights[0].double().T),
                                        ("u", u, exact[1], x.double(), weights[1].double().T)):
        # FP32 sums; in 8 bits half a step more: 2^-4 of the value, or 2^-10 of a scale that is
        # at most 2^-7.8 of the group's largest
        bound = 2.0 ** -20 * (left.abs() @ right.abs())
        if keep == "fp8":
            bound += 2.0 ** -4 * ref.abs() + 2.0 ** -17 * ref.abs().amax(1, keepdim=True)
        assert ((got - ref).abs() <= bound + 1e-30).all(), name
    if keep == "fp8":
        codes, exps = R.pack(x)
        assert torch.equal(saved.x.codes.cpu(), torch.from_numpy(codes))
        assert torch.equal(saved.x.exponents.cpu(), torch.from_numpy(exps))
    grads = gated_ffn_backward(dy.to(DEV), saved, *dev)
    assert [tuple(t.shape) for t in grads] == [(rows, d), (ff, d), (ff, d), (d, ff)]
    _check_backward(grads, dy, xk, g, u, weights, dtype)


@pytest.mark.parametrize("keep", ["full", "fp8"])
@pytest.mark.parametrize("rows,d,ff", [(3, 40, 3001), (70, 72, 2056), (130, 265, 2500), (257, 65, 5001),
                                       (400, 513, 1027)])
def test_ffn_wide_middle(rows, d, ff, keep):
    """ff far above d: sums over ff for few outputs, and results at odd addresses."""
    test_ffn_forward(torch.bfloat16, rows, d, ff)
    test_ffn_training_step(torch.bfloat16, rows, d, ff, keep)


@pytest.mark.parametrize("rows,d,ff", [(100, 1536, 3000), (390, 1001, 4100)])
def test_ffn_some_hundred_rows(rows, d, ff):
    test_ffn_forward(torch.float16, rows, d, ff)
    test_ffn_training_step(torch.float16, rows, d, ff, "full")


@pytest.mark.parametrize("keep", ["full", "fp8"])
@pytest.mark.parametrize("rows,d,ff", [(3, 64, 96), (200, 128, 192)])
def test_ffn_strides(rows, d, ff, keep):
    """Operands that are views: rows of wider tensors, at odd offsets, transposed, expanded, and
    x with leading dimensions."""
    dtype = torch.bfloat16
    gen = torch.Generator().manual_seed(5)
    wide = [normal(gen, rows, d + 24, dtype=dtype), normal(gen, ff, d + 8, scale=d ** -.5, dtype=dtype),
            normal(gen, d, ff, scale=d ** -.5, dtype=dtype), normal(gen, d, ff + 3, scale=ff ** -.5, dtype=dtype)]
    dy = normal(gen, rows, 1, d + 1, dtype=dtype)
    for pick in (lambda x, g, u, w, q: (x[:, 8:8 + d], g[:, :d], u.t(), w[:, 3:], q[:, 0, 1:]),
                 lambda x, g, u, w, q: (x[:, 3:3 + d], g[:, 1:1 + d], u.t(), w[:, :ff], q[:, 0, :d])):
        host, dev = pick(*wide, dy), pick(*(t.to(DEV) for t in wide), dy.to(DEV))
        y, saved = gated_ffn_forward(dev[0], *dev[1:4], keep=keep)
        _check_forward(y, host[0], host[1:4], dtype, "y")
        grads = gated_ffn_backward(dev[4], saved, *dev[1:4])
        _check_backward(grads, host[4], *_kept(saved, rows, ff), host[1:4], dtype)
    # broadcast rows (their rounding errors are alike, not independent): the bits of the copies
    x, g, u, w, q = (t.to(DEV) for t in (*wide, dy))
    views = (x[:1, :d].expand(rows, d), g[:1, :d].expand(ff, d), u.t(), w[:, 2:2 + ff], q[:1, 0, :d].expand(rows, d))
    results = []
    for args in (views, [t.contiguous() for t in views[:3]] + [views[3], views[4].contiguous()]):
        y, saved = gated_ffn_forward(args[0], *args[1:4], keep=keep)
        results.append((y, *gated_ffn_backward(args[4], saved, *args[1:4])))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_ffn_leading_dimensions_and_one_row():
    gen = torch.Generator().manual_seed(9)
    weights = [w.to(DEV) for w in _weights(gen, 64, 160, torch.float16)]
    x = normal(gen, 2, 3, 5, 64, dtype=torch.float16).to(DEV)
    y = gated_ffn(x, *weights)
    assert y.shape == x.shape and torch.equal(y.view(-1, 64), gated_ffn(x.view(-1, 64), *weights))
    _check_forward(gated_ffn(x[0, 0, 0], *weights), x[0, 0, :1], weights, torch.float16, "one row")
    z = x.permute(1, 0, 2, 3)
    assert torch.equal(gated_ffn(z, *weights), gated_ffn(z.contiguous(), *weights))


def test_ffn_same_bits_every_time():
    gen = torch.Generator().manual_seed(2)
    for rows, d, ff in ((1, 512, 1024), (40, 264, 600), (300, 384, 1000)):
        weights = [w.to(DEV) for w in _weights(gen, d, ff, torch.bfloat16)]
        x, dy = (normal(gen, rows, d, dtype=torch.bfloat16).to(DEV) for _ in range(2))

        def step():
            y, saved = gated_ffn_forward(x, *weights, keep="fp8")
            return y, gated_ffn(x, *weights), *gated_ffn_backward(dy, saved, *weights)
        first = step()
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, step()))


def test_ffn_no_rows():
    gen = torch.Generator().manual_seed(2)
    weights = [w.to(DEV) for w in _weights(gen, 64, 96, torch.float16)]
    x = torch.empty(0, 64, dtype=torch.float16, device=DEV)
    assert gated_ffn(x, *weights).shape == (0, 64)
    for keep in ("full", "fp8"):
        y, saved = gated_ffn_forward(x, *weights, keep=keep)
        dx, *dw = gated_ffn_backward(torch.empty_like(x), saved, *weights)
        assert dx.shape == (0, 64)
        for g, w in zip(dw, weights):
            assert g.shape == w.shape and (g == 0).all()


@pytest.mark.parametrize("keep", ["full", "fp8"])
@pytest.mark.parametrize("rows", [3, 200])
def test_ffn_passes_what_is_not_finite(rows, keep):
    """A NaN or an infinity in a row of x makes that row's outputs non-finite and no other's,
    and every weight gradient that the row reaches; one in dy the same."""
    gen = torch.Generator().manual_seed(4)
    weights = [w.to(DEV) for w in _weights(gen, 136, 264, torch.float16)]
    x, dy = (normal(gen, rows, 136, dtype=torch.float16).to(DEV) for _ in range(2))
    clean, kept = gated_ffn_forward(x, *weights, keep=keep)
    clean_dx = gated_ffn_backward(dy, kept, *weights)[0]
    for bad in (math.nan, math.inf, -math.inf):
        x2 = x.clone()
        x2[1, 135] = bad
        y, saved = gated_ffn_forward(x2, *weights, keep=keep)
        others = [i for i in range(rows) if i != 1]
        assert not torch.isfinite(y[1]).any() and torch.equal(y[others], clean[others])
        assert torch.equal(gated_ffn(x2, *weights).isnan(), y.isnan())
        dx, *dw = gated_ffn_backward(dy, saved, *weights)
        assert not torch.isfinite(dx[1]).any() and torch.equal(dx[others], clean_dx[others])
        assert all(not torch.isfinite(g).all() for g in dw)
        dy2 = dy.clone()
        dy2[1, 7] = bad
        dx, *dw = gated_ffn_backward(dy2, kept, *weights)
        assert not torch.isfinite(dx[1]).any() and torch.equal(dx[others], clean_dx[others])
        assert all(not torch.isfinite(g).all() for g in dw)


def test_ffn_overflow_of_the_type_is_infinite():
    """FP16 results beyond 65504 become infinities, which the gradients' detector finds."""
    weights = [torch.full(s, 8.0, dtype=torch.float16, device=DEV) for s in ((64, 64), (64, 64), (64, 64))]
    assert torch.isinf(gated_ffn(torch.full((4, 64), 8.0, dtype=torch.float16, device=DEV), *weights)).all()


@pytest.mark.parametrize("keep", ["full", "fp8"])
def test_ffn_autograd_module(keep):
    gen = torch.Generator().manual_seed(6)
    module = GatedFFN(128, 320, keep=keep, device=DEV, dtype=torch.bfloat16)
    assert set(module.state_dict()) == {"gate.weight", "up.weight", "down.weight"}
    with torch.no_grad():
        for p, w in zip((module.gate, module.up, module.down), _weights(gen, 128, 320, torch.bfloat16)):
            p.weight.copy_(w)
    weights = module.gate.weight, module.up.weight, module.down.weight
    x = normal(gen, 4, 30, 128, dtype=torch.bfloat16).to(DEV).requires_grad_()
    dy = normal(gen, 4, 30, 128, dtype=torch.bfloat16).to(DEV)
    y = module(x)
    y.backward(dy)
    plain, saved = gated_ffn_forward(x, *weights, keep=keep)
    grads = gated_ffn_backward(dy, saved, *weights)
    assert torch.equal(y, plain)
    for a, b in zip((x.grad, *(w.grad for w in weights)), grads):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(module(x), gated_ffn(x, *weights))


def test_ffn_gradient_against_differences():
    """<gradient, direction> against the forward's central difference along it.  The loss is
    sum(y * dy) over 2^14 outputs; FP16 outputs differ by u |y| at random, so the difference's
    noise is u sqrt(2^14) / (2 * 0.05) < 1 beside derivatives of 128 times the direction's
    root mean square (about 1): 5 in all with the cubic term, at 6 deviations."""
    gen = torch.Generator().manual_seed(8)
    rows, d, ff = 128, 128, 256
    dtype = torch.float16
    tensors = [normal(gen, rows, d, dtype=dtype).to(DEV), *(w.to(DEV) for w in _weights(gen, d, ff, dtype))]
    dy = normal(gen, rows, d, dtype=dtype).to(DEV)
    y, saved = gated_ffn_forward(*tensors, keep="full")
    grads = gated_ffn_backward(dy, saved, *tensors[1:])
    for i, (t, g) in enumerate(zip(tensors, grads)):
        direction = torch.sign(g.float()) * t.float().abs().mean()
        eps = 0.05

        def loss(sign):
            moved = list(tensors)
            moved[i] = (t.float() + sign * eps * direction).to(dtype)
            return (gated_ffn(*moved).double() * dy.double()).sum().item(), moved[i].double()
        (hi, at_hi), (lo, at_lo) = loss(1), loss(-1)
        slope = (g.double() * (at_hi - at_lo)).sum().item()  # along the step that was really taken
        assert abs(hi - lo - slope) <= 0.02 * abs(slope) + 1, (i, hi - lo, slope)


def test_ffn_refuses():
    dtype = torch.float16
    x = torch.zeros(4, 64, dtype=dtype, device=DEV)
    gate, up = (torch.zeros(96, 64, dtype=dtype, device=DEV) for _ in range(2))
    down = torch.zeros(64, 96, dtype=dtype, device=DEV)
    for args, error in (((x.float(), gate, up, down), TypeError), ((x, gate.bfloat16(), up, down), TypeError),
                        ((x.cpu(), gate, up, down), ValueError), ((x, gate.cpu(), up, down), ValueError),
                        ((x[:, :63], gate, up, down), ValueError), ((x, gate, up[:95], down), ValueError),
                        ((x, gate, up, down.t()), ValueError), ((x, gate[:0], up[:0], down[:, :0]), ValueError),
                        ((x[:, :0], gate[:, :0], up[:, :0], down[:0]), ValueError), ((x, None, up, down), TypeError)):
        with pytest.raises(error):
            gated_ffn(*args)
    with pytest.raises(ValueError):
        gated_ffn_forward(x, gate, up, down, keep="bf16")
    _, saved = gated_ffn_forward(x, gate, up, down)
    for args, error in (((x[:3], saved, gate, up, down), ValueError), ((x.float(), saved, gate, up, down), TypeError),
                        ((x, saved, gate[:64], up[:64], down[:, :64]), ValueError),
                        ((x, None, gate, up, down), TypeError)):
        with pytest.raises(error):
            gated_ffn_backward(*args)


def test_operators_on_another_stream():
    """Calls with stream= run there, on inputs made there, beside work on the current one."""
    gen = torch.Generator().manual_seed(12)
    weights = [w.to(DEV) for w in _weights(gen, 128, 256, torch.bfloat16)]
    host = normal(gen, 300, 128, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    ref, kept = gated_ffn_forward(host.to(DEV), *weights, keep="fp8")
    grads = gated_ffn_backward(host.to(DEV), kept, *weights)
    packed = pack_activation(host.to(DEV))
    scanned = gated_scan(host.to(DEV)[None], host.to(DEV)[None])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x = host.to(DEV, non_blocking=True)
    for _ in range(3):
        torch.zeros(1 << 22, device=DEV)
        y, saved = gated_ffn_forward(x, *weights, keep="fp8", stream=side)
        got = gated_ffn_backward(x, saved, *weights, stream=side)
        p = pack_activation(x, stream=side)
        u = unpack_activation(p, stream=side)
        s = gated_scan(x[None], x[None], stream=side)
    side.synchronize()
    assert torch.equal(y, ref) and all(torch.equal(a, b) for a, b in zip(got, grads))
    assert torch.equal(p.codes, packed.codes) and torch.equal(u, unpack_activation(packed))
    assert torch.equal(s[0], scanned[0]) and torch.equal(s[1], scanned[1])


# ---- the recurrence ----------------------------------------------------------
SCANS = [  # batch, steps, dim: one step to many spans, widths that fill no line
    (1, 1, 1), (3, 1, 64), (2, 2, 7), (1, 5, 130), (2, 63, 64), (2, 64, 33), (1, 65, 200), (3, 100, 8),
    (1, 129, 65), (2, 300, 96), (1, 1000, 40), (1, 2311, 72), (5, 517, 3), (1, 4160, 128)]


def _scan_inputs(gen, batch, steps, dim, dtype, gate, first):
    f = normal(gen, batch, steps, dim, scale=1.5, mean=2.0, dtype=dtype)
    f[torch.rand(batch, steps, generator=gen) < .02] = -math.inf
    f[torch.rand(batch, steps, dim, generator=gen) < .01] = math.inf
    v = normal(gen, batch, steps, dim, dtype=dtype)
    z = normal(gen, batch, steps, dim, dtype=dtype) if gate else None
    s0 = normal(gen, batch, dim) if first else None
    return f, v, z, s0


def _64(*ts):
    return [t.double() if t is not None else None for t in ts]


def _dev(*ts):
    return [t.to(DEV) if t is not None else None for t in ts]


@pytest.mark.parametrize("gate,first", [(True, True), (False, False), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("batch,steps,dim", SCANS)
def test_scan(dtype, batch, steps, dim, gate, first):
    gen = torch.Generator().manual_seed(batch + steps + dim)
    args = _scan_inputs(gen, batch, steps, dim, dtype, gate, first)
    dy, dlast = normal(gen, batch, steps, dim, dtype=dtype), normal(gen, batch, dim) if first else None
    y, last, states = R.scan(*_64(*args))
    got, glast, saved = gated_scan_forward(*_dev(*args))
    R.assert_scan(got, y, dtype, "y")
    R.assert_scan(glast, last, torch.float32, "last")
    again = gated_scan(*_dev(*args))
    assert torch.equal(again[0], got) and torch.equal(again[1], glast)
    ref = R.scan_backward(*_64(*args), dy.double(), dlast.double() if first else None)
    grads = gated_scan_backward(dy.to(DEV), saved, dlast.to(DEV) if first else None)
    assert (grads[2] is None) == (not gate)
    for name, a, b in zip(("df", "dv", "dz"), grads, ref):
        if a is not None:
            R.assert_scan(a, b, dtype, name)
    R.assert_scan(grads[3], ref[3], torch.float32, "ds0")
    twice = gated_scan_backward(dy.to(DEV), saved, dlast.to(DEV) if first else None)
    assert all(a is None or torch.equal(a, b) for a, b in zip(grads, twice))


@pytest.mark.parametrize("batch,steps,dim", [(2, 16500, 40), (1, 33000, 3)])
def test_scan_of_long_memory(batch, steps, dim):
    """All gates but one in a thousand are 1: a state counts thousands of steps later, with the
    roundings of a few, across every boundary that the kernels set between steps."""
    gen = torch.Generator().manual_seed(steps)
    f, v, z, s0 = _scan_inputs(gen, batch, steps, dim, torch.float32, True, True)
    f = torch.where(torch.rand(f.shape, generator=gen) < .001, f.clamp(-4, 4), torch.tensor(math.inf))
    dy, dlast = normal(gen, batch, steps, dim), normal(gen, batch, dim)
    y, last, _ = R.scan(*_64(f, v, z, s0))
    got, glast, saved = gated_scan_forward(*_dev(f, v, z, s0))
    R.assert_scan(got, y, torch.float32, "y")
    R.assert_scan(glast, last, torch.float32, "last")
    grads = gated_scan_backward(dy.to(DEV), saved, dlast.to(DEV))
    ref = R.scan_backward(*_64(f, v, z, s0), dy.double(), dlast.double())
    for name, a, b in zip(("df", "dv", "dz", "ds0"), grads, ref):
        R.assert_scan(a, b, torch.float32, name)
    for a, b in zip(grads, gated_scan_backward(dy.to(DEV), saved, dlast.to(DEV))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_by_single_steps_equals_the_whole(dtype):
    """Token by token with the state handed on: FP32 states, so the same to their rounding."""
    gen = torch.Generator().manual_seed(7)
    f, v, z, s0 = _dev(*_scan_inputs(gen, 3, 200, 72, dtype, True, True))
    y, last = gated_scan(f, v, z, s0)
    state, parts = s0, []
    for t in range(200):
        out, state = gated_scan(f[:, t:t + 1], v[:, t:t + 1], z[:, t:t + 1], state)
        parts.append(out)
    R.assert_scan(torch.cat(parts, 1), y.double().cpu(), dtype, "y")
    R.assert_scan(state, last.double().cpu(), torch.float32, "state")


@pytest.mark.parametrize("steps", [3, 150])
def test_scan_of_views(steps):
    """Inputs cut from one projection's output, time-major storage, an offset that no wide
    access fits, broadcast gates: as copies give."""
    gen = torch.Generator().manual_seed(7)
    wide = normal(gen, 2, steps, 3 * 72 + 5, dtype=torch.float16).to(DEV)
    major = normal(gen, steps, 2, 72, dtype=torch.float16).to(DEV).transpose(0, 1)
    once = wide[:, :1, :72].expand(2, steps, 72)
    cut = [wide[..., i * 72:(i + 1) * 72] for i in range(3)]
    odd = [wide[..., i * 72 + 5:(i + 1) * 72 + 5] for i in range(3)]
    for f, v, z in (cut, odd, (major, cut[1], cut[2]), (once, major, odd[0])):
        copies = [t.contiguous() for t in (f, v, z)]
        y, last, saved = gated_scan_forward(f, v, z)
        y2, last2, saved2 = gated_scan_forward(*copies)
        assert torch.equal(y, y2) and torch.equal(last, last2)
        for a, b in zip(gated_scan_backward(major, saved, last), gated_scan_backward(major.contiguous(), saved2, last)):
            assert torch.equal(a, b)


def test_scan_forgets_and_passes_on():
    """f = -inf: the state is v exactly, whatever finite state came before; f = +inf: unchanged,
    with no gradient to v; a NaN stays in its channel (0 * NaN is NaN, so for good)."""
    gen = torch.Generator().manual_seed(7)
    f, v = normal(gen, 1, 300, 64, mean=2.0).to(DEV), normal(gen, 1, 300, 64).to(DEV)
    f[0, 100], f[0, 200:] = -math.inf, math.inf
    v[0, 50, 3] = math.nan
    s0 = normal(gen, 1, 64).to(DEV)
    y, last, saved = gated_scan_forward(f, v, None, s0)
    assert y[0, 50:, 3].isnan().all() and int(y.isnan().sum()) == 250 and last[0, 3].isnan()
    keep = [c for c in range(64) if c != 3]
    y2, v2 = y[0][:, keep], v[0][:, keep]
    assert torch.equal(y2[100], v2[100]) and torch.equal(y2[299], y2[199]) and torch.equal(last[0, keep], y2[199])
    dy = normal(gen, 1, 300, 64).to(DEV)
    df, dv, _, ds0 = gated_scan_backward(dy, saved, None)
    df, dv = df[0][:, keep], dv[0][:, keep]
    assert (dv[200:] == 0).all() and (df[200:] == 0).all() and (df[100] == 0).all()
    assert torch.isfinite(ds0).all() and torch.isfinite(df).all() and torch.isfinite(dv).all()


def test_scan_of_nothing():
    empty = torch.empty(2, 0, 64, device=DEV)
    s0 = torch.randn(2, 64, device=DEV)
    y, last, saved = gated_scan_forward(empty, empty, empty, s0)
    assert y.shape == (2, 0, 64) and torch.equal(last, s0)
    assert torch.equal(gated_scan_backward(empty, saved, s0)[3], s0)
    assert (gated_scan(empty, empty)[1] == 0).all()
    for shape in ((0, 5, 64), (2, 5, 0)):
        none = torch.empty(shape, device=DEV)
        y, last, saved = gated_scan_forward(none, none)
        assert y.shape == shape and gated_scan_backward(none, saved)[0].shape == shape


def test_scan_autograd_and_differences():
    """Through autograd, and every gradient against the FP32 forward's central difference along
    a random direction (eps 1e-2: the cubic term and the rounding are below 1e-3 of it each)."""
    gen = torch.Generator().manual_seed(11)
    f, v, z = (normal(gen, 2, 150, 40, mean=m).to(DEV).requires_grad_() for m in (2.0, 0.0, 0.0))
    s0 = normal(gen, 2, 40).to(DEV).requires_grad_()
    dy, dlast = normal(gen, 2, 150, 40).to(DEV), normal(gen, 2, 40).to(DEV)
    y, last = gated_recurrence(f, v, z, s0)
    torch.autograd.backward([y, last], [dy, dlast])
    _, _, saved = gated_scan_forward(f, v, z, s0)
    for t, g in zip((f, v, z, s0), gated_scan_backward(dy, saved, dlast)):
        assert torch.equal(t.grad, g)
    tensors = [f, v, z, s0]
    for i, t in enumerate(tensors):
        direction = t.grad / t.grad.square().mean().sqrt()

        def loss(eps):
            moved = [x.detach() for x in tensors]
            moved[i] = moved[i] + eps * direction
            y, last = gated_scan(*moved)
            return (y.double() * dy.double()).sum() + (last.double() * dlast.double()).sum()
        slope = (t.grad.double() * direction.double()).sum()
        found = (loss(1e-2) - loss(-1e-2)) / 2e-2
        assert abs(found - slope) <= 5e-3 * abs(slope), (i, found.item(), slope.item())


def test_scan_refuses():
    f = torch.zeros(2, 5, 64, device=DEV)
    for args, error in (((f.cpu(), f), ValueError), ((f, f.half()), TypeError), ((f.double(), f), TypeError),
                        ((f[0], f), ValueError), ((f, f[:, :4]), ValueError), ((f, f, f[:1]), ValueError),
                        ((f, f, None, f[:, 0].half()), TypeError), ((f, f, None, f[:1, 0]), ValueError),
                        ((f, f, None, f[:, 0].cpu()), ValueError)):
        with pytest.raises(error):
            gated_scan(*args)
    _, _, saved = gated_scan_forward(f, f)
    for args, error in (((f[:, :4], saved), ValueError), ((f.half(), saved), TypeError), ((f, None), TypeError),
                        ((f, saved, f[:1, 0]), ValueError)):
        with pytest.raises(error):
            gated_scan_backward(*args)


# ---- the native path of the wrappers -------------------------------------------
def test_native_path_equals_the_python_path(monkeypatch):
    """Calls that hostlayers.cpp takes give what the Python path gives (taken here by naming
    the stream), and calls that it does not take arrive there."""
    from morph_amd import _lib, activations, ffn, recurrence
    gen = torch.Generator().manual_seed(5)
    weights = [w.to(DEV) for w in _weights(gen, 72, 200, torch.bfloat16)]
    x, dy = (normal(gen, 3, 50, 72, dtype=torch.bfloat16).to(DEV) for _ in range(2))
    s0, ds = (normal(gen, 3, 72).to(DEV) for _ in range(2))

    def results(stream):
        out = [gated_ffn(x, *weights, stream=stream)]
        for keep in ("full", "fp8"):
            y, saved = gated_ffn_forward(x, *weights, keep=keep, stream=stream)
            out += [y, *saved.tensors(), *gated_ffn_backward(dy, saved, *weights, stream=stream)]
            assert saved.shape == x.shape and saved.ff == 200 and saved.dtype == x.dtype and saved.nbytes > 0
        packed = pack_activation(x, stream=stream)
        assert packed.shape == x.shape and packed.dtype == x.dtype
        out += [packed.codes, packed.exponents, unpack_activation(packed, stream=stream),
                unpack_activation(packed, torch.float32, stream=stream)]
        for z in (x, None):
            for state in (s0, None):
                out += gated_scan(x, dy, z, state, stream=stream)
                y, last, saved = gated_scan_forward(x, dy, z, state, stream=stream)
                out += [y, last, saved.states]
                out += [t for t in gated_scan_backward(dy, saved, ds, stream=stream) if t is not None]
        return out

    class Counting:
        def __init__(self):
            self.calls, self.taken = 0, 0

        def __getattr__(self, name):
            def call(*args):
                result = getattr(_lib.layer_calls(), name)(*args)
                self.calls += 1
                self.taken += result is not None
                return result
            return call
    count = Counting()
    for module in (activations, ffn, recurrence):
        monkeypatch.setattr(module, "layer_calls", lambda: count)
    native = results(None)
    assert count.calls == count.taken == 20
    python = results(torch.cuda.current_stream())
    assert count.calls == 20
    assert len(native) == len(python)
    for a, b in zip(native, python):
        assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)
    count.taken = 0
    gated_ffn(x.transpose(0, 1), *weights)                      # a layout that needs a copy
    pack_activation(x[..., :30])
    gated_scan(x[:, :0], x[:, :0])
    assert count.taken == 0


def test_native_path_under_autograd_keeps_no_graph():
    x = torch.randn(4, 64, device=DEV, dtype=torch.float16, requires_grad=True)
    weights = [torch.randn(s, device=DEV, dtype=torch.float16) for s in ((96, 64), (96, 64), (64, 96))]
    y, saved = gated_ffn_forward(x, *weights)
    assert not y.requires_grad and not saved.x.requires_grad
    _, _, kept = gated_scan_forward(x[None], x[None])
    assert not kept.f.requires_grad


def test_operators_in_a_graph():
    """Captured once and replayed, with other inputs in the same places and eager work between:
    each time what the eager calls give."""
    gen = torch.Generator().manual_seed(13)
    rows, d, ff = 130, 72, 2056
    x, dy = (normal(gen, rows, d, dtype=torch.bfloat16).to(DEV) for _ in range(2))
    weights = [w.to(DEV) for w in _weights(gen, d, ff, torch.bfloat16)]
    f, v, z = (normal(gen, 2, 1300, d, mean=m, dtype=torch.bfloat16).to(DEV) for m in (2.0, 0.0, 0.0))

    def step():
        y, saved = gated_ffn_forward(x, *weights, keep="fp8")
        out = [y, *gated_ffn_backward(dy, saved, *weights), gated_ffn(x[:5], *weights)]
        ys, last, kept = gated_scan_forward(f, v, z)
        out += [ys, last, *gated_scan_backward(ys, kept, last)[:3], *gated_scan(f[:, :1], v[:, :1], z[:, :1], last)]
        return out + [unpack_activation(pack_activation(dy))]

    step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(4):
        for t in (x, dy, f, v, z):
            t.copy_(normal(gen, *t.shape, dtype=t.dtype))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), k


def test_another_stream_is_the_callers():
    """On a stream of the caller's own the calls, their workspaces and results stay in its order."""
    gen = torch.Generator().manual_seed(17)
    x = normal(gen, 300, 64, dtype=torch.bfloat16).to(DEV)
    weights = [w.to(DEV) for w in _weights(gen, 64, 2048, torch.bfloat16)]
    f = normal(gen, 1, 4200, 64, dtype=torch.bfloat16).to(DEV)
    y, (s, last) = gated_ffn(x, *weights), gated_scan(f, f)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(20):
            again, (s2, last2) = gated_ffn(x * 1, *weights), gated_scan(f * 1, f * 1)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(y, again) and torch.equal(s, s2) and torch.equal(last, last2)


def test_offsets_past_32_bits():
    """Arrays of more than 2^31 values, whose last rows, steps and groups are those of a small call."""
    rows = 64 * 10990
    x = torch.empty(rows, 3072, dtype=torch.bfloat16, device=DEV)
    assert x.numel() > 1 << 31
    gen = torch.Generator(DEV).manual_seed(19)
    for part in x.split(1 << 16):
        part.normal_(generator=gen)

    packed, tail = pack_activation(x), pack_activation(x[-300:])
    assert torch.equal(packed.codes[-300:], tail.codes) and torch.equal(packed.exponents[-300:], tail.exponents)
    assert torch.equal(unpack_activation(packed)[-300:], unpack_activation(tail))
    del packed, tail

    narrow = x.view(-1, 64)[:1 << 21]
    wide = [(torch.randn(s, generator=gen, device=DEV) / 8).bfloat16() for s in ((1088, 64), (1088, 64), (64, 1088))]
    assert narrow.shape[0] * 1088 > 1 << 31
    assert torch.equal(gated_ffn(narrow, *wide)[-512:], gated_ffn(narrow[-(1 << 19):], *wide)[-512:])

    f, state = x[None], torch.randn(1, 3072, generator=gen, device=DEV)
    y, last, saved = gated_scan_forward(f, f, None, state)
    grads = gated_scan_backward(f, saved, last)
    end = f[:, -128:]
    y2, last2, saved2 = gated_scan_forward(end, end, None, saved.states[:, -2].contiguous())
    # the same formulas on the same values: FP32 sums in another order, each rounded to a step of 2^-7 at most
    for a, b in zip((y, *grads[:2]), (y2, *gated_scan_backward(end, saved2, last2)[:2])):
        a, b = a[:, -128:].float(), b.float()
        assert ((a - b).abs() <= 2.0 ** -7 * b.abs() + 1e-4).all()
    R.assert_scan(last, last2.double().cpu(), torch.float32, "last")
