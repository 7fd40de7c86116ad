"""Every form of the layer operators' kernels against float64: the sizes are such that the rules in
ffn.hip and scan.hip choose each of them at least once."""
import math

import pytest
import torch

import layer_reference as R
from morph_amd.activations import unpack_activation
from morph_amd.ffn import gated_ffn, gated_ffn_backward, gated_ffn_forward
from morph_amd.recurrence import gated_scan_backward, gated_scan_forward

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)

# rows, d, ff, none a multiple of 32 and few of 8, with the tiles that they stand for: of gate and up, of
# down, of the gate's gradient (FP32 kept / 8 bits), of dx and of the weights' gradients; "/ n": K in n parts.
TILES = [
    (127, 80, 72),       # 64 x 64 throughout
    (4242, 520, 67),     # down and dx 128
    (4086, 1032, 1001),  # 128, but dx 256 x 128
    (4410, 1832, 514),   # gate 256 x 128, down and dx 256, weights 128
    (4104, 913, 920),    # gate 128, down and dx 256 x 128, weights 128
    (457, 904, 4112),    # gate 256 x 128, down and dx 128 / 8, weights 256
    (4049, 480, 4064),   # gate 256, down and dx 128 / 4, gradient 64 / 256, weights 256 x 128
    (1217, 1928, 4724),  # gate 256, down and dx 128 / 2, gradient 256 x 128, weights 256
    (3730, 837, 4300),   # gate and gradient 256, down 128, dx 128 / 2, weights 256
    (2381, 132, 3056),   # gate 256, down and dx 64 / 2
    (86, 72, 1008),      # dx 64 / 4
    (82, 80, 2216),      # down 64 / 4, dx 64 / 8
    (69, 72, 4768),      # down and dx 64 / 8
    (29, 185, 519),      # 17 to 32 rows at odd elements: gate and down by the few-rows kernels
    (50, 185, 519),      # 33 to 64 rows
    (61, 196, 262),      # the same with rows at even elements
]


def _near(got, left, right, what, dtype):
    """layer_reference.assert_product's bound, computed where the tensors are."""
    ref, u = left @ right, R.UNIT[dtype]
    bound = (u * ref.abs() + 6 * u * math.sqrt(1 / 3) * ((left ** 2) @ (right ** 2)).sqrt()
             + 2.0 ** -20 * (left.abs() @ right.abs()) + R.TINY[dtype] * (1 + right.abs().sum(0, keepdim=True)))
    assert torch.isfinite(got).all(), what
    worst = ((got.double() - ref).abs() / bound).max().item()
    assert worst <= 1, f"{what}: error {worst:.3g} of its bound"


def _check_ffn(x, dy, weights, keep):
    dtype, ff = x.dtype, weights[0].shape[0]
    gate, up, down = (w.double() for w in weights)
    g, u, h, _ = R.ffn(x.double(), gate, up, down)
    _near(gated_ffn(x, *weights), h, down.T, "y, nothing kept", dtype)
    y, saved = gated_ffn_forward(x, *weights, keep=keep)
    _near(y, h, down.T, "y", dtype)
    if keep == "full":
        assert (saved.gate[:, ff:] == 0).all() and (saved.up[:, ff:] == 0).all()
        kept = x.double(), saved.gate[:, :ff].double(), saved.up[:, :ff].double()
    else:  # FP32 holds what a code stands for
        kept = tuple(unpack_activation(p, torch.float32).double() for p in saved.packed)
        for p in saved.packed[1:]:
            assert (p.codes[:, ff:] == 0).all()
    for name, got, ref, w in (("g", kept[1], g, gate), ("u", kept[2], u, up)):
        bound = 2.0 ** -20 * (x.double().abs() @ w.abs().T) + 1e-30
        if keep == "fp8":  # half a step: 2^-4 of the value, or 2^-10 of a scale of at most 2^-7.8 of the largest
            bound += 2.0 ** -4 * ref.abs() + 2.0 ** -17 * ref.abs().amax(1, keepdim=True)
        assert ((got - ref).abs() <= bound).all(), name
    ref = R.ffn_backward(dy.double(), *kept, gate, up, down)
    dx, dgate, dup, ddown = gated_ffn_backward(dy, saved, *weights)
    _near(dx, torch.cat([ref["dg"], ref["du"]], 1), torch.cat([gate, up]), "dx", dtype)
    _near(dgate, ref["dg"].T, kept[0], "dgate", dtype)
    _near(dup, ref["du"].T, kept[0], "dup", dtype)
    _near(ddown, dy.double().T, ref["h"], "ddown", dtype)


def _ffn_inputs(rows, d, ff, dtype, more=0):
    """x, dy and the weights, with `more` columns behind each row."""
    gen = torch.Generator(DEV).manual_seed(rows + d + ff)

    def normal(rows, cols, scale=1.0):
        return (torch.randn(rows, cols + more, generator=gen, device=DEV) * scale).to(dtype)
    return (normal(rows, d), normal(rows, d), normal(ff, d, d ** -.5), normal(ff, d, d ** -.5), normal(d, ff, ff ** -.5))


@pytest.mark.parametrize("keep", ["full", "fp8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,d,ff", TILES)
def test_ffn_tiles(rows, d, ff, dtype, keep):
    x, dy, *weights = _ffn_inputs(rows, d, ff, dtype)
    _check_ffn(x, dy, weights, keep)


@pytest.mark.parametrize("keep", ["full", "fp8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,d,ff", [(200, 136, 264), (700, 329, 515), (40, 72, 328)])
def test_ffn_at_other_addresses(rows, d, ff, dtype, keep):
    """One operand, then all, at an address or with a row stride that no 16-byte access fits; gate and up with
    strides of their own."""
    whole = _ffn_inputs(rows, d, ff, dtype)
    wide = _ffn_inputs(rows, d, ff, dtype, more=5)
    cut = [t[:, 3:3 + p.shape[1]] for t, p in zip(wide, whole)]
    for views in [range(5), *((k,) for k in range(5))]:
        x, dy, *weights = (cut[k] if k in views else whole[k] for k in range(5))
        _check_ffn(x, dy, weights, keep)
    spaced = torch.zeros(ff, d + 16, dtype=dtype, device=DEV)[:, :d].copy_(whole[2])
    _check_ffn(whole[0], whole[1], [spaced, *whole[3:]], keep)


# ---- the recurrence -----------------------------------------------------------------
def _long_memory(batch, steps, dim, dtype, gate):
    """All gates but one in a thousand are 1: what enters a tile, a run and a stretch counts until the end."""
    gen = torch.Generator(DEV).manual_seed(batch + steps + dim)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)
    f = torch.full((batch, steps, dim), math.inf, device=DEV)
    some = torch.rand(batch, steps, dim, generator=gen, device=DEV) < .001
    f[some] = (1.5 * normal(int(some.sum())) + 2).clamp_(-4, 4)
    f = f.to(dtype)
    v, dy = (normal(batch, steps, dim).to(dtype) for _ in range(2))
    z = normal(batch, steps, dim).to(dtype) if gate else None
    return f, v, z, normal(batch, dim), dy, normal(batch, dim)


def _check_scan(batch, steps, dim, dtype, gate, sampled):
    f, v, z, s0, dy, dlast = _long_memory(batch, steps, dim, dtype, gate)
    y, last, saved = gated_scan_forward(f, v, z, s0)
    grads = gated_scan_backward(dy, saved, dlast)
    # channels at both ends of the kernels' groups of 64 and 128, and others
    ends = [0, 1, 62, 63, 64, 65, 126, 127, 128, 129, dim - 130, dim - 129, dim - 128, dim - 65, dim - 64, dim - 2, dim - 1]
    c = torch.tensor(sorted({k for k in ends if 0 <= k < dim} | set(range(5, dim, max(1, dim // sampled)))), device=DEV)

    def cut(t):
        return None if t is None else t.index_select(-1, c).double().cpu()
    args = cut(f), cut(v), cut(z), cut(s0)
    ref_y, ref_last, _ = R.scan(*args)
    R.assert_scan(cut(y), ref_y, dtype, "y")
    R.assert_scan(cut(last), ref_last, torch.float32, "last")
    ref = R.scan_backward(*args, cut(dy), cut(dlast))
    for name, a, b in zip(("df", "dv", "dz"), grads, ref):
        if a is not None:
            R.assert_scan(cut(a), b, dtype, name)
    R.assert_scan(cut(grads[3]), ref[3], torch.float32, "ds0")


@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,steps,dim", [(2, 3333, 1100), (1, 2500, 2048), (2, 2111, 1101), (3, 5001, 330), (17, 1300, 64)])
def test_scan_of_many_groups(batch, steps, dim, dtype, gate):
    """Channel groups from 9 to 36, runs that are stretches of their own from 16 on, one and two channels a
    lane."""
    _check_scan(batch, steps, dim, dtype, gate, 12)


@pytest.mark.parametrize("dtype,batch,steps,dim,gate", [
    (torch.bfloat16, 1, 16500, 2048, True), (torch.float16, 3, 5600, 2048, True), (torch.float32, 1, 33000, 512, True),
    (torch.bfloat16, 2, 11000, 2048, False), (torch.float16, 1, 22000, 2048, False), (torch.float32, 1, 22000, 1024, False)])
def test_scan_past_the_caches(dtype, batch, steps, dim, gate):
    """Whole cache lines, and more than 256 MB of them in the forward as in the backward."""
    assert batch * steps * dim * (4 if gate else 3) * (4 if dtype == torch.float32 else 2) > 256 << 20
    _check_scan(batch, steps, dim, dtype, gate, 12)
