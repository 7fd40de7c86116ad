"""FusedAdamW with its moments in 8 bits against its definition: codes and exponents bit for bit, masters to
what the hardware's root and reciprocal leave open."""
import numpy as np
import pytest
import torch

import state_space_reference as R
from morph_amd import DynamicLossScale, FusedAdamW

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HYPER = dict(lr=3e-4, betas=(.9, .999), eps=1e-8, weight_decay=.1)


class Twin:
    """One parameter's step on the CPU."""

    def __init__(self, oracle, master, index, seed, scale, hyper=HYPER):
        self.o, self.w, self.index, self.seed, self.scale = oracle, master.numpy().ravel().copy(), index, seed, scale
        self.change, self.hyper, self.step_ = 0 * self.w, hyper, 0
        groups = -(-self.w.size // 32)
        self.m, self.v = (np.zeros(33 * groups, np.uint8) for _ in range(2))

    def step(self, grad):
        self.step_ += 1
        n, f32 = self.w.size, np.float32
        m, v = (x.astype(f32) for x in R.decode_moments(self.m, self.v, n))
        h = self.hyper
        hp = self.o.torch_adamw_hp(h["lr"], *h["betas"], h["eps"], h["weight_decay"], self.step_, scale=self.scale)
        g = grad.float().numpy().ravel() / f32(self.scale)  # a power of two
        with np.errstate(under="ignore"):
            m = m + f32(hp.lerp_weight) * (g - m)
            v = v * f32(hp.beta2) + (f32(hp.one_minus_beta2) * g) * g
        assert m.dtype == v.dtype == f32
        m64, v64, p = m.astype(np.float64), v.astype(np.float64), self.w.astype(np.float64) * hp.decay
        self.change = hp.neg_step_size * m64 / (np.sqrt(v64) / hp.bias_correction2_sqrt + hp.eps)
        self.w = p + self.change
        self.m, self.v = R.encode_moments(m64, v64, R.rounding_bits(n, self.seed, self.index, self.step_))


def compare(opt, twins):
    for k, (p, t) in enumerate(zip(opt.param_groups[0]["params"], twins)):
        got = p.detach().cpu().numpy().ravel().astype(np.float64)
        # root and reciprocal (2^-23 each), the bias correction's inverse and three roundings of 2^-24 are less than
        # 2^-20 of the change; the master is rounded once behind its decay and once at the end
        wrong = np.abs(got - t.w) - 2.0 ** -20 * np.abs(t.change) - 2.0 ** -23 * np.abs(t.w)
        assert (wrong <= 2.0 ** -149).all(), f"master {k}: {wrong.max()}"
        t.w = got  # the next step goes on from here
        for name, mine in (("exp_avg", t.m), ("exp_avg_sq", t.v)):
            held = opt.state[p][name].cpu().numpy()
            assert (held == mine).all(), f"{name} {k}: {np.flatnonzero(held != mine)[:5]} of {held.size}"
        if opt.exports:
            assert torch.equal(opt.exports[k], p.detach().to(opt.exports[k].dtype)), f"export {k}"


SHAPES = [(1,), (31,), (32,), (33,), (255,), (256,), (257,), (40, 50), (1021, 3), (4096, 5), (3, 7, 11)]


@pytest.mark.parametrize("grad_dtype,out_dtype", [(torch.float32, None), (torch.float16, torch.float16),
                                                  (torch.bfloat16, torch.bfloat16), (torch.float16, torch.bfloat16)])
def test_steps_bit_for_bit(oracle, grad_dtype, out_dtype):
    gen = torch.Generator().manual_seed(1)
    scale = 1.0 if grad_dtype == torch.float32 else 1024.0
    masters = [torch.randn(s, generator=gen) * .02 for s in SHAPES]
    opt = FusedAdamW([m.to(DEV) for m in masters], **HYPER, loss_scale=scale, export_dtype=out_dtype, state_bits=8,
                     rounding_seed=77)
    twins = [Twin(oracle, m, i, 77, scale) for i, m in enumerate(masters)]
    for step in range(6):
        size = 10.0 ** (-step)  # moments that have to fade: codes that round to 0, least codes that are kept
        grads = [(torch.randn(s, generator=gen) * torch.randn(s, generator=gen).exp() * 1e-2 * size * scale).to(grad_dtype)
                 for s in SHAPES]
        if step == 3:
            grads[4].zero_()
        opt.step([g.to(DEV) for g in grads])
        for t, g in zip(twins, grads):
            t.step(g)
        compare(opt, twins)
    for (m, v), t, p in zip(opt.moments(), twins, masters):
        em, ev = R.decode_moments(t.m, t.v, p.numel())
        assert m.shape == p.shape and (m.cpu().numpy().ravel() == em).all() and (v.cpu().numpy().ravel() == ev).all()
    exact = opt.moments()
    for dtype in (torch.bfloat16, torch.float16):
        for (m, v), (em, ev) in zip(opt.moments(dtype=dtype), exact):
            assert torch.equal(m, em.to(dtype)) and torch.equal(v, ev.to(dtype))


def test_many_tensors_views_and_a_skip(oracle):
    """More tensors than a launch's arguments hold (the table from the second step on), gradients and masters at odd
    addresses, a parameter without a gradient, and a step that overflows."""
    gen = torch.Generator().manual_seed(2)
    sizes = [int(n) for n in torch.randint(1, 700, (150,), generator=gen)]
    flat = torch.randn(sum(sizes) + 1, generator=gen) * .02
    cut = [flat[1 + sum(sizes[:i]):1 + sum(sizes[:i + 1])] for i in range(len(sizes))]
    held = flat.to(DEV)
    params = [held[1 + sum(sizes[:i]):1 + sum(sizes[:i + 1])] for i in range(len(sizes))]
    scaler = DynamicLossScale(512.0)
    opt = FusedAdamW(params, **HYPER, loss_scale=scaler, export_dtype=torch.float16, sync=True, state_bits=8, rounding_seed=3)
    twins = [Twin(oracle, m, i, 3, 512.0) for i, m in enumerate(cut)]
    for step in range(5):
        grads = [(torch.randn(n, generator=gen) * 5).half() for n in sizes]
        given = torch.cat(grads).to(DEV)
        at = [sum(sizes[:i]) for i in range(len(sizes))]
        device = [given[a:a + n] for a, n in zip(at, sizes)]
        if step == 2:
            device[7] = device[7].clone()
            device[7][0] = float("inf")
            before = [opt.state[p]["exp_avg_sq"].clone() for p in params]
            assert opt.step(device) is False
            assert all(torch.equal(opt.state[p]["exp_avg_sq"], b) for p, b in zip(params, before))
            for t in twins:
                t.scale = scaler.scale
        else:
            device[11] = None
            assert opt.step(device) is True
            for i, (t, g) in enumerate(zip(twins, grads)):
                if i != 11:
                    t.step(g)
        compare(opt, twins)


def test_state_dict_goes_on_where_it_was():
    gen = torch.Generator().manual_seed(3)
    masters = [torch.randn(300, generator=gen), torch.randn(5, 40, generator=gen)]
    grads = [[torch.randn(m.shape, generator=gen).to(DEV) for m in masters] for _ in range(4)]

    def fresh(values):
        return FusedAdamW([v.clone().to(DEV) for v in values], **HYPER, state_bits=8, rounding_seed=9)
    whole, first = fresh(masters), fresh(masters)
    for g in grads:
        whole.step(g)
    for g in grads[:2]:
        first.step(g)
    kept = first.state_dict()
    kept["state"] = {i: {k: v.clone() if torch.is_tensor(v) else v for k, v in s.items()} for i, s in kept["state"].items()}
    second = fresh([p.detach().cpu() for p in first.param_groups[0]["params"]])
    second.load_state_dict(kept)
    for g in grads[2:]:
        second.step(g)
    for a, b in zip(whole.param_groups[0]["params"], second.param_groups[0]["params"]):
        assert torch.equal(a, b)
        assert all(torch.equal(whole.state[a][k], second.state[b][k]) for k in ("exp_avg", "exp_avg_sq"))
    wide = FusedAdamW([m.clone().to(DEV) for m in masters], **HYPER)
    with pytest.raises(ValueError, match="not in 8 bits"):
        second.load_state_dict(wide.state_dict())


def test_the_mean_follows_32_bits():
    """A constant gradient for 400 steps: m goes to g and v to g^2 with beta2 = 0.99, whose steps are smaller than a code's;
    rounding to nearest would leave v where 1% of the way is less than half a code's step.  Over 4096 elements the
    mean of v is within 6 standard deviations of it: a hop of D = v / 8 at most with probability (change / D) gives a
    stationary variance of at most v D / 2, so a deviation of v / 4 an element and v / 256 of the mean."""
    n, g = 4096, 3e-3
    opt = FusedAdamW([torch.zeros(n, device=DEV)], lr=1e-3, betas=(.9, .99), weight_decay=0.0, state_bits=8)
    grad = [torch.full((n,), g, device=DEV)]
    for _ in range(400):
        opt.step(grad)
    (m, v), = opt.moments()
    expected = g * g * (1 - .99 ** 400)
    assert abs(v.double().mean().item() / expected - 1) <= 6 / 256
    assert abs(m.double().mean().item() / g - 1) <= 6 / 256


def test_what_is_beyond_the_largest_float_becomes_it():
    opt = FusedAdamW([torch.zeros(64, device=DEV)], lr=0.0, betas=(.9, .9), weight_decay=0.0, state_bits=8)
    grad = torch.full((64,), 3e38, device=DEV)
    grad[40:] = 1.0
    for _ in range(3):
        opt.step([grad])
    (m, v), = opt.moments()
    assert m.isfinite().all() and v.isfinite().all() and (v[:40] > 2e38).all() and (v[40:] > 0).all()


def test_streams_and_graphs_of_moments():
    gen = torch.Generator().manual_seed(4)
    opt = FusedAdamW([torch.randn(1000, generator=gen).to(DEV) for _ in range(70)], **HYPER, state_bits=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        opt.step([torch.randn(1000, device=DEV) for _ in range(70)])
    torch.cuda.synchronize()
    expected = opt.moments()
    got = opt.moments(stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for x, y in zip(expected, got) for a, b in zip(x, y))


def test_refusals():
    p = torch.zeros(64, device=DEV)
    with pytest.raises(ValueError, match="state_bits must be 8 or 32"):
        FusedAdamW([p], state_bits=4)
    with pytest.raises(ValueError, match="arena"):
        FusedAdamW([p], state_bits=8, arena=True)
    with pytest.raises(ValueError, match="on the CPU"):
        FusedAdamW([torch.zeros(64)], state_bits=8)
    with pytest.raises(ValueError, match="rounding_seed"):
        FusedAdamW([p], state_bits=8, rounding_seed=1 << 32)
    opt = FusedAdamW([p], state_bits=8)
    with pytest.raises(ValueError, match="one pair"):
        opt.moments(out=[])
    with pytest.raises(ValueError, match="must hold 64 values"):
        opt.moments(out=[(torch.empty(63, device=DEV), torch.empty(64, device=DEV))])
    with pytest.raises(ValueError, match="share one dtype"):
        opt.moments(out=[(torch.empty(64, device=DEV), torch.empty(64, device=DEV).half())])
    with pytest.raises(ValueError, match="contiguous"):
        opt.moments(out=[(torch.empty(128, device=DEV)[::2], torch.empty(64, device=DEV))])
    with pytest.raises(TypeError, match="unsupported dtype"):
        opt.moments(dtype=torch.float64)
