"""The float64 references of the state space operators, on the CPU: gradients against differences, and the 8-bit
moments against what their definition promises."""
import numpy as np
import pytest
import torch

import state_space_reference as R


def _close_to_differences(f, grads, tensors, gen):
    """d/de f(t + e v) at e = 0 for a random v against the gradient; f is smooth, so central differences with
    e = 1e-5 are off by about 1e-10 of f's size."""
    for k, (t, g) in enumerate(zip(tensors, grads)):
        v = torch.randn(t.shape, generator=gen, dtype=torch.float64)
        ends = [f(*(x + s * 1e-5 * v if i == k else x for i, x in enumerate(tensors))) for s in (1, -1)]
        slope = (ends[0] - ends[1]).item() / 2e-5
        assert abs(slope - (g * v).sum().item()) <= 1e-7 * (1 + abs(slope)), k


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, dtype=torch.float64)


def test_norm_gradients():
    gen = torch.Generator().manual_seed(1)
    x, w, b, dy = _normal(gen, 5, 13), _normal(gen, 13), _normal(gen, 13), _normal(gen, 5, 13)
    _, r, xh, _ = R.norm(x, w, b, 1e-5)
    _close_to_differences(lambda x, w, b: (R.norm(x, w, b, 1e-5)[3] * dy).sum(), R.norm_backward(dy, xh, r, w), [x, w, b], gen)


@pytest.mark.parametrize("steps", [1, 2, 7])
def test_conv_gradients(steps):
    gen = torch.Generator().manual_seed(2)
    x, w, b, s = _normal(gen, 2, steps, 3), _normal(gen, 3, 4), _normal(gen, 3), _normal(gen, 2, 3, 3)
    dy, dafter = _normal(gen, 2, steps, 3), _normal(gen, 2, 3, 3)

    def f(x, w, b, s):
        _, y, after = R.conv(x, w, b, s)
        return (y * dy).sum() + (after * dafter).sum()
    _close_to_differences(f, R.conv_backward(dy, x, w, b, s, dafter), [x, w, b, s], gen)


def test_scan_gradients():
    gen = torch.Generator().manual_seed(3)
    b, t, d, n = 2, 6, 3, 4
    inputs = [_normal(gen, b, t, d), _normal(gen, b, t, d), -_normal(gen, d, n).exp(), _normal(gen, b, t, n),
              _normal(gen, b, t, n), _normal(gen, d), _normal(gen, b, t, d), _normal(gen, d), _normal(gen, b, d, n)]
    dy, dlast = _normal(gen, b, t, d), _normal(gen, b, d, n)

    def f(*inputs):
        *_, states, _, y = R.scan(*inputs)
        return (y * dy).sum() + (states[-1] * dlast).sum()
    _close_to_differences(f, R.scan_backward(dy, dlast, *inputs), inputs, gen)


# ---- moments ---------------------------------------------------------------------
def test_moments_round_without_bias():
    """Over all 2^16 roundings a moment's mean is itself, to the 2^-16 of a code's step that the bits resolve."""
    rng = np.random.default_rng(4)
    m, v = rng.normal(size=32) * 1e-3, np.square(rng.normal(size=32) * 1e-3)
    bits = np.arange(0, 1 << 16, 64)
    mean = [np.zeros(32), np.zeros(32)]
    for b in bits:
        pair = R.decode_moments(*R.encode_moments(m, v, [np.full(32, b, np.uint64)] * 2), 32)
        mean = [a + x / bits.size for a, x in zip(mean, pair)]
    # a code's step is an eighth of its value, or the least code; 64 roundings at once leave 2^-10 of it
    for got, x, least in ((mean[0], m, np.abs(m).max() / 448 * 2.0 ** -8), (mean[1], v, v.max() * 2.0 ** -32)):
        assert (np.abs(got - x) <= (np.abs(x) / 8 + least) * 2.0 ** -9).all()


def test_moments_keep_what_is_not_zero():
    v = np.zeros(40)
    v[3], v[5], v[35] = 1.0, 1e-30, 1e-44
    m, s = R.encode_moments(np.zeros(40), v, [np.zeros(40, np.uint64)] * 2)
    got = R.decode_moments(m, s, 40)[1]
    assert got[3] == 1.0 and got[5] == 2.0 ** -33 and got[35] > 0 and (got[v == 0] == 0).all()


def test_rounding_bits_are_spread():
    """Frequencies of the upper 4 bits, and of pairs of neighbouring places, steps and tensors: each count is within 6
    standard deviations of its mean."""
    n = 1 << 16
    words = {k: np.stack(R.rounding_bits(n, *k)) >> np.uint64(12) for k in ((0, 0, 1), (0, 0, 2), (0, 1, 1), (1, 0, 1))}
    base = words[0, 0, 1]
    pairs = [(base[0], base[1]), (base[0][:-1], base[0][1:]), (base[1][:-1], base[1][1:])]
    pairs += [(base[h], words[k][h]) for k in words if k != (0, 0, 1) for h in (0, 1)]
    for a, b in pairs:
        counts = np.bincount((a * np.uint64(16) + b).astype(np.int64), minlength=256)
        assert (np.abs(counts - a.size / 256) <= 6 * (a.size / 256) ** 0.5).all()
