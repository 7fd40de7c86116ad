"""Plain float64 implementations of the layer norm, the causal convolution, the selective scan and the 8-bit
moments, and how far a result may be off.

They state the definitions (include/morph_state_space.h, morph_optim.h) directly; the scan is a loop over steps."""
import numpy as np
import torch

from layer_reference import TINY, UNIT, e4m3_values, sigmoid

EPS32 = 2.0 ** -24


# ---- layer norm ----------------------------------------------------------------
def norm(x, w, b, eps):
    mean = x.mean(-1, keepdim=True)
    r = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * r
    return mean, r, xh, (xh if w is None else xh * w) + (0 if b is None else b)


def norm_backward(dy, xh, r, w):
    g = dy if w is None else dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def norm_bounds(x, w, b, dy, eps, dtype, wdtype):
    """Bounds of y, dx, dweight and dbias.

    A row's sum takes at most 64 additions in a row a lane and a tree: 64 units of 2^-24 of the mean magnitude, so
    x - mean is off by 64 (|x| + mean |x|) units, xh by r times that and by 64 of itself for r.  What is made of it is off
    by as much times its factors; sums over rows add 256 units of their terms (their longest chain is shorter)."""
    _, r, xh, y = norm(x, w, b, eps)
    w = torch.ones_like(x[:1]) if w is None else w
    b = torch.zeros_like(x[:1]) if b is None else b
    e = 64 * EPS32 * (r * (x.abs() + x.abs().mean(-1, keepdim=True)) + xh.abs())
    ey = UNIT[dtype] * y.abs() + e * w.abs() + 2 * EPS32 * (y.abs() + b.abs()) + TINY[dtype]
    if dy is None:
        return ey
    dx, dw, db = norm_backward(dy, xh, r, w)
    g = (dy * w).abs()
    sizes = g + g.mean(-1, keepdim=True) + xh.abs() * (g * xh.abs()).mean(-1, keepdim=True)
    through = e * (g * xh.abs()).mean(-1, keepdim=True) + xh.abs() * (g * e).mean(-1, keepdim=True)
    edx = UNIT[dtype] * dx.abs() + r * (128 * EPS32 * sizes + through) + TINY[dtype]
    own = 0.0 if wdtype == torch.float32 else UNIT[wdtype]
    edw = own * dw.abs() + (dy.abs() * (e + 256 * EPS32 * xh.abs())).sum(0) + TINY[wdtype]
    edb = own * db.abs() + 256 * EPS32 * dy.abs().sum(0) + TINY[wdtype]
    return ey, edx, edw, edb


# ---- causal convolution ----------------------------------------------------------
def _joined(x, before, taps):
    if before is None:
        before = torch.zeros(x.shape[0], taps - 1, x.shape[2], dtype=x.dtype)
    return torch.cat([before, x], 1)


def conv(x, w, b, before):
    taps, steps = w.shape[1], x.shape[1]
    xs = _joined(x, before, taps)
    p = torch.zeros_like(x) + (0 if b is None else b)
    for k in range(taps):
        p = p + w[:, k] * xs[:, k:k + steps]
    return p, p * sigmoid(p), xs[:, steps:]


def conv_backward(dy, x, w, b, before, dafter):
    taps, steps = w.shape[1], x.shape[1]
    xs = _joined(x, before, taps)
    p, _, _ = conv(x, w, b, before)
    dp = dy * sigmoid(p) * (1 + p * sigmoid(-p))
    dxs, dw = torch.zeros_like(xs), torch.zeros_like(w)
    for k in range(taps):
        dxs[:, k:k + steps] += w[:, k] * dp
        dw[:, k] = (dp * xs[:, k:k + steps]).sum((0, 1))
    if dafter is not None:
        dxs[:, steps:] += dafter
    return dxs[:, taps - 1:], dw, dp.sum((0, 1)), dxs[:, :taps - 1]


def conv_bounds(x, w, b, before, dy, dafter, dtype, wdtype):
    """Bounds of y, and with dy of dx, dweight, dbias and dbefore.

    p is off by (taps + 2) units of 2^-24 of its terms; silu and its slope change by at most 1.1 times that, and their
    own arithmetic (an exponential whose argument is rounded, a reciprocal) is off by 2^-20 for |p| <= 8.  Sums of
    gradients add 256 units of their terms (a lane adds one run's steps, then parts are joined)."""
    taps, steps = w.shape[1], x.shape[1]
    xs = _joined(x, before, taps).abs()
    p, y, _ = conv(x, w, b, before)
    ep = torch.zeros_like(p) + (0 if b is None else b.abs())
    for k in range(taps):
        ep = ep + w[:, k].abs() * xs[:, k:k + steps]
    ep = ep * (taps + 2) * EPS32
    ey = UNIT[dtype] * y.abs() + 1.1 * ep + 2.0 ** -20 * y.abs() + TINY[dtype]
    if dy is None:
        return ey
    dx, dw, db, dbefore = conv_backward(dy, x, w, b, before, dafter)
    edp = dy.abs() * (1.1 * ep + 2.0 ** -20)
    full = edp + 8 * EPS32 * dy.abs()
    edx, edw = torch.zeros_like(xs), torch.zeros_like(w)
    for k in range(taps):
        edx[:, k:k + steps] += w[:, k].abs() * full
        edw[:, k] = ((edp + 256 * EPS32 * dy.abs() * 1.1) * xs[:, k:k + steps]).sum((0, 1))
    if dafter is not None:
        edx[:, steps:] += 2 * EPS32 * dafter.abs()
    own = 0.0 if wdtype == torch.float32 else UNIT[wdtype]
    u, tiny = UNIT[dtype], TINY[dtype]
    return (ey, edx[:, taps - 1:] + u * dx.abs() + tiny, edw + own * dw.abs() + TINY[wdtype],
            (edp + 256 * EPS32 * dy.abs() * 1.1).sum((0, 1)) + own * db.abs() + TINY[wdtype],
            edx[:, :taps - 1] + u * dbefore.abs() + tiny)


# ---- selective scan ----------------------------------------------------------------
def softplus(x):
    return torch.logaddexp(x, torch.zeros_like(x))


def scan(x, dt, A, B, C, skip, z, bias, first):
    raw = dt if bias is None else dt + bias
    d = softplus(raw)
    h = torch.zeros(x.shape[0], *A.shape, dtype=x.dtype) if first is None else first
    states, s = [h], torch.zeros_like(x)
    for t in range(x.shape[1]):
        h = torch.exp(d[:, t, :, None] * A) * h + (d[:, t] * x[:, t])[..., None] * B[:, t, None]
        s[:, t] = (h * C[:, t, None]).sum(2)
        states.append(h)
    if skip is not None:
        s = s + skip * x
    return raw, d, states, s, (s if z is None else s * z * sigmoid(z))


def scan_backward(dy, dlast, x, dt, A, B, C, skip, z, bias, first):
    """In selective_scan's order of arguments."""
    raw, d, states, s, _ = scan(x, dt, A, B, C, skip, z, bias, first)
    dz = None if z is None else dy * s * sigmoid(z) * (1 + z * sigmoid(-z))
    ds = dy if z is None else dy * z * sigmoid(z)
    dx = torch.zeros_like(x) if skip is None else skip * ds
    dd, dA, dB, dC = torch.zeros_like(x), torch.zeros_like(A), torch.zeros_like(B), torch.zeros_like(C)
    r = torch.zeros_like(states[0]) if dlast is None else dlast
    for t in range(x.shape[1] - 1, -1, -1):
        r = r + ds[:, t, :, None] * C[:, t, None]
        rB = (r * B[:, t, None]).sum(2)
        dx[:, t] += d[:, t] * rB
        dB[:, t] = (r * (d[:, t] * x[:, t])[..., None]).sum(1)
        dC[:, t] = (states[t + 1] * ds[:, t, :, None]).sum(1)
        r = torch.exp(d[:, t, :, None] * A) * r
        w = r * states[t]
        dA += (w * d[:, t, :, None]).sum(0)
        dd[:, t] = x[:, t] * rB + (w * A).sum(2)
    ddt = dd * sigmoid(raw)
    return (dx, ddt, dA, dB, dC, None if skip is None else (ds * x).sum((0, 1)), dz,
            None if bias is None else ddt.sum((0, 1)), r)


def assert_scan(got, ref, dtype, what):
    """A result of the scan or its backward: FP32 arithmetic, then one rounding to dtype.

    A gate is off by 2^-23 or so of itself each step, in either direction, and a state remembers 1 / (d |A|) steps, up to
    2000 in these tests: 6 standard deviations are 6 sqrt(2000) 2^-23 = 3.2e-5 of the results' size.  Sums over steps and
    channels add what is off independently in their terms, so they are off by no more of their own size."""
    ref = ref.double()
    size = ref.square().mean().sqrt().item() if ref.numel() else 0.0
    u = 0.0 if dtype == torch.float32 else UNIT[dtype]
    assert_within(got, ref, u * ref.abs() + 3.2e-5 * (size + ref.abs()) + TINY[dtype], what)


def assert_within(got, ref, bound, what):
    assert tuple(got.shape) == tuple(ref.shape), f"{what}: {tuple(got.shape)}"
    err = (got.double().cpu() - ref).abs()
    assert torch.isfinite(err).all(), f"{what}: not finite"
    worst = (err / bound.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1, f"{what}: error {worst:.3g} of its bound"


# ---- moments in 8 bits ------------------------------------------------------------
GROUP = 32
SECOND = np.array([(c & 7) / 8 * 2.0 ** -30 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 31) for c in range(256)])


def mix(x):
    x = np.asarray(x, np.uint64) & 0xFFFFFFFF
    x = x ^ (x >> np.uint64(16))
    x = x * np.uint64(0x6A09E667) & np.uint64(0xFFFFFFFF)
    x = x ^ (x >> np.uint64(15))
    x = x * np.uint64(0xBB67AE85) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def rounding_bits(n, seed, tensor, step):
    """(16 bits for the first moment, 16 for the second) of every place."""
    key = mix(mix(seed + (tensor + 1) * 0x9E3779B9) ^ np.uint64(step & 0xFFFFFFFF))
    words = mix(np.arange(n, dtype=np.uint64) ^ key)
    return words & np.uint64(0xFFFF), words >> np.uint64(16)


def _grouped(x):
    full = np.zeros(-(-x.size // GROUP) * GROUP)
    full[:x.size] = x
    return full.reshape(-1, GROUP)


def _encode(x, values, top, least, most, bits):
    """Codes and exponents of x >= 0: the code below x, or the next one where the part of the way to it that x has gone
    and `bits` / 2^16 come to one."""
    groups, amax = _grouped(x), _grouped(x).max(1)
    e = np.full(amax.size, least)
    for i in np.flatnonzero(amax > np.ldexp(top, least - 127)):
        e[i] = min(most, int(np.ceil(np.log2(amax[i] / top) - 1e-9)) + 127)
        while e[i] > least and amax[i] <= np.ldexp(top, e[i] - 128):
            e[i] -= 1
        while e[i] < most and amax[i] > np.ldexp(top, e[i] - 127):
            e[i] += 1
    scaled = groups / np.ldexp(1.0, e - 127)[:, None]
    low = np.searchsorted(values, scaled, side="right") - 1
    low = low.clip(0, values.size - 2)
    part = (scaled - values[low]) / (values[low + 1] - values[low])
    code = low + (np.floor(part * 65536 + _grouped(bits)) >= 65536)
    return code.clip(0, values.size - 1), e


def encode_moments(m, v, bits):
    """Two float64 arrays of FP32 values as the two moments' uint8 buffers."""
    out = []
    first, second = e4m3_values()[:127], SECOND[:255]
    code, e = _encode(np.abs(m), first, 448.0, 1, 247, bits[0])
    code = np.where(np.signbit(np.concatenate([m, np.zeros(code.size - m.size)])).reshape(code.shape), code | 128, code)
    out.append(np.concatenate([code.ravel(), e]).astype(np.uint8))
    code, e = _encode(v, second, 1.75, 11, 254, bits[1])
    code = np.where((_grouped(v) > 0) & (code == 0), 1, code)
    out.append(np.concatenate([code.ravel(), e]).astype(np.uint8))
    return out


def decode_moments(m, v, n):
    """The float64 values of the two buffers."""
    out = []
    for buffer, values, zero in ((m, e4m3_values(), 127), (v, SECOND, 127)):
        groups = buffer.size // (GROUP + 1)
        codes, e = buffer[:groups * GROUP], buffer[groups * GROUP:].astype(np.int64)
        out.append((values[codes].reshape(-1, GROUP) * np.ldexp(1.0, e - zero)[:, None]).ravel()[:n])
    return out
