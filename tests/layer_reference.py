"""Plain float64 implementations of the layer operators, and how far a 16-bit result may be off.

They state the definitions (include/morph_layers.h) directly: the recurrence as a loop over
steps, the 8-bit form value by value."""
import math

import numpy as np
import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
GROUP = 32


def sigmoid(x):
    return torch.special.expit(x)


# ---- 8-bit activations -------------------------------------------------------
def e4m3_values():
    """The value of every E4M3FN code (NaN for 0x7F and 0xFF)."""
    out = np.empty(256)
    for c in range(256):
        sign, exp, man = -1.0 if c & 128 else 1.0, (c >> 3) & 15, c & 7
        out[c] = math.nan if c & 127 == 127 else sign * (
            man * 2.0 ** -9 if exp == 0 else (1 + man / 8) * 2.0 ** (exp - 7))
    return out


def pack(x):
    """(codes [rows, 32 G], exponents [rows, G]) of a 2-D tensor, as numpy uint8 arrays."""
    x = x.double().cpu().numpy()
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    full = np.zeros((rows, groups * GROUP))
    full[:, :cols] = x
    full = full.reshape(rows, groups, GROUP)
    finite = np.isfinite(full)
    amax = np.where(finite, np.abs(full), 0).max(-1)
    exps = np.empty((rows, groups), np.uint8)
    for i in np.ndindex(rows, groups):
        e = 1
        while e < 247 and amax[i] > math.ldexp(448.0, e - 127):
            e += 1 if amax[i] <= math.ldexp(448.0, e - 126) else max(1, int(math.log2(amax[i])) - 9 - (e - 127))
        exps[i] = e
    values = e4m3_values()
    order = values[:127]  # 0 .. 448 ascending with the code
    scaled = np.where(finite, np.abs(full), 0) * np.exp2(127.0 - exps.astype(np.float64))[..., None]
    hi = np.searchsorted(order, scaled).clip(0, 126)
    lo = (hi - 1).clip(0, 126)
    dl, dh = scaled - order[lo], order[hi] - scaled
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.signbit(full), code | 128, code)
    code = np.where(finite, code, 127)
    return code.astype(np.uint8).reshape(rows, -1), exps


def unpack(codes, exponents, cols):
    values = torch.from_numpy(e4m3_values())[codes.cpu().long()]
    scale = torch.exp2(exponents.cpu().double() - 127).repeat_interleave(GROUP, 1)
    return (values * scale)[:, :cols]


# ---- the feed-forward block --------------------------------------------------
def ffn(x, gate, up, down):
    g, u = x @ gate.T, x @ up.T
    h = g * sigmoid(g) * u
    return g, u, h, h @ down.T


def ffn_backward(dy, x, g, u, gate, up, down):
    s = sigmoid(g)
    dh = dy @ down
    dg, du = dh * u * s * (1 + g * (1 - s)), dh * g * s
    h = g * s * u
    return dict(h=h, dg=dg, du=du, dx=dg @ gate + du @ up, dgate=dg.T @ x, dup=du.T @ x, ddown=dy.T @ h)


def assert_product(got, left, right, dtype, what, rounded=1):
    """got against left @ right (float64) where `rounded` of each term's factors were rounded to
    dtype before FP32 sums and one rounding of the result.

    An element's terms carry independent relative errors of at most u each: its error's standard
    deviation is at most u sqrt(rounded / 3) sqrt(sum of squared terms).  Six of them, u |result| for the last
    rounding, and 2^-20 of the terms' magnitudes for FP32 sums and the gate's arithmetic."""
    ref = left @ right
    u = UNIT[dtype]
    spread = ((left ** 2) @ (right ** 2)).sqrt()
    bound = (u * ref.abs() + 6 * u * math.sqrt(rounded / 3) * spread + 2.0 ** -20 * (left.abs() @ right.abs())
             + TINY[dtype] * (1 + right.abs().sum(0, keepdim=True)))
    err = (got.double().cpu() - ref).abs()
    assert torch.isfinite(got).all(), what
    worst = (err / bound.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    assert worst <= 1, f"{what}: error {worst:.3g} of its bound"


# ---- the recurrence ----------------------------------------------------------
def scan(f, v, z, s0):
    a, b = sigmoid(f), sigmoid(-f)
    s = torch.zeros(f.shape[0], f.shape[2], dtype=torch.float64) if s0 is None else s0
    states = []
    for t in range(f.shape[1]):
        s = a[:, t] * s + b[:, t] * v[:, t]
        states.append(s)
    states = torch.stack(states, 1) if states else f.clone()
    return (states if z is None else states * z * sigmoid(z)), s, states


def scan_backward(f, v, z, s0, dy, dlast):
    _, _, states = scan(f, v, z, s0)
    first = torch.zeros_like(f[:, 0]) if s0 is None else s0
    r = torch.zeros_like(first) if dlast is None else dlast
    df, dv = torch.zeros_like(f), torch.zeros_like(f)
    dz = None if z is None else torch.zeros_like(f)
    for t in range(f.shape[1] - 1, -1, -1):
        a, b = sigmoid(f[:, t]), sigmoid(-f[:, t])
        w, prev = dy[:, t], states[:, t - 1] if t else first
        if z is not None:
            q = sigmoid(z[:, t])
            dz[:, t] = w * states[:, t] * q * (1 + z[:, t] * sigmoid(-z[:, t]))
            w = w * z[:, t] * q
        r = r + w
        dv[:, t], df[:, t] = b * r, r * (prev - v[:, t]) * a * b
        r = a * r
    return df, dv, dz, r


def assert_scan(got, ref, dtype, what):
    """A result of the recurrence: FP32 arithmetic, then one rounding to dtype.

    Every step multiplies the state by a gate that is off by 2^-23 or so, and a state remembers
    1 / (1 - a) steps, a hundred or two for the gates in these tests: 2e-5 of the results' size.
    The last rounding adds u of the value itself."""
    ref = ref.double()
    size = ref.square().mean().sqrt().item() if ref.numel() else 0.0
    u = 0.0 if dtype == torch.float32 else UNIT[dtype]
    err = (got.double().cpu() - ref).abs()
    bound = u * ref.abs() + 2e-5 * (size + ref.abs()) + TINY[dtype]
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1, f"{what}: error {worst:.3g} of its bound"
