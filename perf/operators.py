"""Performance cases of the layer operators: the gated feed-forward block, activation
checkpoints in 8 bits, and the gated linear recurrence.

listed() names the cases, draw() gives more over the same ranges; prepare() makes what the
program holds before the call, run() makes one pass and returns everything it computed:
through morph_amd where `own` is true, else in plain FP32 torch operations.  exact() is the
same pass in float64, written on its own.

Kinds:
  ffn     y = (silu(x Wg^T) * (x Wu^T)) Wd^T, forward only (serving)
  train   the block's forward and its backward; keep says what lies between them:
          "full" the projections in FP32, "fp8" x and the projections in 8 bits
  pack    an activation to 8 bits and back
  scan    a = sigmoid(f), s_t = a_t s_(t-1) + (1 - a_t) v_t, y = s silu(z): outputs and the
          last state, from a first one
  scan_train  the same with its backward: gradients of f, v, z and the first state

The 8-bit form: 32 consecutive values of a row share the scale 2^k with the least k for
which their largest magnitude is at most 448 * 2^k; each is the nearest E4M3 value times it.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
GROUP = 32  # values that share a scale


# ---------------------------------------------------------------- the cases --
def listed():
    return [
        # one token through the 5B model's block: the weights cross once
        dict(name="ffn_token", kind="ffn", rows=1, d=3072, ff=6144, dtype="bf16"),
        # a batch of tokens of an ordinary model while it answers: latency
        dict(name="ffn_few", kind="ffn", rows=24, d=768, ff=2048, dtype="f16"),
        # a prompt through the 5B model's block
        dict(name="ffn_prompt", kind="ffn", rows=2048, d=3072, ff=6144, dtype="bf16"),
        # a small model's training step, a batch that fills no tile and an odd width
        dict(name="ffn_step_small", kind="train", rows=333, d=200, ff=535, dtype="f16", keep="full"),
        # the 5B stage's step over 4 sequences of 1024 tokens, FP16 compute
        dict(name="ffn_step", kind="train", rows=4096, d=3072, ff=6144, dtype="f16", keep="full"),
        # its largest batch, kept in 8 bits between forward and backward
        dict(name="ffn_step_fp8", kind="train", rows=8192, d=3072, ff=6144, dtype="bf16", keep="fp8"),
        # a small model's boundary activation
        dict(name="pack_small", kind="pack", rows=96, d=200, dtype="f16"),
        # the boundary of 16 sequences of the 5B model, on its way to the host
        dict(name="pack_boundary", kind="pack", rows=16384, d=3072, dtype="bf16"),
        # one step of 64 sequences being written
        dict(name="scan_token", kind="scan", batch=64, steps=1, d=3072, dtype="bf16", gate=True),
        # prompts of a small model in FP32, of a length and width that fit nothing
        dict(name="scan_prompt", kind="scan", batch=3, steps=1000, d=1100, dtype="f32", gate=False),
        # the 5B stage's step over 4 sequences of 1024 tokens
        dict(name="scan_step", kind="scan_train", batch=4, steps=1024, d=3072, dtype="f16", gate=True),
        # one long document
        dict(name="scan_step_long", kind="scan_train", batch=1, steps=65536, d=3072, dtype="bf16",
             gate=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Widths in use are multiples of 64, or at least of 8; a few are neither."""
    w, by = _log(rng, lo, hi), rng.choice([64, 64, 8, 8, 1])
    return max(by, w // by * by)


def draw(rng):
    kind = rng.choice(["ffn", "ffn", "train", "train", "pack", "scan", "scan_train", "scan_train"])
    half = rng.choice(["f16", "bf16"])
    if kind in ("ffn", "train"):
        d = _width(rng, 64, 3072)
        ff = min(6144, max(d, int(d * rng.uniform(1.3, 4)) // 8 * 8))
        if d % 8:
            ff += rng.randint(0, 7)
        case = dict(kind=kind, rows=_log(rng, 1, 8192), d=d, ff=min(6144, ff), dtype=half)
        return dict(case, keep=rng.choice(["full", "fp8"])) if kind == "train" else case
    if kind == "pack":
        return dict(kind=kind, rows=_log(rng, 1, 16384), d=_width(rng, 64, 3072),
                    dtype=rng.choice([half, half, "f32"]))
    d, dtype = _width(rng, 64, 3072), rng.choice([half, half, "f32"])
    steps = 1 if kind == "scan" and rng.random() < 0.3 else _log(rng, 2, 65536)
    most = max(1, (65536 * 3072) // (steps * d * (2 if dtype == "f32" else 1)))
    return dict(kind=kind, batch=_log(rng, 1, min(64, most)), steps=min(steps, most * steps), d=d,
                dtype=dtype, gate=rng.random() < 0.7)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(shape, scale=1.0, mean=0.0, to=dtype):
        x = torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, 1.0, generator=gen)
        return x.mul_(scale).add_(mean).to(to)

    state = dict(case=case)
    if case["kind"] in ("ffn", "train"):
        rows, d, ff = case["rows"], case["d"], case["ff"]
        state.update(x=normal((rows, d)), gate=normal((ff, d), d ** -0.5), up=normal((ff, d), d ** -0.5),
                     down=normal((d, ff), ff ** -0.5))
        if case["kind"] == "train":
            state.update(dy=normal((rows, d)))
    elif case["kind"] == "pack":
        # channels of a residual stream differ in size, a few by much
        x = normal((case["rows"], case["d"]), to=torch.float32)
        x *= torch.exp(1.5 * normal((case["d"],), to=torch.float32))
        state.update(x=x.clamp_(-60000, 60000).to(dtype))
    else:
        shape = (case["batch"], case["steps"], case["d"])
        f = normal(shape, 1.5, 2.0)
        # packed documents: the state is forgotten where a new one begins
        begins = torch.rand(shape[:2], device="cuda", generator=gen) < 1 / 500
        f.masked_fill_(begins[..., None], -math.inf)
        state.update(f=f, v=normal(shape), z=normal(shape) if case["gate"] else None,
                     s0=normal((case["batch"], case["d"]), to=torch.float32))
        if case["kind"] == "scan_train":
            state.update(dy=normal(shape), ds=normal((case["batch"], case["d"]), to=torch.float32))
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] in ("ffn", "train"):
        rows, d, ff = case["rows"], case["d"], case["ff"]
        if case["kind"] == "ffn":  # x and the weights in, y out
            return {"bytes": size * (2 * rows * d + 3 * d * ff), "flops": 6 * rows * d * ff}
        # x, dy and the weights in; y, dx and their gradients out
        return {"bytes": size * (4 * rows * d + 6 * d * ff), "flops": 18 * rows * d * ff}
    if case["kind"] == "pack":  # values in, codes out and in again, values out
        n = case["rows"] * case["d"]
        return {"bytes": 2 * n * (size + 1 + 1 / GROUP), "flops": 4 * n}
    n, tensors = case["batch"] * case["steps"] * case["d"], 3 if case["gate"] else 2
    ends = 8 * case["batch"] * case["d"]
    if case["kind"] == "scan":  # the inputs and y; the two states
        return {"bytes": size * n * (tensors + 1) + ends, "flops": 10 * n}
    # forward as above; backward, which in use comes much later: the inputs and dy, their gradients
    return {"bytes": size * n * (3 * tensors + 2) + 2 * ends, "flops": 30 * n}


# ------------------------------------------------------- the framework's calls --
def _run_own(state):
    from morph_amd.activations import pack_activation, unpack_activation
    from morph_amd.ffn import gated_ffn, gated_ffn_backward, gated_ffn_forward
    from morph_amd.recurrence import gated_scan, gated_scan_backward, gated_scan_forward

    case = state["case"]
    if case["kind"] == "ffn":
        return gated_ffn(state["x"], state["gate"], state["up"], state["down"])
    if case["kind"] == "train":
        weights = state["gate"], state["up"], state["down"]
        y, saved = gated_ffn_forward(state["x"], *weights, keep=case["keep"])
        return y, *gated_ffn_backward(state["dy"], saved, *weights)
    if case["kind"] == "pack":
        return unpack_activation(pack_activation(state["x"]))
    inputs = state["f"], state["v"], state["z"], state["s0"]
    if case["kind"] == "scan":
        return gated_scan(*inputs)
    y, last, saved = gated_scan_forward(*inputs)
    return y, last, *gated_scan_backward(state["dy"], saved, state["ds"])


# --------------------------------------------------------------- the plain form --
def _grouped(x):
    """x with its rows filled up to whole groups, as [rows, groups, GROUP]."""
    rows, d = x.shape
    full = torch.zeros(rows, -(-d // GROUP) * GROUP, device=x.device, dtype=x.dtype)
    full[:, :d] = x
    return full.view(rows, -1, GROUP)


def _eight_bits(x):
    """The values that x's 8-bit form stands for, in x's type (float32)."""
    groups = _grouped(x)
    most = groups.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(most / 448)
    k = (exponent - (mantissa == 0.5).to(exponent.dtype)).clamp(-126, 120)
    one = torch.ones_like(most)
    codes = torch.ldexp(groups, -k).to(torch.float8_e4m3fn)
    values = codes.to(torch.float32) * torch.ldexp(one, k)
    return values.view(x.shape[0], -1)[:, :x.shape[1]]


def _linear_scan(a, b):
    """s_t = a_t s_(t-1) + b_t along dim 1, s_0 = 0: each pass joins every step's span with
    the equally long one before it, so log2 of the steps passes (a product of the gates over
    the whole length and a division would underflow)."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _run_plain(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] in ("ffn", "train"):
        x, wg, wu, wd = (state[k].float() for k in ("x", "gate", "up", "down"))
        g, u = x @ wg.T, x @ wu.T
        y = (g * torch.sigmoid(g) * u) @ wd.T
        if case["kind"] == "ffn":
            return y.to(dtype)
        if case["keep"] == "fp8":
            x, g, u = _eight_bits(x), _eight_bits(g), _eight_bits(u)
        dy, s = state["dy"].float(), torch.sigmoid(g)
        dh = dy @ wd
        dg, du = dh * u * s * (1 + g * (1 - s)), dh * g * s
        out = y, dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ (g * s * u)
        return tuple(o.to(dtype) for o in out)
    if case["kind"] == "pack":
        return _eight_bits(state["x"].float()).to(dtype)
    f, v = state["f"].float(), state["v"].float()
    a, keep = torch.sigmoid(f), torch.sigmoid(-f)
    b = keep * v
    b[:, 0] += a[:, 0] * state["s0"]
    s = _linear_scan(a, b)
    z = state["z"].float() if case["gate"] else None
    out = s if z is None else s * z * torch.sigmoid(z)
    if case["kind"] == "scan":
        return out.to(dtype), s[:, -1].clone()
    dy = state["dy"].float()
    dz = None
    w = dy
    if z is not None:
        sz = torch.sigmoid(z)
        dz = (dy * s * sz * (1 + z * (1 - sz))).to(dtype)
        w = dy * z * sz
    w = w.clone() if z is None else w
    w[:, -1] += state["ds"]
    # the gradient of the state runs backward: r_t = w_t + a_(t+1) r_(t+1)
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    r = _linear_scan(after.flip(1), w.flip(1)).flip(1)
    before = torch.cat([state["s0"][:, None], s[:, :-1]], 1)
    df = r * (before - v) * a * keep
    return out.to(dtype), s[:, -1].clone(), df.to(dtype), (r * keep).to(dtype), dz, a[:, 0] * r[:, 0]


# ------------------------------------------------------------------ in 64 bits --
def _nearest_e4m3(q):
    """The nearest E4M3 value (3 bits of mantissa, ties to even, subnormals of 2^-9)."""
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(q / step) * step


def _exact_eight_bits(x):
    groups = _grouped(x)
    most = groups.abs().amax(-1, keepdim=True)
    k = torch.ceil(torch.log2((most / 448).clamp_min(2.0 ** -126))).clamp(-126, 120)
    scale = torch.exp2(k)
    return (_nearest_e4m3(groups / scale) * scale).view(x.shape[0], -1)[:, :x.shape[1]]


def _exact_scan(a, b, s0):
    """States by the recurrence itself, in blocks: every block's from zero side by side, then
    the blocks one after the other."""
    batch, steps, d = a.shape
    size = max(1, int(steps ** 0.5))
    count = -(-steps // size)
    pa = torch.ones(batch, count * size, d, device=a.device, dtype=torch.float64)
    pb = torch.zeros_like(pa)
    pa[:, :steps], pb[:, :steps] = a, b
    pa, pb = pa.view(batch, count, size, d), pb.view(batch, count, size, d)
    for i in range(1, size):
        pb[:, :, i] += pa[:, :, i] * pb[:, :, i - 1]
        pa[:, :, i] *= pa[:, :, i - 1]
    carry = s0
    for c in range(count):
        pb[:, c] += pa[:, c] * carry[:, None]
        carry = pb[:, c, -1]
    return pb.reshape(batch, -1, d)[:, :steps]


def exact(case, seed):
    state = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    sigma = torch.special.expit
    if case["kind"] in ("ffn", "train"):
        x, wg, wu, wd = (state[k] for k in ("x", "gate", "up", "down"))
        g, u = torch.mm(x, wg.t()), torch.mm(x, wu.t())
        y = torch.mm(g * sigma(g) * u, wd.t())
        if case["kind"] == "ffn":
            return y
        if case["keep"] == "fp8":
            x, g, u = _exact_eight_bits(x), _exact_eight_bits(g), _exact_eight_bits(u)
        dy, s = state["dy"], sigma(g)
        dh = torch.mm(dy, wd)
        dg, du = dh * u * (s + g * s * (1 - s)), dh * (g * s)
        return (y, torch.mm(dg, wg) + torch.mm(du, wu), torch.mm(dg.t(), x), torch.mm(du.t(), x),
                torch.mm(dy.t(), g * s * u))
    if case["kind"] == "pack":
        return _exact_eight_bits(state["x"])
    f, v, z, s0 = state["f"], state["v"], state["z"], state["s0"]
    a, b = sigma(f), sigma(-f)
    s = _exact_scan(a, b * v, s0)
    gate = torch.ones_like(s) if z is None else z * sigma(z)
    if case["kind"] == "scan":
        return s * gate, s[:, -1]
    dy = state["dy"]
    # reversed time: the gate that multiplies step t's result is the one of the step after it
    late = torch.ones_like(a)
    late[:, 1:] = a[:, 1:].flip(1)
    r = _exact_scan(late, (dy * gate).flip(1), state["ds"]).flip(1)
    dz = None if z is None else dy * s * (sigma(z) + z * sigma(z) * sigma(-z))
    before = torch.cat([s0[:, None], s[:, :-1]], 1)
    return s * gate, s[:, -1], r * (before - v) * a * b, r * b, dz, a[:, 0] * r[:, 0]
