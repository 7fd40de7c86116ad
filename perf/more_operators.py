"""Performance cases of a state space stage and its optimizer step: the layer norm, the short causal
convolution, the selective scan, and AdamW with its moments in 8 bits.

listed() names the cases, draw() gives more over the same ranges; prepare() makes what the
program holds before the call, run() makes one pass and returns everything it computed:
through morph_amd where `own` is true, else in plain FP32 torch operations.  exact() is the
same pass in float64, written on its own.

Kinds (with train: the forward and its backward, every gradient returned):
  norm   y = (x - mean) / sqrt(var + eps) * weight + bias along a row
  conv   y = silu(bias + sum_k weight_k x_(t-K+1+k)) along the steps, with the K - 1 inputs before the
         first step, and those behind the last one returned
  scan   d = softplus(dt + dt_bias), h_t = exp(d_t A) h_(t-1) + d_t x_t B_t,
         y = (sum_n C_t h_t + skip x_t) silu(z_t): outputs and the last state, from a first one
  adamw  a step of FusedAdamW(state_bits=8) over a list of tensors: the masters, their FP16 copies, and
         the values that the moments' codes stand for

The moments' 8-bit form: 32 consecutive values share the power of two 2^(e - 127).  A first moment is an
E4M3 code, a second one an unsigned code of 5 exponent bits (bias 31) and 3 mantissa bits.  Each is
rounded down or up with the probabilities that leave its mean as it is, by 16 bits of a hash of
seed, tensor, step and place; a second moment that is not 0 keeps the least code at least.
"""
import itertools
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
GROUP = 32  # values that share a scale
SCALE = 65536.0  # loss scale of the gradients
HYPER = dict(lr=3e-4, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
STEP = 100  # steps taken before the measured one
SEED = 5  # of the rounding
EPS = 1e-5  # of the norm


# ---------------------------------------------------------------- the cases --
def listed():
    return [
        # the rows of a few tokens while they are being written: latency
        dict(name="norm_token", kind="norm", rows=8, d=4096, dtype="bf16", train=False),
        # a small model's training step: an odd width, a batch that fills nothing
        dict(name="norm_step_odd", kind="norm", rows=333, d=1021, dtype="f16", train=True),
        # a training batch of 16 sequences of 1024 tokens
        dict(name="norm_step", kind="norm", rows=16384, d=4096, dtype="bf16", train=True),
        # one token of 64 sequences being written
        dict(name="conv_token", kind="conv", batch=64, steps=1, d=5120, taps=4, dtype="bf16", train=False),
        # a training batch of 4 sequences
        dict(name="conv_step", kind="conv", batch=4, steps=2048, d=5120, taps=4, dtype="bf16", train=True),
        # one token of 64 sequences being written: the states cross in and out
        dict(name="scan_token", kind="scan", batch=64, steps=1, d=5120, states=16, dtype="bf16", gate=True,
             train=False),
        # prompts of a small model in FP32, of a length and width that fit nothing
        dict(name="scan_prompt", kind="scan", batch=3, steps=777, d=1100, states=16, dtype="f32", gate=False,
             train=False),
        # one long document read in
        dict(name="scan_prompt_long", kind="scan", batch=1, steps=32768, d=2048, states=16, dtype="bf16",
             gate=True, train=False),
        # a small model's training step
        dict(name="scan_step_small", kind="scan", batch=2, steps=333, d=200, states=8, dtype="f16", gate=True,
             train=True),
        # a training batch of 4 sequences of 1024 tokens
        dict(name="scan_step", kind="scan", batch=4, steps=1024, d=5120, states=16, dtype="bf16", gate=True,
             train=True),
        # the norms, biases and convolutions of a model: many small tensors, odd sizes among them
        dict(name="adamw8_vectors", kind="adamw", shapes="4096*120,5120*30,20480*30,1021*20", dtype="f16"),
        # a stage's three feed-forward matrices
        dict(name="adamw8_window", kind="adamw", shapes="25165824*3", dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Widths in use are multiples of 64, or at least of 8; a few are neither."""
    w, by = _log(rng, lo, hi), rng.choice([64, 64, 8, 8, 1])
    return max(by, w // by * by)


def draw(rng):
    kind = rng.choice(["norm", "conv", "scan", "scan", "scan", "adamw"])
    half = rng.choice(["f16", "bf16"])
    dtype = rng.choice([half, half, "f32"])
    if kind == "norm":
        d, train = _width(rng, 64, 8192), rng.random() < 0.6
        most = 16384 * 4096 // (d * (2 if dtype == "f32" else 1))
        return dict(kind=kind, rows=_log(rng, 1, min(65536, most)), d=d, dtype=dtype, train=train)
    if kind == "adamw":
        sizes = []
        for _ in range(rng.randint(1, 6)):
            n = _log(rng, 200, 1 << 24)
            sizes.append(f"{n}*{rng.randint(1, max(1, min(60, (1 << 24) // n)))}")
        return dict(kind=kind, shapes=",".join(sizes), dtype=dtype)
    train = rng.random() < 0.5
    steps = 1 if not train and rng.random() < 0.35 else _log(rng, 2, 16384)
    d = _width(rng, 64, 5120)
    if kind == "conv":
        most = 4 * 2048 * 5120 // (2 if dtype == "f32" else 1) // d
        steps = min(steps, most)
        return dict(kind=kind, batch=_log(rng, 1, min(64, most // steps)), steps=steps, d=d,
                    taps=rng.choice([4, 4, 4, 3, 2]), dtype=dtype, train=train)
    n = rng.choice([16, 16, 16, 8, 4, 12, 32, 64])
    most = (4 * 1024 * 5120 * 16 if train else 32768 * 2048 * 16) // (2 if dtype == "f32" else 1) // (d * n)
    steps = min(steps, most)
    return dict(kind=kind, batch=_log(rng, 1, min(64, most // steps)), steps=steps, d=d, states=n, dtype=dtype,
                gate=rng.random() < 0.7, train=train)


def _sizes(case):
    """Elements of each tensor."""
    out = []
    for part in case["shapes"].split(","):
        n, _, count = part.partition("*")
        out += [int(n)] * int(count or 1)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(shape, scale=1.0, mean=0.0, to=dtype):
        x = torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, 1.0, generator=gen)
        return x.mul_(scale).add_(mean).to(to)

    def uniform(shape, lo, hi):
        return torch.empty(shape, device="cuda", dtype=torch.float32).uniform_(lo, hi, generator=gen)

    state = dict(case=case)
    if case["kind"] == "norm":
        rows, d = case["rows"], case["d"]
        # channels of a residual stream differ in size, and it is not centred
        size = torch.exp(0.7 * normal((d,), to=torch.float32))
        state.update(x=(normal((rows, d), to=torch.float32) * size + 0.3 * normal((d,), to=torch.float32)).to(dtype),
                     weight=normal((d,), 0.2, 1.0, torch.float32), bias=normal((d,), 0.2, to=torch.float32))
        if case["train"]:
            state.update(dy=normal((rows, d)))
    elif case["kind"] == "conv":
        shape, taps = (case["batch"], case["steps"], case["d"]), case["taps"]
        state.update(x=normal(shape), weight=uniform((case["d"], taps), -taps ** -0.5, taps ** -0.5),
                     bias=uniform((case["d"],), -taps ** -0.5, taps ** -0.5),
                     before=normal((case["batch"], taps - 1, case["d"])))
        if case["train"]:
            state.update(dy=normal(shape), dafter=normal((case["batch"], taps - 1, case["d"])))
    elif case["kind"] == "scan":
        b, steps, d, n = case["batch"], case["steps"], case["d"], case["states"]
        # A near -1 .. -N and steps of 0.001 to 0.1, as such layers are initialised, and spread by training
        A = torch.arange(-1, -n - 1, -1, device="cuda") * torch.exp(normal((d, n), 0.2, to=torch.float32))
        step = torch.exp(uniform((d,), math.log(0.001), math.log(0.1)))
        state.update(x=normal((b, steps, d)), dt=normal((b, steps, d), 0.7), A=A,
                     B=normal((b, steps, n)), C=normal((b, steps, n)), skip=normal((d,), 0.2, 1.0, torch.float32),
                     z=normal((b, steps, d)) if case["gate"] else None, dt_bias=torch.log(torch.expm1(step)),
                     h0=normal((b, d, n), 0.5, to=torch.float32))
        if case["train"]:
            state.update(dy=normal((b, steps, d)), dlast=normal((b, d, n), to=torch.float32))
    else:
        # the tensors lie behind each other, each from a group's first place on
        sizes = _sizes(case)
        ends = list(itertools.accumulate(-(-n // GROUP) * GROUP for n in sizes))
        starts, total = [0, *ends[:-1]], ends[-1]
        inside = torch.zeros(total, device="cuda", dtype=torch.bool)
        for at, n in zip(starts, sizes):
            inside[at:at + n] = True

        def flat(scale, to=torch.float32):
            return normal((total,), scale, to=torch.float32).mul_(inside).to(to)
        grads, masters = flat(1e-4 * SCALE, dtype), flat(0.02)
        # moments after some steps: groups of them differ in size by much
        size = 1e-4 * torch.exp(normal((total // GROUP, 1), 1.0, to=torch.float32))
        m = (flat(0.3).view(-1, GROUP) * size).reshape(-1)
        v = ((flat(0.5).view(-1, GROUP).abs() + 0.5) * size).square().reshape(-1).mul_(inside)
        half = torch.full((total,), 1 << 15, device="cuda", dtype=torch.int64)
        first, second = _encode_first(m, half), _encode_second(v, half)
        state.update(sizes=sizes, starts=starts, masters=masters, grads=grads, exports=masters.to(torch.float16),
                     first=first, second=second, step=STEP)
        if own:
            state.update(_optimizer(state))
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] == "norm":
        n = case["rows"] * case["d"]
        # the input in, the output out; backward, which in use comes much later: both and their gradients
        return {"bytes": n * size * (5 if case["train"] else 2) + case["d"] * (24 if case["train"] else 8),
                "flops": n * (24 if case["train"] else 8)}
    if case["kind"] == "conv":
        n, ends = case["batch"] * case["steps"] * case["d"], case["batch"] * case["d"] * (case["taps"] - 1)
        times, both = (5, 4) if case["train"] else (2, 2)
        return {"bytes": size * (n * times + ends * both) + 2 * both * case["d"] * (case["taps"] + 1),
                "flops": n * case["taps"] * (8 if case["train"] else 2)}
    if case["kind"] == "scan":
        n = case["batch"] * case["steps"] * case["d"]
        small = 2 * case["batch"] * case["steps"] * case["states"]
        ends, gate = case["batch"] * case["d"] * case["states"] * 4, 1 if case["gate"] else 0
        if not case["train"]:  # x, dt, z, B, C and the first state in, y and the last state out
            return {"bytes": size * (n * (3 + gate) + small) + 2 * ends + 4 * case["d"] * (case["states"] + 2),
                    "flops": 7 * n * case["states"]}
        return {"bytes": size * (n * (3 + gate + 3 + gate + 2 + gate) + 3 * small) + 4 * ends
                + 12 * case["d"] * (case["states"] + 2), "flops": 28 * n * case["states"]}
    # the gradient; master and moments in and out; the FP16 copy; the moments' values in 16 bits
    n = sum(_sizes(case))
    return {"bytes": n * (size + 8 + 4 * (1 + 1 / GROUP) + 2 + 4), "flops": 30 * n}


# ------------------------------------------------------- the framework's calls --
def _optimizer(state):
    """The optimizer over the state's masters, with its moments and step."""
    from morph_amd import FusedAdamW

    def views(flat):
        return [flat[at:at + n] for at, n in zip(state["starts"], state["sizes"])]

    def buffers(codes, exponents):
        return [torch.cat([codes[at:at + -(-n // GROUP) * GROUP], exponents[at // GROUP:at // GROUP + -(-n // GROUP)]])
                for at, n in zip(state["starts"], state["sizes"])]

    params = views(state["masters"])
    opt = FusedAdamW(params, **HYPER, loss_scale=SCALE, export_dtype=torch.float16, state_bits=8, rounding_seed=SEED)
    opt.set_exports(views(state["exports"]))
    kept = opt.state_dict()
    kept["state"] = {i: dict(step=STEP, exp_avg=m, exp_avg_sq=v) for i, (m, v) in enumerate(
        zip(buffers(*state["first"]), buffers(*state["second"])))}
    opt.load_state_dict(kept)
    first, second = (torch.zeros_like(state["masters"], dtype=torch.bfloat16) for _ in range(2))
    return dict(opt=opt, views=views(state["grads"]), values=(first, second),
                out=list(zip(views(first), views(second))))


def _run_own(state):
    case = state["case"]
    if case["kind"] == "norm":
        from morph_amd.norm import layer_norm, layer_norm_backward, layer_norm_forward
        if not case["train"]:
            return layer_norm(state["x"], state["weight"], state["bias"], EPS)
        y, saved = layer_norm_forward(state["x"], state["weight"], state["bias"], EPS)
        return y, *layer_norm_backward(state["dy"], saved)
    if case["kind"] == "conv":
        from morph_amd.selective import causal_conv, causal_conv_backward, causal_conv_forward
        inputs = state["x"], state["weight"], state["bias"], state["before"]
        if not case["train"]:
            return causal_conv(*inputs)
        y, after, saved = causal_conv_forward(*inputs)
        return y, after, *causal_conv_backward(state["dy"], saved, state["dafter"])
    if case["kind"] == "scan":
        from morph_amd.selective import selective_scan, selective_scan_backward, selective_scan_forward
        inputs = [state[k] for k in ("x", "dt", "A", "B", "C", "skip", "z", "dt_bias", "h0")]
        if not case["train"]:
            return selective_scan(*inputs)
        y, last, saved = selective_scan_forward(*inputs)
        return y, last, *selective_scan_backward(state["dy"], saved, state["dlast"])
    state["opt"].step(state["views"])
    state["opt"].moments(out=state["out"])
    return state["masters"], state["exports"], *state["values"]


# --------------------------------------------------------------- the plain form --
def _mix(x):
    """A hash of 32-bit words (int64 tensors that hold them)."""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random(sizes, step):
    """32 bits for every place of the tensors' groups."""
    spans = torch.tensor([-(-n // GROUP) * GROUP for n in sizes])
    starts = torch.cumsum(spans, 0) - spans
    tensor = torch.arange(1, len(sizes) + 1)
    key = _mix((SEED + tensor * 0x9E3779B9) & 0xFFFFFFFF)
    key = _mix(key ^ step)
    spans, starts, key = (t.cuda() for t in (spans, starts, key))
    total = sum(-(-n // GROUP) * GROUP for n in sizes)
    place = torch.arange(total, device="cuda") - starts.repeat_interleave(spans, output_size=total)
    return _mix(place ^ key.repeat_interleave(spans, output_size=total))


def _scales(x, top, least):
    """The exponent byte of each group: the least e >= `least` with every value at most top * 2^(e - 127)."""
    most = x.view(-1, GROUP).abs().amax(1)
    mantissa, e = torch.frexp(most / top)
    e = (e - (mantissa == 0.5).to(e.dtype) + 127).clamp(least, 254)
    return torch.where(most > 0, e, torch.full_like(e, least))


def _bits(x, shift, random):
    """x * 2^shift's upper 12 bits as an FP32 number, rounded by 16 random bits."""
    scaled = torch.ldexp(x, shift.repeat_interleave(GROUP))
    return (scaled.view(torch.int32).to(torch.int64) + (random << 4)) >> 20


def _encode_first(m, random):
    e = _scales(m, 448.0, 1)
    code = _bits(m.abs(), 7 - e, random) | (m.view(torch.int32) < 0).to(torch.int64) << 7
    return code.to(torch.uint8), e.to(torch.uint8)


def _encode_second(v, random):
    e = _scales(v, 1.75, 11)
    code = _bits(v, 31 - e, random)
    return torch.where(v > 0, code.clamp_min(1), code).to(torch.uint8), e.to(torch.uint8)


def _decode_first(codes, e):
    code = codes.to(torch.int32)
    value = torch.ldexp(((code & 127) << 20).view(torch.float32), (e.to(torch.int32) - 7).repeat_interleave(GROUP))
    return torch.where(code > 127, -value, value)


def _decode_second(codes, e):
    bits = codes.to(torch.int32) << 20
    return torch.ldexp(bits.view(torch.float32), (e.to(torch.int32) - 31).repeat_interleave(GROUP))


def _linear_scan(a, b):
    """s_t = a_t s_(t-1) + b_t along dim 1, s_0 = 0: each pass joins every step's span with
    the equally long one before it, so log2 of the steps passes."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _run_plain(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    forms = dict(norm=_plain_norm, conv=_plain_conv, scan=_plain_scan, adamw=_plain_adamw)
    return forms[case["kind"]](state, case, dtype)


def _plain_norm(state, case, dtype):
    x, w, b = state["x"].float(), state["weight"], state["bias"]
    centred = x - x.mean(1, keepdim=True)
    r = torch.rsqrt(centred.square().mean(1, keepdim=True) + EPS)
    xh = centred * r
    y = (xh * w + b).to(dtype)
    if not case["train"]:
        return y
    dy = state["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return y, dx.to(dtype), (dy * xh).sum(0), dy.sum(0)


def _plain_conv(state, case, dtype):
    steps, taps = case["steps"], case["taps"]
    w = state["weight"]
    x = torch.cat([state["before"], state["x"]], 1)
    after = x[:, steps:].clone()
    x = x.float()
    # [taps, batch, steps, d]: what each tap sees
    seen = x.unfold(1, steps, 1).permute(1, 0, 3, 2) if steps else x.new_zeros(taps, x.shape[0], 0, x.shape[2])
    p = (seen * w.t()[:, None, None]).sum(0) + state["bias"]
    s = torch.sigmoid(p)
    y = (p * s).to(dtype)
    if not case["train"]:
        return y, after
    dp = state["dy"].float() * s * (1 + p * (1 - s))
    dw = (seen * dp).sum((1, 2)).t().contiguous()
    # every input's gradient gathers from the taps that saw it: those of later steps
    late = torch.cat([torch.zeros_like(x[:, :taps - 1]), dp, torch.zeros_like(x[:, :taps - 1])], 1)
    late = late.unfold(1, taps, 1)  # [batch, steps + taps - 1, d, taps]: dp of t .. t + taps - 1
    dx = (late * w.flip(1)).sum(3)
    dx[:, steps:] += state["dafter"].float()
    return y, after, dx[:, taps - 1:].to(dtype), dw, dp.sum((0, 1)), dx[:, :taps - 1].to(dtype)


def _plain_scan(state, case, dtype):
    x, dt, B, C = (state[k].float() for k in ("x", "dt", "B", "C"))
    A, skip, h0 = state["A"], state["skip"], state["h0"]
    z = state["z"].float() if case["gate"] else None
    raw = dt + state["dt_bias"]
    d = raw.clamp_min(0) + torch.log1p(torch.exp(-raw.abs()))
    a = torch.exp(d[..., None] * A)
    u = (d * x)[..., None] * B[:, :, None]
    u[:, 0] += a[:, 0] * h0
    h = _linear_scan(a, u)
    s = (h * C[:, :, None]).sum(3) + skip * x
    sz = torch.sigmoid(z) if z is not None else None
    y = (s if z is None else s * z * sz).to(dtype)
    last = h[:, -1].clone()
    if not case["train"]:
        return y, last
    dy = state["dy"].float()
    dz = (dy * s * sz * (1 + z * (1 - sz))).to(dtype) if z is not None else None
    ds = dy if z is None else dy * z * sz
    w = ds[..., None] * C[:, :, None]
    w[:, -1] += state["dlast"]
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    r = _linear_scan(after.flip(1), w.flip(1)).flip(1)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    rB = (r * B[:, :, None]).sum(3)
    rha = r * before * a
    dd = x * rB + (rha * A).sum(3)
    ddt = dd * torch.sigmoid(raw)
    return (y, last, (d * rB + skip * ds).to(dtype), ddt.to(dtype), (rha * d[..., None]).sum((0, 1)),
            (r * (d * x)[..., None]).sum(2).to(dtype), (h * ds[..., None]).sum(2).to(dtype), (ds * x).sum((0, 1)), dz,
            ddt.sum((0, 1)), a[:, 0] * r[:, 0])


def _plain_adamw(state, case, dtype):
    beta1, beta2 = HYPER["betas"]
    g = state["grads"].float()
    fine = torch.isfinite(g).all()
    g = g * (1 / SCALE)
    m, v = _decode_first(*state["first"]), _decode_second(*state["second"])
    state["step"] += 1
    t = state["step"]
    m = m + (1 - beta1) * (g - m)
    v = v * beta2 + (1 - beta2) * g * g
    d = torch.sqrt(v) / math.sqrt(1 - beta2 ** t) + HYPER["eps"]
    p = state["masters"] * (1 - HYPER["lr"] * HYPER["weight_decay"]) - HYPER["lr"] / (1 - beta1 ** t) * m / d
    random = _random(state["sizes"], t)
    first, second = _encode_first(m, random & 0xFFFF), _encode_second(v, random >> 16)
    for name, new in (("masters", p), ("exports", p.to(torch.float16))):
        state[name].copy_(torch.where(fine, new, state[name]))
    for name, new in (("first", first), ("second", second)):
        state[name] = tuple(torch.where(fine, b, a) for a, b in zip(state[name], new))
    return (state["masters"], state["exports"], _decode_first(*state["first"]).to(torch.bfloat16),
            _decode_second(*state["second"]).to(torch.bfloat16))


# ------------------------------------------------------------------ in 64 bits --
def exact(case, seed):
    given = prepare(case, seed)
    state = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in given.items()}
    forms = dict(norm=_exact_norm, conv=_exact_conv, scan=_exact_scan, adamw=_exact_adamw)
    return forms[case["kind"]](state, case)


def _exact_norm(state, case):
    x, w, b = state["x"], state["weight"], state["bias"]
    n = case["d"]
    mean = torch.einsum("ij->i", x)[:, None] / n
    var = torch.einsum("ij,ij->i", x, x)[:, None] / n - mean * mean
    xh = (x - mean) / torch.sqrt(var + EPS)
    if not case["train"]:
        return xh * w + b
    dy = state["dy"]
    g = dy * w
    dot = torch.einsum("ij,ij->i", g, xh)[:, None]
    dx = (n * g - torch.einsum("ij->i", g)[:, None] - xh * dot) / (n * torch.sqrt(var + EPS))
    return xh * w + b, dx, torch.einsum("ij,ij->j", dy, xh), torch.einsum("ij->j", dy)


def _exact_conv(state, case):
    steps, taps = case["steps"], case["taps"]
    w, x = state["weight"], torch.cat([state["before"], state["x"]], 1)
    p = torch.zeros_like(state["x"]) + state["bias"]
    for k in range(taps):
        p = p + w[:, k] * x[:, k:k + steps]
    sigma = torch.special.expit
    y = p * sigma(p)
    if not case["train"]:
        return y, x[:, steps:]
    dp = state["dy"] * (sigma(p) + p * sigma(p) * sigma(-p))
    dx, dw = torch.zeros_like(x), torch.empty_like(w)
    for k in range(taps):
        dx[:, k:k + steps] += w[:, k] * dp
        dw[:, k] = (x[:, k:k + steps] * dp).flatten(0, 1).sum(0)
    dx[:, steps:] += state["dafter"]
    return y, x[:, steps:], dx[:, taps - 1:], dw, dp.flatten(0, 1).sum(0), dx[:, :taps - 1]


def _exact_scan(state, case):
    """Step by step, forward and back; the states stay for the way back."""
    x, dt, A, B, C, skip, z, h = (state[k] for k in ("x", "dt", "A", "B", "C", "skip", "z", "h0"))
    sigma = torch.special.expit
    raw = dt + state["dt_bias"]
    d = torch.logaddexp(raw, torch.zeros_like(raw))
    train, steps = case["train"], case["steps"]
    s, states = torch.empty_like(x), [h]
    for t in range(steps):
        h = torch.exp(d[:, t, :, None] * A) * h + (d[:, t] * x[:, t])[..., None] * B[:, t, None]
        s[:, t] = torch.matmul(h, C[:, t, :, None])[..., 0]
        if train:
            states.append(h)
    s += skip * x
    gate = torch.ones_like(x) if z is None else z * sigma(z)
    if not train:
        return s * gate, h
    dy = state["dy"]
    ds = dy * gate
    dz = None if z is None else dy * s * (sigma(z) + z * sigma(z) * sigma(-z))
    dx, dd, dB, dC, dA = skip * ds, torch.empty_like(d), torch.empty_like(B), torch.empty_like(C), torch.zeros_like(A)
    r = state["dlast"]
    for t in range(steps - 1, -1, -1):
        r = r + ds[:, t, :, None] * C[:, t, None]
        rB = torch.matmul(r, B[:, t, :, None])[..., 0]
        dx[:, t] += d[:, t] * rB
        dB[:, t] = (r * (d[:, t] * x[:, t])[..., None]).sum(1)
        dC[:, t] = (states[t + 1] * ds[:, t, :, None]).sum(1)
        r = torch.exp(d[:, t, :, None] * A) * r
        through = r * states[t]
        dA += (through * d[:, t, :, None]).sum(0)
        dd[:, t] = x[:, t] * rB + (through * A).sum(2)
    ddt = dd * sigma(raw)
    return (s * gate, states[-1], dx, ddt, dA, dB, dC, (ds * x).flatten(0, 1).sum(0), dz, ddt.flatten(0, 1).sum(0), r)


def _exact_round(x, top, exponents, least, most_exponent, random):
    """x [groups, GROUP] >= 0 on the 8-bit form's values: `exponents` binades below most_exponent in steps of
    an eighth, of groups scaled to at most `top`."""
    k = torch.ceil(torch.log2(x.amax(1, keepdim=True).clamp_min(1e-300) / top)).clamp(least - 127, 127)
    scaled = x * torch.exp2(-k)
    floor = most_exponent - exponents + 1
    step = torch.exp2(torch.floor(torch.log2(scaled.clamp_min(2.0 ** floor))).clamp_min(floor) - 3)
    return torch.floor(scaled / step + random.view(-1, GROUP).double() / 65536), step, torch.exp2(k)


def _exact_adamw(state, case):
    beta1, beta2 = HYPER["betas"]
    g = state["grads"] / SCALE
    t = STEP + 1
    m = _decode_first(*state["first"]).double()
    v = _decode_second(*state["second"]).double()
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g ** 2
    mhat, vhat = m / (1 - beta1 ** t), v / (1 - beta2 ** t)
    p = state["masters"]
    p = p - HYPER["lr"] * HYPER["weight_decay"] * p - HYPER["lr"] * mhat / (vhat.sqrt() + HYPER["eps"])
    random = _random(state["sizes"], t)
    count, step, scale = _exact_round(m.abs().view(-1, GROUP), 448.0, 15, 1, 8, random & 0xFFFF)
    first = (count * step * scale).reshape(-1) * torch.sign(m)
    v = v.view(-1, GROUP)
    count, step, scale = _exact_round(v, 1.75, 31, 11, 0, random >> 16)
    second = (torch.where(v > 0, count.clamp_min(1), count) * step * scale).reshape(-1)
    return p, p, first, second
