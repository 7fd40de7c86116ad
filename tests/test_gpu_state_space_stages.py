"""The example that runs the state space operators together, with the 8-bit optimizer step."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch

import state_space_reference as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "state_space_stages.py"
    spec = importlib.util.spec_from_file_location("state_space_stages", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _plain_operators():
    def norm(x, w=None, b=None):
        return R.norm(x, w, b, 1e-5)[3]

    def conv(x, w, b, state):
        _, y, after = R.conv(x, w, b, state)
        return y, after

    def scan(x, dt, A, B, C, skip, z, bias, first):
        d, h, s = R.softplus(dt + bias), torch.zeros(x.shape[0], *A.shape, dtype=x.dtype), []
        for t in range(x.shape[1]):
            h = torch.exp(d[:, t, :, None] * A) * h + (d[:, t] * x[:, t])[..., None] * B[:, t, None]
            s.append((h * C[:, t, None]).sum(2))
        return (torch.stack(s, 1) + skip * x) * z * torch.sigmoid(z), h
    return norm, conv, scan


def test_the_example_runs():
    losses, _ = _example().main(["--steps", "3"])
    assert len(losses) == 3 and all(math.isfinite(x) for x in losses)


def test_the_models_gradients():
    """The loss in FP32 and the gradients of every weight, against the same model in float64."""
    m = _example()
    gen = torch.Generator().manual_seed(2)
    tokens = torch.randint(m.VOCAB, (2, 40), generator=gen)

    def run(cast, operators, tokens):
        table, stages = m.first_weights(torch.Generator().manual_seed(3))
        table, stages = cast(table), [tuple({k: cast(t) for k, t in part.items()} for part in s) for s in stages]
        leaves = [table] + [t for s in stages for part in s for t in part.values()]
        loss = m.loss_of(tokens, table, stages, operators)
        return loss, torch.autograd.grad(loss, leaves)
    ref, refs = run(lambda t: t.double().requires_grad_(), _plain_operators(), tokens)
    loss, grads = run(lambda t: t.to(DEV).requires_grad_(), m.OPERATORS, tokens.to(DEV))
    R.assert_scan(loss.detach(), ref.detach(), torch.float32, "loss")
    for k, (g, r) in enumerate(zip(grads, refs)):
        R.assert_scan(g, r, torch.float32, f"gradient {k}")


def test_token_by_token_is_the_prompt():
    """In FP32 on the model's own weights: the last output over a prompt, and fed token by token."""
    m = _example()
    table, stages = m.first_weights(torch.Generator().manual_seed(4))
    table, stages = table.to(DEV), [tuple({k: t.to(DEV) for k, t in part.items()} for part in s) for s in stages]
    tokens = torch.randint(m.VOCAB, (2, 70), generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.no_grad():
        whole = torch.nn.functional.embedding(tokens, table)
        for w, v in stages:
            whole, _ = m.stage(whole, w, v)
        states, out = [(None, None)] * m.STAGES, []
        for t in range(70):
            x = torch.nn.functional.embedding(tokens[:, t:t + 1], table)
            for i, (w, v) in enumerate(stages):
                x, states[i] = m.stage(x, w, v, states[i])
            out.append(x)
    R.assert_scan(torch.cat(out, 1), whole.cpu(), torch.float32, "token by token")
