"""A small language model of state space stages, trained by the optimizer step that keeps its moments in 8 bits.

Each stage is a layer norm, a projection, the short causal convolution and the selective scan, and a projection
back.  FP16 weights and activations under a dynamic loss scale, FP32 vectors (norms, convolution, scan), FP32
masters; the gradients of the micro-batches are summed in FP32 windows that test them for the step.  Then the model
continues a sequence token by token from the states that its prompt left.

    python examples/state_space_stages.py [--steps 60]

The text is synthetic: each symbol is followed by another one nine times out of ten, drawn once.
"""
import argparse
import math
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from morph_amd import DynamicLossScale, FusedAdamW  # noqa: E402
from morph_amd.grads import StageGradients  # noqa: E402
from morph_amd.norm import layer_normalization  # noqa: E402
from morph_amd.selective import causal_convolution, selective_state_space  # noqa: E402

VOCAB, WIDTH, INNER, STATES, TAPS, STAGES = 64, 96, 160, 16, 4, 3
MATRICES = dict(into=(2 * INNER, WIDTH), mix=(2 * STATES + INNER, INNER), out=(WIDTH, INNER))
VECTORS = dict(scale=(WIDTH,), shift=(WIDTH,), taps=(INNER, TAPS), tap_bias=(INNER,), log_a=(INNER, STATES),
               skip=(INNER,), dt_bias=(INNER,))
OPERATORS = layer_normalization, causal_convolution, selective_state_space


def stage(x, w, v, states=(None, None), operators=OPERATORS):
    """(x behind the stage, its states); x: [batch, steps, WIDTH], w and v: the matrices and vectors by name."""
    norm, conv, scan = operators
    u, z = (norm(x, v["scale"], v["shift"]) @ w["into"].T).split(INNER, -1)
    u, inputs = conv(u, v["taps"], v["tap_bias"], states[0])
    B, C, dt = (u @ w["mix"].T).split([STATES, STATES, INNER], -1)
    y, state = scan(u, dt, -v["log_a"].exp(), B, C, v["skip"], z, v["dt_bias"], states[1])
    return x + y @ w["out"].T, (inputs, state)


def head(x, table, norm=layer_normalization):
    return norm(x) @ table.T


def loss_of(tokens, table, stages, operators=OPERATORS):
    """Mean cross entropy of each token's successor; stages: (matrices, vectors) of each."""
    x = F.embedding(tokens[:, :-1], table)
    for w, v in stages:
        x, _ = stage(x, w, v, operators=operators)
    logits = head(x, table, operators[0]).to(torch.promote_types(x.dtype, torch.float32))
    return F.cross_entropy(logits.flatten(0, 1), tokens[:, 1:].flatten())


def first_weights(gen):
    """(table, [(matrices, vectors), ..]) as FP32 tensors on the CPU."""
    def matrix(shape):
        return torch.randn(shape, generator=gen) * shape[1] ** -0.5

    stages = []
    for _ in range(STAGES):
        step = torch.exp(torch.empty(INNER).uniform_(math.log(0.001), math.log(0.1), generator=gen))
        v = dict(scale=torch.ones(WIDTH), shift=torch.zeros(WIDTH), taps=torch.randn(INNER, TAPS, generator=gen) * TAPS ** -0.5,
                 tap_bias=torch.zeros(INNER), log_a=torch.arange(1.0, STATES + 1).log().expand(INNER, -1).clone(),
                 skip=torch.ones(INNER), dt_bias=torch.log(torch.expm1(step)))
        stages.append(({name: matrix(shape) for name, shape in MATRICES.items()}, v))
    return matrix((VOCAB, WIDTH)), stages


class Trainer:
    def __init__(self, seed, device):
        table, stages = first_weights(torch.Generator().manual_seed(seed))
        matrices = [table] + [t for w, _ in stages for t in w.values()]
        vectors = [t for _, v in stages for t in v.values()]
        self.matrices, self.vectors = ([t.to(device) for t in ts] for ts in (matrices, vectors))
        self.scaler = DynamicLossScale(1024.0)
        self.optimizer = FusedAdamW([dict(params=self.matrices), dict(params=self.vectors, weight_decay=0.0)], lr=3e-3,
                                    betas=(0.9, 0.95), weight_decay=0.01, loss_scale=self.scaler,
                                    export_dtype=torch.float16, sync=True, state_bits=8, rounding_seed=seed)
        self.windows = [StageGradients([t.shape for t in ts], device) for ts in (self.matrices, self.vectors)]

    def weights(self, leaves=False):
        """(table, stages) of the FP16 copies and the FP32 vectors; leaves: to be differentiated."""
        matrices = [t.detach().requires_grad_(leaves) for t in self.optimizer.exports[:len(self.matrices)]]
        vectors = [t.detach().requires_grad_(leaves) for t in self.vectors]
        w, v = len(MATRICES), len(VECTORS)
        stages = [(dict(zip(MATRICES, matrices[1 + i * w:])), dict(zip(VECTORS, vectors[i * v:]))) for i in range(STAGES)]
        return (matrices[0], stages), matrices, vectors

    def step(self, batches):
        (table, stages), matrices, vectors = self.weights(leaves=True)
        scale, total = self.scaler.scale, 0.0
        for window in self.windows:
            window.zero_()
        for k, tokens in enumerate(batches):
            loss = loss_of(tokens, table, stages)
            total += loss.item()
            grads = torch.autograd.grad(loss * (scale / len(batches)), matrices + vectors)
            for window, part in zip(self.windows, (grads[:len(matrices)], grads[len(matrices):])):
                window.accumulate([g.contiguous() for g in part], scale, final=k == len(batches) - 1,
                                  found_inf=self.optimizer.found_inf)
        # the windows hold unscaled FP32 gradients and have tested them
        applied = self.optimizer.step(self.windows[0].views + self.windows[1].views, checked=True)
        return total / len(batches), applied

    @torch.no_grad()
    def generate(self, tokens, count):
        """tokens [1, n] continued: the prompt in one call per stage, then step by step."""
        (table, stages), _, _ = self.weights()
        states, fed, out = [(None, None)] * STAGES, tokens, []
        for _ in range(count):
            x = F.embedding(fed, table)
            for i, (w, v) in enumerate(stages):
                x, states[i] = stage(x, w, v, states[i])
            fed = head(x[:, -1:], table).argmax(-1)
            out.append(int(fed))
        return out


def text(gen, follow, batch, length):
    tokens = torch.empty(batch, length, dtype=torch.long)
    tokens[:, 0] = torch.randint(VOCAB, (batch,), generator=gen)
    for t in range(1, length):
        anything = torch.randint(VOCAB, (batch,), generator=gen)
        tokens[:, t] = torch.where(torch.rand(batch, generator=gen) < 0.9, follow[tokens[:, t - 1]], anything)
    return tokens


def main(argv=None):
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--seed", type=int, default=0)
    args = parser.parse_args(argv)
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator().manual_seed(args.seed)
    follow = torch.randperm(VOCAB, generator=gen)
    trainer, losses = Trainer(args.seed, device), []
    for step in range(args.steps):
        loss, applied = trainer.step([text(gen, follow, 4, 129).to(device) for _ in range(2)])
        losses.append(loss)
        if step % 10 == 0 or step == args.steps - 1:
            print(f"step {step}: loss {loss:.3f}{'' if applied else ' (skipped)'}", flush=True)
    prompt = text(gen, follow, 1, 20)
    written = trainer.generate(prompt.to(device), 16)
    expected = [int(prompt[0, -1])]
    right = sum(int(follow[a]) == b for a, b in zip(expected + written, written))
    print(f"continued with {written}: {right} of {len(written)} as the text goes on")
    return losses, right


if __name__ == "__main__":
    main()
