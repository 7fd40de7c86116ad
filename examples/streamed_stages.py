"""A small language model trained stage by stage, as the streamed engine runs its stages.

Each stage is a gated recurrence and a gated feed-forward block.  A step's forward keeps one
boundary activation per stage in 8 bits; the backward replays the stages from the last to
the first from those boundaries (the feed-forward blocks keep their own activations in 8 bits
meanwhile), sums the FP16 gradients of the micro-batches into an FP32 window and updates the FP32 masters, which
write the FP16 weights of the next step.  Then the model continues a sequence token by token.

    python examples/streamed_stages.py [--steps 60]

The text is synthetic: each symbol is followed by another one nine times out of ten, drawn once.
"""
import argparse
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from morph_amd import DynamicLossScale, FusedAdamW  # noqa: E402
from morph_amd.activations import pack_activation, unpack_activation  # noqa: E402
from morph_amd.ffn import gated_feed_forward  # noqa: E402
from morph_amd.grads import StageGradients  # noqa: E402
from morph_amd.recurrence import gated_recurrence  # noqa: E402

VOCAB, WIDTH, HIDDEN, STAGES = 64, 128, 352, 3
SHAPES = [(3 * WIDTH, WIDTH), (WIDTH, WIDTH), (HIDDEN, WIDTH), (HIDDEN, WIDTH), (WIDTH, HIDDEN)]  # of a stage


def norm(x):
    return F.rms_norm(x, x.shape[-1:])


def stage(x, weights, state=None):
    """(x behind the stage, the recurrence's state); x: [batch, steps, WIDTH]."""
    mix, out, gate, up, down = weights
    f, v, z = (norm(x) @ mix.T).split(WIDTH, -1)
    y, state = gated_recurrence(f + 2, v, z, state)
    x = x + y @ out.T
    return x + gated_feed_forward(norm(x), gate, up, down, keep="fp8"), state


def head(x, table, targets):
    return F.cross_entropy((norm(x) @ table.T).float().flatten(0, 1), targets.flatten())


class Trainer:
    def __init__(self, seed, device):
        gen = torch.Generator().manual_seed(seed)
        shapes = [(VOCAB, WIDTH)] + STAGES * SHAPES
        masters = [torch.randn(s, generator=gen).mul_(s[1] ** -0.5).to(device) for s in shapes]
        self.scaler = DynamicLossScale(1024.0)
        self.optimizer = FusedAdamW(masters, lr=3e-3, betas=(0.9, 0.95), weight_decay=0.01,
                                    loss_scale=self.scaler, export_dtype=torch.float16, sync=True)
        self.window = StageGradients(shapes, device)

    def weights(self):
        """The embedding table and every stage's weights: the optimizer's FP16 copies."""
        table, *rest = self.optimizer.exports
        return table, [rest[i:i + len(SHAPES)] for i in range(0, len(rest), len(SHAPES))]

    def step(self, batches):
        table, stages = self.weights()
        scale, total = self.scaler.scale, 0.0
        self.window.zero_()
        for k, tokens in enumerate(batches):
            with torch.no_grad():  # forward: only the boundaries stay
                x, boundaries = F.embedding(tokens[:, :-1], table), []
                for weights in stages:
                    boundaries.append(pack_activation(x))
                    x, _ = stage(x, weights)
            leaf, table_leaf = x.requires_grad_(), table.detach().requires_grad_()
            loss = head(leaf, table_leaf, tokens[:, 1:])
            total += loss.item()
            dx, dtable = torch.autograd.grad(loss * (scale / len(batches)), (leaf, table_leaf))
            grads = []
            for weights, boundary in zip(reversed(stages), reversed(boundaries)):  # backward: replayed
                x = unpack_activation(boundary).requires_grad_()
                leaves = [w.detach().requires_grad_() for w in weights]
                dx, *dw = torch.autograd.grad(stage(x, leaves)[0], [x, *leaves], dx)
                grads = dw + grads
            # the tied table: its share as the embedding
            dtable = dtable.index_add(0, tokens[:, :-1].flatten(), dx.flatten(0, 1))
            self.window.accumulate([dtable, *(g.contiguous() for g in grads)], scale,
                                   final=k == len(batches) - 1, found_inf=self.optimizer.found_inf)
        # the window holds unscaled FP32 gradients and has tested them
        applied = self.optimizer.step(self.window.views, checked=True)
        return total / len(batches), applied

    @torch.no_grad()
    def generate(self, tokens, count):
        """tokens [1, n] continued: the prompt in one call per stage, then step by step."""
        table, stages = self.weights()
        states, fed, out = [None] * STAGES, tokens, []
        for _ in range(count):
            x = F.embedding(fed, table)
            for i, weights in enumerate(stages):
                x, states[i] = stage(x, weights, states[i])
            fed = (norm(x[:, -1:]) @ table.T).argmax(-1)
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
