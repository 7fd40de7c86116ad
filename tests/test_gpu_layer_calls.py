"""Calls of the layer operators as users make them: on another stream, under autograd, at the ends
of a type's range, and with what they refuse."""
import pytest
import torch

from morph_amd.ffn import gated_ffn, gated_ffn_backward, gated_ffn_forward

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def normal(gen, *shape, scale=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen) * scale + mean).to(dtype)


@pytest.mark.parametrize("keep", ["full", "fp8"])
def test_ffn_views_written_on_the_calls_stream(keep):
    """Weights that are no rows (transposed, expanded), written on the call's stream behind other work:
    the copies that the kernels read are made in that stream's order, not in the current one's."""
    gen = torch.Generator().manual_seed(21)
    rows, d, ff, dtype = 130, 96, 160, torch.bfloat16
    x, dy = (normal(gen, rows, d, dtype=dtype).to(DEV) for _ in range(2))
    sources = [normal(gen, d, ff, scale=d ** -.5, dtype=dtype).to(DEV), normal(gen, 1, d, scale=d ** -.5, dtype=dtype).to(DEV),
               normal(gen, ff, d, scale=ff ** -.5, dtype=dtype).to(DEV)]

    def views(gate, up, down):
        return gate.t(), up.expand(ff, d), down.t()
    copies = [w.contiguous() for w in views(*sources)]
    y, saved = gated_ffn_forward(x, *copies, keep=keep)
    grads = gated_ffn_backward(dy, saved, *copies)
    work = torch.randn(4096, 4096, device=DEV)
    side = torch.cuda.Stream()
    for _ in range(3):
        written = [torch.zeros_like(s) for s in sources]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(4):
                work @ work
            for w, s in zip(written, sources):
                w.copy_(s)
        got, kept = gated_ffn_forward(x, *views(*written), keep=keep, stream=side)
        served = gated_ffn(x, *views(*written), stream=side)
        with torch.cuda.stream(side):  # written anew between the calls
            for w in written:
                w.zero_()
            for _ in range(4):
                work @ work
            for w, s in zip(written, sources):
                w.copy_(s)
        back = gated_ffn_backward(dy, kept, *views(*written), stream=side)
        side.synchronize()
        assert torch.equal(got, y) and torch.equal(served, gated_ffn(x, *copies))
        assert all(torch.equal(a, b) for a, b in zip(back, grads))
