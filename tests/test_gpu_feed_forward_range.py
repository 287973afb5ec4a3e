"""Feed-forward products at the ends of their range: the longest batches,
every magnitude of the gate, values beyond fp16, and sums whose every bit is
known."""
from __future__ import annotations

import pytest
import torch

import pax_b200

pytestmark = pytest.mark.gpu
F16, F32, I8 = torch.float16, torch.float32, torch.int8


@pytest.fixture
def gen(cuda):
    g = torch.Generator(device=cuda)
    g.manual_seed(4321)
    return g


def randn(g, *shape, scale=1.0, dtype=F16):
    return (torch.randn(shape, generator=g, device=g.device) * scale).to(dtype)


def ints(g, top, *shape, dtype=F16):
    """Whole numbers from -top to top."""
    return torch.randint(-top, top + 1, shape, generator=g, device=g.device, dtype=torch.int32).to(dtype)


@pytest.mark.parametrize("shape", [(64 * 65535 + 1, 8, 8), (64 * 65535 + 1, 64, 64), (1 << 23, 64, 64), (64 * 65535 + 1, 72, 136)])
@pytest.mark.parametrize("parts", ["both", "dX"])
def test_glu_backward_of_more_tokens_than_chunks_of_a_grid(gen, shape, parts):
    """G = 0 makes silu' 1/2 and silu 0, so that every gradient is a whole number: at most 2^23 tokens of +-1 in dWg, 72 in dX."""
    M, D, F = shape
    X, Wg, Wu = ints(gen, 1, M, D), ints(gen, 1, D, F), ints(gen, 1, D, F)
    G, U, dH = torch.zeros(M, F, device=gen.device, dtype=F16), torch.ones(M, F, device=gen.device, dtype=F16), 2 * ints(gen, 1, M, F)
    base = [torch.ones(D, F, device=gen.device) for _ in range(2)]
    kw = dict(dWg=base[0], dWu=base[1], accumulate=True) if parts == "both" else dict(need_dW=False)
    dX, dWg, dWu = pax_b200.glu_backward(dH, X, Wg, Wu, G, U, **kw)
    assert torch.equal(dX, ((dH.float() / 2) @ Wg.float().T).half())  # whole numbers below 2^11: exact in any order
    if parts == "both":
        assert (dWu == 1).all()
        want = sum(x.double().T @ h.double() for x, h in zip(X.split(1 << 20), (dH / 2).split(1 << 20)))
        assert torch.equal(dWg.double(), want + 1)
    assert pax_b200.device_error() == pax_b200.Status.OK
