"""Feed-forward products at the ends of their range: the longest batches,
every magnitude of the gate, values beyond fp16, and sums whose every bit is
known."""
from __future__ import annotations

import pytest
import torch

import pax_b200
from _feed_forward import ACTS

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


# ------------------------------------------------------------------ the gate's whole range
def gate_parts(x, name):
    """64-bit act(x), act'(x), the sum of the magnitudes of act's two terms, and the bound on the relative error of each term.

    sigmoid(y) = 1 / (1 + exp(-y)): y takes up to 5 roundings of 2^-24, the exponential's base-2 argument 1 more, which the
    exponential turns into up to 6 |y| of them; the exponential, the sum, the reciprocal and the products are good to 2 or 3
    each, below 16 in all.  erfc: 3 roundings of its argument x^2 / 2, below 24 for polynomial and products.  Below
    y = -104 the true value is under 2^-149."""
    if name == "gelu_erf":
        cdf, phi = 0.5 * torch.special.erfc(-x / 2 ** 0.5), torch.exp(-0.5 * x * x) / (2 * torch.pi) ** 0.5
        a, d1, d2, y = x * cdf, cdf, x * phi, 0.5 * x * x
    else:
        k = 2 * (2 / torch.pi) ** 0.5
        y = x if name == "silu" else k * (x + 0.044715 * x ** 3)
        dy = 1.0 if name == "silu" else k * (1 + 3 * 0.044715 * x * x)
        p, q = torch.sigmoid(y), torch.sigmoid(-y)
        a, d1, d2 = x * p, p, x * p * q * dy
    return a, d1 + d2, d1.abs() + d2.abs(), 2.0 ** -24 * (32 + 8 * y.abs().clamp_max(104.0))


def whole_range(gen, n):
    """n fp16 values of both signs: every magnitude from 2^-24 to 65504, and half of them in the steep part and the tails."""
    wide = torch.logspace(-7.2, 4.816, n // 4, device=gen.device, dtype=torch.float64).clamp_max(65504.0)
    near = torch.linspace(0, 14, n // 2 - n // 4, device=gen.device, dtype=torch.float64)
    m = torch.cat([wide, near]).half()
    return torch.cat([m, -m])[torch.randperm(n, generator=gen, device=gen.device)]


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("up", [1.0, 1000.0])
@pytest.mark.parametrize("M,pad", [(5, 0), (200, 0), (1200, 0), (60, 1)])
def test_glu_keeps_the_gates_tails(gen, name, up, M, pad):
    """One term a sum, so that G and U are exact and H is off by the gate's own relative error and one rounding."""
    D, F = 64, 1024 + pad
    X = torch.eye(D, device=gen.device, dtype=F16).repeat(M // D + 1, 1)[:M].contiguous()
    Wg, Wu = whole_range(gen, D * 1024).view(D, 1024)[:, torch.arange(F, device=gen.device) % 1024].contiguous(), randn(gen, D, F, scale=up)
    H, G, U = pax_b200.glu(X, Wg, Wu, activation=name, save=True)
    g, u = (X.double() @ w.double() for w in (Wg, Wu))
    assert torch.equal(G.double(), g) and torch.equal(U.double(), u)
    a, _, _, rel = gate_parts(g, name)
    h = a * u
    fits = h.abs() < 65000  # beyond fp16 a right result is an infinity
    t = (rel + 2.0 ** -24) * h.abs()
    tol = t + 2.0 ** -11 * (h.abs() + t) + 2.0 ** -25
    bad = ((H.double() - h).abs() > tol) & fits
    assert not bad.any(), (int(bad.sum()), g[bad][0].item(), H[bad][0].item(), h[bad][0].item())


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("size", [1.0, 1000.0])
@pytest.mark.parametrize("shape", [(64, 1024), (63, 1025)])
def test_glu_backward_keeps_the_gates_tails(gen, name, size, shape):
    """dG and dU over every magnitude of G: each off by its terms' relative error and one rounding."""
    M, F = shape
    G, U, dH = whole_range(gen, 65536).repeat(2)[: M * F].view(M, F).contiguous(), randn(gen, M, F), randn(gen, M, F, scale=size)
    X, W = torch.zeros(M, 8, device=gen.device, dtype=F16), torch.zeros(8, F, device=gen.device, dtype=F16)
    dG, dU = torch.empty_like(G), torch.empty_like(G)
    pax_b200.glu_backward(dH, X, W, W.clone(), G, U, activation=name, need_dX=False, need_dW=False, dG=dG, dU=dU)
    g, u, dh = G.double(), U.double(), dH.double()
    a, d, terms, rel = gate_parts(g, name)
    for what, got, want, t in (("dG", dG, dh * u * d, (dh * u).abs() * terms), ("dU", dU, dh * a, (dh * a).abs())):
        t = (rel + 2.0 ** -23) * t
        tol = t + 2.0 ** -11 * (want.abs() + t) + 2.0 ** -25
        bad = ((got.double() - want).abs() > tol) & (want.abs() < 65000)
        assert not bad.any(), (what, int(bad.sum()), g[bad][0].item(), got[bad][0].item(), want[bad][0].item())


# ------------------------------------------------------------------ beyond fp16
@pytest.mark.parametrize("M,D,F", [(5, 64, 72), (40, 264, 136), (300, 136, 520), (50, 65, 77)])
def test_what_is_not_finite_stays_in_its_token(gen, M, D, F):
    """A NaN or an infinity in a token's dH, U or X reaches that token's dX, or none, and the weight gradients; other tokens keep
    their bits."""
    a = [randn(gen, M, F), randn(gen, M, D), randn(gen, D, F, scale=0.1), randn(gen, D, F, scale=0.1), randn(gen, M, F), randn(gen, M, F)]
    clean = pax_b200.glu_backward(*a)
    for i in (0, 5):
        for v in (float("nan"), float("inf")):
            b = [t.clone() for t in a]
            b[i][2, 3] = v
            dX, dWg, dWu = pax_b200.glu_backward(*b)
            rest = [m for m in range(M) if m != 2]
            assert torch.equal(dX[rest], clean[0][rest]) and not dX[2].isfinite().any()
            cols = [f for f in range(F) if f != 3]
            assert torch.equal(dWg[:, cols], clean[1][:, cols]) and not dWg[:, 3].isfinite().any()
            assert torch.equal(dWu[:, cols], clean[2][:, cols]) and (i == 5 or not dWu[:, 3].isfinite().any())
    b = [t.clone() for t in a]
    b[1][2, 3] = float("nan")
    dX, dWg, _ = pax_b200.glu_backward(*b)
    rest = [d for d in range(D) if d != 3]
    assert torch.equal(dX, clean[0]) and dWg[3].isnan().all() and torch.equal(dWg[rest], clean[1][rest])


@pytest.mark.parametrize("M", [9, 200])
def test_products_of_the_gradient_beyond_fp16(gen, M):
    """dG and dU are fp16, as pax.h says: what exceeds its range becomes an infinity, what is at most 2^-25 zero."""
    F, D = 136, 64
    G, one = torch.full((M, F), 40.0, device=gen.device, dtype=F16), torch.ones(M, F, device=gen.device, dtype=F16)
    X, W = ints(gen, 1, M, D), ints(gen, 1, D, F)
    dG, dU = torch.empty_like(G), torch.empty_like(G)
    call = lambda dH, U: pax_b200.glu_backward(dH, X, W, W.clone(), G, U, dG=dG, dU=dU)  # noqa: E731  silu(40) = 40, silu' = 1
    dX, dWg, dWu = call(512 * one, 200 * one)
    assert (dG == float("inf")).all() and (dU == 512 * 40).all()
    assert not dX[W.float().abs().sum(1).gt(0).expand(M, D)].isfinite().any() and not dWg[X.float().abs().sum(0) > 0].isfinite().any()
    assert torch.equal(dWu, (X.double().T @ dU.double()).half())
    call(-512 * one, 200 * one)
    assert (dG == float("-inf")).all()
    tiny = 2.0 ** -13 * one
    call(tiny, 2.0 ** -12 * one)  # dG = 2^-25, half of the smallest fp16: to even
    assert (dG == 0).all() and (dU == 40 * 2.0 ** -13).all()
    call(tiny, 1.5 * 2.0 ** -12 * one)
    assert (dG == 2.0 ** -24).all()


@pytest.mark.parametrize("M", [9, 200])
def test_gate_products_beyond_fp16(gen, M):
    """H comes from the unrounded products: finite where G is kept as an infinity."""
    D, F = 64, 136
    X = torch.full((M, D), 64.0, device=gen.device, dtype=F16)
    Wg, Wu = torch.full((D, F), -32.0, device=gen.device, dtype=F16), torch.full((D, F), 2.0 ** -14, device=gen.device, dtype=F16)
    Wg[:, ::2] = 32.0
    H, G, U = pax_b200.glu(X, Wg, Wu, save=True)  # g = -+131072, u = 1/4
    assert (G[:, ::2] == float("inf")).all() and (G[:, 1::2] == float("-inf")).all() and (U == 0.25).all()
    assert (H[:, ::2] == 32768).all() and (H[:, 1::2] == 0).all()
