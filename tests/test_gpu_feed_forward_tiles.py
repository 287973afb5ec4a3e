"""Feed-forward products through every kernel that takes them, the widest
tiles and several rounds of tiles included: sums of whole numbers, every bit of
which is known, and random values against the 64-bit forms by their 2-norm.

Whole numbers: every partial sum stays below 2^24, so that an fp32 sum is exact
in any order, and a result is the exact sum rounded once to its type.  A
product left out, or a partial sum rounded to fewer bits, shows.

2-norm: one rounding to fp16 is uniform within 2^-11 of a value's leading power
of two, 2^-11 / sqrt 3 of the norm at most; 5 % are allowed for what else
differs (fp32 sums and the gate are good to some 1e-6) and for chance, small
with 10^5 values or more."""
from __future__ import annotations

import pytest
import torch

import pax_b200
from _feed_forward import ACTS, glu, glu_grad
from test_feed_forward_items import items
from test_gpu_feed_forward import F16, F32, back_inputs, codes, gen, padded, randn, weights  # noqa: F401
from test_gpu_feed_forward_range import ints

pytestmark = pytest.mark.gpu
ROUNDED = 1.05 * 2.0 ** -11 / 3 ** 0.5


def off(got, ref):
    return ((got.double() - ref).norm() / ref.norm()).item()


def pairs():
    return torch.cuda.get_device_properties(0).multi_processor_count // 2


# few tokens; one tile to several pairs; chunks; narrow tiles, in pieces and in several rounds; any layout
GLU_SHAPES = [(1, 4096, 1032), (17, 4096, 520), (64, 2056, 4104), (300, 4096, 136), (512, 4096, 1024), (100, 4096, 264),
              (1300, 520, 9480), (2000, 264, 4104), (70, 1001, 333)]
# 512-column tiles: less than a round, and several rounds with ragged edges
WIDE_GLU = [(777, 1544, 4104), (2100, 4096, 9000), (1922, 2864, 6024)]


@pytest.mark.parametrize("shape", GLU_SHAPES + WIDE_GLU)
def test_glu_sums_are_exact(gen, shape):
    M, D, F = shape
    X, Wg, Wu = ints(gen, 2, M, D), ints(gen, 100, D, F), ints(gen, 100, D, F)
    _, G, U = pax_b200.glu(X, Wg, Wu, save=True)
    for got, w in ((G, Wg), (U, Wu)):
        assert torch.equal(got, (X.double() @ w.double()).half())


@pytest.mark.parametrize("shape", WIDE_GLU)
@pytest.mark.parametrize("name", ACTS)
def test_glu_in_wide_tiles(gen, shape, name):
    M, D, F = shape
    width, work = items(0, M, D, F, pairs())
    assert width == 2 and (M < 1000 or len(work) > 2 * pairs())
    X, (Wg, Wu) = randn(gen, M, D), weights(gen, D, F)
    ref = glu(X, Wg, Wu, name)
    saved = pax_b200.glu(X, Wg, Wu, activation=name, save=True)
    for got, what in zip(saved, "HGU"):
        v, bound = ref[what]
        assert off(got, v) <= ROUNDED, what
        assert not ((got.double() - v).abs() > bound).any(), what
    assert torch.equal(pax_b200.glu(X, Wg, Wu, activation=name), saved[0])
    wide = torch.full((M + 1, F + 24), 7.0, device=gen.device, dtype=F16)
    pax_b200.glu(X, Wg, Wu, activation=name, out=wide[:M, :F])
    assert torch.equal(wide[:M, :F], saved[0]) and (wide[:, F:] == 7).all() and (wide[M] == 7).all()


BACK_SHAPES = [(17, 520, 4096), (130, 768, 2048), (600, 264, 2056), (2500, 136, 264), (700, 1024, 2816), (1300, 520, 2568),
               (1031, 1288, 2824), (90, 65, 130)]
WIDE_BACK = [(2051, 2056, 5480), (2300, 3000, 4104), (1500, 4096, 4096)]


@pytest.mark.parametrize("shape", BACK_SHAPES + WIDE_BACK)
@pytest.mark.parametrize("dw", [F16, F32])
def test_glu_backward_sums_are_exact(gen, shape, dw):
    """Exact GeLU at 8: Phi is 1 and the density 5e-15, so that dG = dH U and dU = 8 dH."""
    M, D, F = shape
    X, Wg, Wu, U, dH = ints(gen, 3, M, D), ints(gen, 4, D, F), ints(gen, 4, D, F), ints(gen, 20, M, F), ints(gen, 3, M, F)
    G = torch.full_like(U, 8.0)
    dG, dU = (dH * U).double(), 8 * dH.double()
    want = dG @ Wg.double().T + dU @ Wu.double().T, X.double().T @ dG, X.double().T @ dU
    got = pax_b200.glu_backward(dH, X, Wg, Wu, G, U, activation="gelu_erf", dW_dtype=dw)
    assert torch.equal(got[0], want[0].half())
    assert torch.equal(got[1], want[1].to(dw)) and torch.equal(got[2], want[2].to(dw))
    base = [ints(gen, 1000, D, F, dtype=F32) for _ in range(2)]
    _, *acc = pax_b200.glu_backward(dH, X, Wg, Wu, G, U, activation="gelu_erf", dWg=base[0].clone(), dWu=base[1].clone(), accumulate=True)
    for a, b, w in zip(acc, base, want[1:]):
        assert torch.equal(a.double(), b.double() + w)


# narrow tiles in more than one round, whose pairs go from the input gradient's to the weight gradients', and wide ones
@pytest.mark.parametrize("shape,width", [((1320, 1568, 688), 1), ((2400, 1488, 1960), 1), ((4096, 1032, 6152), 1),
                                         *((s, 2) for s in WIDE_BACK)])
@pytest.mark.parametrize("dw", [F16, F32])
def test_glu_backward_in_many_tiles(gen, shape, width, dw):
    M, D, F = shape
    got_width, work = items(1, M, D, F, pairs())
    mixed = set(work[work[:, 1] == 0][:, 0]) & set(work[work[:, 1] == 1][:, 0])
    assert got_width == width and len(work) > pairs() and mixed  # pairs with tiles of both kinds
    name = ACTS[(M + F) % 3]
    a = back_inputs(gen, M, D, F)
    ref = glu_grad(*a, name, dw_f16=dw == F16)
    full = pax_b200.glu_backward(*a, activation=name, dW_dtype=dw)
    for got, what in zip(full, ("dX", "dWg", "dWu")):
        v, bound = ref[what]
        # dG and dU are rounded to fp16 on the way; a result in fp16 once more
        assert off(got, v) <= ROUNDED * (1.0 if got.dtype == F32 else 2.0 ** 0.5), what
        assert not ((got.double() - v).abs() > bound).any(), what
    only_x = pax_b200.glu_backward(*a, activation=name, need_dW=False)
    only_w = pax_b200.glu_backward(*a, activation=name, need_dX=False, dW_dtype=dw)
    assert torch.equal(only_x[0], full[0]) and torch.equal(only_w[1], full[1]) and torch.equal(only_w[2], full[2])


@pytest.mark.parametrize("shape", [(24, 11264, 4096), (1235, 4099, 2064), (2300, 3000, 1040)])
def test_gemm_i8_rounds_once(gen, shape):
    """Scales that are powers of two: the exact sum, scaled, rounded to fp32 and then to fp16 where asked."""
    M, N, K = shape
    A, B = codes(gen, M, K), codes(gen, N, K)
    sa, sb = (2.0 ** -torch.randint(4, 10, (n,), generator=gen, device=gen.device).float() for n in (M, N))
    C = (A.double() @ B.double().T).float() * sa[:, None] * sb[None, :]
    for t in (F32, F16):
        assert torch.equal(pax_b200.gemm_i8(A, B, sa, sb, out_dtype=t), C.to(t))
