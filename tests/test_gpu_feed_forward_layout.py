"""Layouts of the feed-forward products' operands: single rows."""
from __future__ import annotations

import pytest
import torch

import pax_b200
from _feed_forward import close, gemm_i8, glu, glu_grad, quantize
from test_gpu_feed_forward import F16, codes, gen, padded, randn  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,F", [(1001, 2000), (4093, 4096), (131, 72)])
def test_one_token_of_an_odd_width_runs_as_one_of_two_does(gen, D, F):
    """A single row has no pitch: beside weights in padded rows, the same kernel and the same bits as in a batch of two."""
    X = padded(randn(gen, 2, D), 4096 + 8 - D)
    Wg, Wu = (padded(w, 8) for w in (randn(gen, D, F, scale=D ** -0.5), randn(gen, D, F, scale=D ** -0.5)))
    two = pax_b200.glu(X, Wg, Wu, save=True)
    for one in (X[:1], X[:1].clone()):
        for a, b in zip(two, pax_b200.glu(one, Wg, Wu, save=True)):
            assert torch.equal(a[:1], b)
    # the input gradient: one row of dG and dU of an odd length
    back = [randn(gen, 2, D), Wg.new_zeros(2, F), randn(gen, 2, D), randn(gen, 2, D)]
    W = [padded(randn(gen, F, D, scale=F ** -0.5), 4096 + 8 - D) for _ in range(2)]
    kw = dict(need_dW=False)
    dH, X2, G, U = (padded(t, 4096 + 8 - t.shape[1]) for t in back)
    dG, dU = (padded(torch.zeros_like(G), 4096 + 8 - D) for _ in range(2))
    two = pax_b200.glu_backward(dH, X2, *W, G, U, dG=dG, dU=dU, **kw)[0]
    one = pax_b200.glu_backward(dH[:1].clone(), X2[:1].clone(), *W, G[:1].clone(), U[:1].clone(), **kw)[0]
    assert torch.equal(two[:1], one)
    A, B = padded(codes(gen, 2, D), 4112 - D, 55), padded(codes(gen, F, D), 4112 - D, 55)
    sa, sb = torch.rand(2, generator=gen, device=gen.device), torch.rand(F, generator=gen, device=gen.device)
    two = pax_b200.gemm_i8(A, B, sa, sb)
    assert torch.equal(two[:1], pax_b200.gemm_i8(A[:1].clone(), B, sa[:1].clone(), sb))


def test_single_rows_end_where_they_do(gen):
    """What lies behind a single row's end is NaN, 55 or 7: never read into a sum, never written."""
    for D, F in ((133, 264), (70, 137), (1001, 72)):
        row = padded(randn(gen, 1, D), 27)
        Wg, Wu = (padded(randn(gen, D, F, scale=0.1), 280 - F) for _ in range(2))
        buf = [torch.full((1, F + 23), 7.0, device=gen.device, dtype=F16) for _ in range(3)]
        got = pax_b200.glu(row, Wg, Wu, out=buf[0][:, :F], G=buf[1][:, :F], U=buf[2][:, :F])
        for what, t, b in zip("HGU", got, buf):
            close(t, glu(row, Wg, Wu, "silu")[what], what)
            assert (b[:, F:] == 7).all()
        q = torch.full((1, D + 9), 99, device=gen.device, dtype=torch.int8)
        Q, s = pax_b200.quantize_rows(row, out=q[:, :D])
        assert torch.equal(Q, quantize(row)[0]) and (q[:, D:] == 99).all()
        A, B = padded(codes(gen, 1, D), 19, 55), padded(codes(gen, F, D), 1040 - D, 55)
        sa, sb = torch.rand(1, generator=gen, device=gen.device), torch.rand(F, generator=gen, device=gen.device)
        for N in (F, 1):  # one row of tokens, and one of weights too
            c = torch.full((1, F + 5), 7.0, device=gen.device)
            close(pax_b200.gemm_i8(A, B[:N], sa, sb[:N], out=c[:, :N]), gemm_i8(A, B[:N], sa, sb[:N], None, False), "C")
            assert (c[:, N:] == 7).all()


def test_one_feature_and_one_weight_row(gen):
    """D = 1: the weights are single rows; the outer product is exact but for its roundings."""
    M, F = 70, 137
    X, Wg, Wu = randn(gen, M, 1), randn(gen, 1, F), randn(gen, 1, F)
    for what, t in zip("HGU", pax_b200.glu(X, Wg, Wu, save=True)):
        close(t, glu(X, Wg, Wu, "silu")[what], what)
    dX, dWg, dWu = pax_b200.glu_backward(randn(gen, M, F), X, Wg, Wu, randn(gen, M, F), randn(gen, M, F))
    assert dX.shape == (M, 1) and dWg.shape == dWu.shape == (1, F) and dWg.isfinite().all()


@pytest.mark.parametrize("M", [1, 70, 600])
@pytest.mark.parametrize("F", [136, 137])
def test_weight_gradients_of_a_single_feature(gen, M, F):
    """Weight gradients of one row, from tokens in padded rows and as a column of their own; what lies around stays."""
    X, Wg, Wu, G, U, dH = randn(gen, M, 1), randn(gen, 1, F), randn(gen, 1, F), randn(gen, M, F), randn(gen, M, F), randn(gen, M, F)
    ref = glu_grad(dH, X, Wg, Wu, G, U, "silu", dw_f16=False)
    for x in (X, padded(X, 7)):
        buf = [torch.full((3, F + 7), 7.0, device=gen.device) for _ in range(2)]
        got = pax_b200.glu_backward(dH, x, Wg, Wu, G, U, dWg=buf[0][1:2, :F], dWu=buf[1][1:2, :F])
        for t, what in zip(got, ("dX", "dWg", "dWu")):
            close(t, ref[what], what)
        for b in buf:
            assert (b[0] == 7).all() and (b[2] == 7).all() and (b[1, F:] == 7).all()
