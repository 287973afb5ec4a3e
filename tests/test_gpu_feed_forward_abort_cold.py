"""The kernels that share a tile's sum (few tokens, few tiles) give up too,
where their loads come from memory: with the caches flushed a load takes longer
than the shortened limit and the hardware's own suspension together."""
from __future__ import annotations

import pytest
import torch

import pax_b200
from _feed_forward import close, gemm_i8, glu, glu_grad
from test_gpu_feed_forward_abort import abort_run, codes, gen, randn  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def cold_run(cuda):
    flush = torch.empty(1 << 28, device=cuda, dtype=torch.uint8)  # 256 MB, twice the L2

    def run(fn):
        gave_up = 0
        for _ in range(40):
            flush.zero_()
            torch.cuda.synchronize()
            status = abort_run(fn)
            assert status in (pax_b200.Status.TIMEOUT, pax_b200.Status.OK)
            assert pax_b200.device_error() == pax_b200.Status.OK
            gave_up += status == pax_b200.Status.TIMEOUT
            if gave_up == 4:
                return
        # 40 of 40 gave up when this was written; of the weight gradients' split 20
        assert gave_up > 0

    return run


# few tokens, in one chunk and in several; one tile to several pairs, one row block and two
@pytest.mark.parametrize("M,F", [(16, 2048), (64, 11264), (100, 264), (300, 264), (512, 1024)])
def test_glu_gives_up_and_recovers(gen, cold_run, M, F):
    X, Wg, Wu = randn(gen, M, 8192), randn(gen, 8192, F, scale=0.01), randn(gen, 8192, F, scale=0.01)
    cold_run(lambda: pax_b200.glu(X, Wg, Wu, save=True))
    for got, what in zip(pax_b200.glu(X, Wg, Wu, save=True), "HGU"):
        close(got, glu(X, Wg, Wu, "silu")[what], what)
    assert pax_b200.device_error() == pax_b200.Status.OK


@pytest.mark.parametrize("M,N", [(16, 4099), (64, 16384), (1000, 256)])
def test_gemm_i8_gives_up_and_recovers(gen, cold_run, M, N):
    K = 32768
    A, B = codes(gen, M, K), codes(gen, N, K)
    sa, sb = torch.rand(M, generator=gen, device=gen.device), torch.rand(N, generator=gen, device=gen.device)
    cold_run(lambda: pax_b200.gemm_i8(A, B, sa, sb, out_dtype=torch.float32))
    close(pax_b200.gemm_i8(A, B, sa, sb, out_dtype=torch.float32), gemm_i8(A, B, sa, sb, None, False), "C")
    assert pax_b200.device_error() == pax_b200.Status.OK


# the input gradient for few tokens and of one tile to several pairs; the weight gradients of one tile to several pairs
@pytest.mark.parametrize("M,D,F,part", [(40, 1024, 8192, "need_dW"), (700, 1024, 2816, "need_dW"), (8192, 512, 512, "need_dX")])
def test_glu_backward_gives_up_and_recovers(gen, cold_run, M, D, F, part):
    a = [randn(gen, M, F), randn(gen, M, D), randn(gen, D, F, scale=0.03), randn(gen, D, F, scale=0.03), randn(gen, M, F), randn(gen, M, F)]
    cold_run(lambda: pax_b200.glu_backward(*a, **{part: False}))
    ref = glu_grad(*a, "silu")
    for got, what in zip(pax_b200.glu_backward(*a), ("dX", "dWg", "dWu")):
        close(got, ref[what], what)
    assert pax_b200.device_error() == pax_b200.Status.OK
