"""The feed-forward kernels' waits that run out, without a fault.

With the limit of the abandonable waits shortened to a microsecond, a real
launch gives up: its issued loads land, its issued MMAs drain, TMEM is freed,
a timeout is recorded and the kernel ends.  The next call must be right.

A tile of the CTA-pair kernel keeps its epilogue waiting for tens of
microseconds, so those calls always give up.  The waits of the kernels that
share a tile's sum (few tokens, few tiles) are for one load each and mostly end
within the hardware's own suspension, before the clock is looked at: there a
call may give up or not.
"""
from __future__ import annotations

import pytest
import torch

import pax_b200
from _feed_forward import close, gemm_i8, glu, glu_grad

pytestmark = pytest.mark.gpu
F16, I8 = torch.float16, torch.int8
SHORT_NS = 1000


def abort_run(fn):
    lib = pax_b200.lib
    pax_b200.device_error()  # start from a clear error word
    assert lib.pax_selftest_set_wait_limit(SHORT_NS) == 0
    try:
        fn()
        torch.cuda.synchronize()
    finally:
        assert lib.pax_selftest_set_wait_limit(0) == 0
    return pax_b200.device_error()


def gives_up(fn, always):
    for _ in range(3):
        st = abort_run(fn)
        assert st == pax_b200.Status.TIMEOUT or (not always and st == pax_b200.Status.OK)
        assert pax_b200.device_error() == pax_b200.Status.OK


@pytest.fixture
def gen(cuda):
    g = torch.Generator(device=cuda)
    g.manual_seed(77)
    return g


def randn(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g, device=g.device) * scale).to(F16)


def codes(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, device=g.device, dtype=torch.int32).to(I8)


# 16 tokens: the few-token kernel, in clusters; 1024 x 2048: narrow tiles of
# CTA pairs; 2048 x 9472: wide ones; 300 x 264: one tile to several
# pairs.
@pytest.mark.parametrize("M,F", [(16, 2048), (1024, 2048), (2048, 9472), (300, 264)])
def test_glu_gives_up_and_recovers(gen, M, F):
    X, Wg, Wu = randn(gen, M, 8192), randn(gen, 8192, F, scale=0.01), randn(gen, 8192, F, scale=0.01)
    gives_up(lambda: pax_b200.glu(X, Wg, Wu, save=True), always=M > 1000)
    X, Wg, Wu = X[:, :192].contiguous(), Wg[:192], Wu[:192]
    close(pax_b200.glu(X, Wg, Wu), glu(X, Wg, Wu, "silu")["H"], "H")
    assert pax_b200.device_error() == pax_b200.Status.OK


@pytest.mark.parametrize("M", [40, 2048])
def test_glu_backward_gives_up_and_recovers(gen, M):
    D, F = 1024, 8192
    a = [randn(gen, M, F), randn(gen, M, D), randn(gen, D, F, scale=0.03), randn(gen, D, F, scale=0.03), randn(gen, M, F),
         randn(gen, M, F)]
    gives_up(lambda: pax_b200.glu_backward(*a), always=M > 64)
    a = [t[:200, :136].contiguous() if t.shape == (M, F) else t[:200].contiguous() if t.shape[0] == M else t[:, :136].contiguous()
         for t in a]
    for got, what in zip(pax_b200.glu_backward(*a), ("dX", "dWg", "dWu")):
        close(got, glu_grad(*a, "silu")[what], what)
    assert pax_b200.device_error() == pax_b200.Status.OK


@pytest.mark.parametrize("M", [16, 1100])
def test_gemm_i8_gives_up_and_recovers(gen, M):
    N, K = 4099, 32768
    A, B = codes(gen, M, K), codes(gen, N, K)
    sa, sb = torch.rand(M, generator=gen, device=gen.device), torch.rand(N, generator=gen, device=gen.device)
    gives_up(lambda: pax_b200.gemm_i8(A, B, sa, sb), always=M > 64)
    A, B = A[:, :272].contiguous(), B[:, :272].contiguous()
    C = pax_b200.gemm_i8(A, B, sa, sb, out_dtype=torch.float32)
    close(C, gemm_i8(A, B, sa, sb, None, False), "C")
    assert pax_b200.device_error() == pax_b200.Status.OK
