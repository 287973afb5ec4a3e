"""The feed-forward products in a row: what each call may read and write while
others run."""
from __future__ import annotations

import pytest
import torch

import pax_b200
from test_gpu_feed_forward import F16, F32, I8, back_inputs, codes, gen, padded, randn, shifted, weights  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [65, 100, 300, 512])
def test_more_than_64_tokens_load_no_weights_early(gen, M):
    """w_const and b_const let up to 64 tokens start on the weights before the previous kernel ends; more of them wait, on
    whichever kernel they run.  Here that kernel writes the weights."""
    D, F = 4096, 1024
    P, R = randn(gen, D, 64), randn(gen, 64, F, scale=0.002)
    W, Wu, X = randn(gen, D, F), randn(gen, D, F, scale=0.02), randn(gen, M, D)
    A, V, s = codes(gen, M, D), randn(gen, F, D), torch.ones(D, device=gen.device)
    pax_b200.gemm(P, R, out=W)
    Q, _ = pax_b200.quantize_rows(V)
    aligned, odd = randn(gen, M, F), shifted(randn(gen, M, F))  # an odd base keeps the product off the tiles
    want = pax_b200.glu(X, W, Wu, out=torch.empty_like(aligned)), pax_b200.glu(X, W, Wu, out=shifted(aligned)), \
        pax_b200.gemm_i8(A, Q, s[:M], s[:F], out_dtype=F32)
    for _ in range(10):
        for out, ref in ((aligned, want[0]), (odd, want[1])):
            W.zero_()
            pax_b200.gemm(P, R, out=W)
            assert torch.equal(pax_b200.glu(X, W, Wu, out=out, w_const=True), ref)
        Q.zero_()
        pax_b200.quantize_rows(V, out=Q)
        assert torch.equal(pax_b200.gemm_i8(A, Q, s[:M], s[:F], out_dtype=F32, b_const=True), want[2])


@pytest.mark.parametrize("M", [100, 300])
def test_chain_in_chunks_with_constant_weights(gen, M):
    """As a decoding chain, with more tokens than one chunk: narrow layers of long sums, which run in chunks."""
    D, F, L = 2048, 520, 5
    X = randn(gen, M, D)
    W = [(*weights(gen, D, F), *pax_b200.quantize_rows(randn(gen, D, F, scale=F ** -0.5))) for _ in range(L)]

    def chain(const):
        x = X
        for Wg, Wu, Wq, sw in W:
            Q, s = pax_b200.quantize_rows(pax_b200.glu(x, Wg, Wu, w_const=const))
            x = pax_b200.gemm_i8(Q, Wq, s, sw, b_const=const)
            x = x / x.float().std().clamp_min(1e-3).half()
        return x

    want = chain(False)
    for _ in range(20):
        assert torch.equal(chain(True), want)
