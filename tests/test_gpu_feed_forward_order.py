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


LONG = {"quantize_rows, one long row": 0, "quantize_rows, one long odd row": 1, "glu_backward, few tiles of many tokens": 2}


@pytest.mark.parametrize("before", LONG)
@pytest.mark.parametrize("after", ["glu, few tokens", "glu, tiles", "glu, split", "glu_backward", "gemm_i8, tiles", "gemm, tiles", "gemm, few rows"])
def test_waits_count_from_the_end_of_the_kernel_before(cuda, before, after):
    """A kernel of several milliseconds that leaves most of the GPU free, so that the next one is resident long before its
    inputs are ready: with a limit of half a millisecond none of its waits may run out."""
    g = torch.Generator(device=cuda)
    g.manual_seed(5)
    kind = LONG[before]
    if kind < 2:
        row = randn(g, 1, (1 << 26) + 8 - kind)
        first = lambda: pax_b200.quantize_rows(row)  # noqa: E731
    else:
        tall = [randn(g, 1 << 21, 8) for _ in range(4)]
        small = [randn(g, 8, 8) for _ in range(2)]
        first = lambda: pax_b200.glu_backward(tall[0], tall[1], *small, *tall[2:], need_dX=False)  # noqa: E731
    M, D, F = {"glu, few tokens": (16, 1024, 512), "glu, tiles": (512, 128, 512), "glu, split": (256, 2048, 128)}.get(after, (512, 128, 512))
    X, Wg, Wu, G, U, dH = randn(g, M, D), randn(g, D, F), randn(g, D, F), randn(g, M, F), randn(g, M, F), randn(g, M, F)
    A, B, sa, sb = codes(g, M, D), codes(g, F, D), torch.ones(M, device=cuda), torch.ones(F, device=cuda)
    second = {"glu": lambda: pax_b200.glu(X, Wg, Wu), "glu_backward": lambda: pax_b200.glu_backward(dH, X, Wg, Wu, G, U)[0],
              "gemm_i8": lambda: pax_b200.gemm_i8(A, B, sa, sb),
              "gemm": lambda: pax_b200.gemm(X if "tiles" in after else X[:4], Wg)}[after.split(",")[0]]
    first()
    want = second()
    torch.cuda.synchronize()
    lib = pax_b200.lib
    assert pax_b200.device_error() == pax_b200.Status.OK
    assert lib.pax_selftest_set_wait_limit(500_000) == 0
    try:
        for _ in range(2):
            first()
            got = second()
            torch.cuda.synchronize()
            assert pax_b200.device_error() == pax_b200.Status.OK
            assert torch.equal(got, want)
    finally:
        assert lib.pax_selftest_set_wait_limit(0) == 0


@pytest.mark.parametrize("call", ["glu", "glu_backward", "quantize_rows", "gemm_i8"])
def test_inputs_freed_after_a_call_on_another_stream_are_not_reused_under_it(gen, call):
    """torch's allocator hands memory that the caller frees to the next tensor of the current stream at once, unless it knows
    that another stream still reads it."""
    M, D, F = 512, 256, 512
    make = {"glu": lambda: [randn(gen, M, D), *weights(gen, D, F)], "glu_backward": lambda: [t.clone() for t in back_inputs(gen, M, D, F)],
            "quantize_rows": lambda: [randn(gen, M, D)],
            "gemm_i8": lambda: [codes(gen, M, D), codes(gen, F, D), torch.ones(M, device=gen.device), torch.ones(F, device=gen.device)]}[call]
    getattr(pax_b200, call)(*make())
    s = torch.cuda.Stream()
    a = make()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(200_000_000)  # about 0.1 s
    out = getattr(pax_b200, call)(*a, stream=s)
    sizes, was = [(t.numel(), t.dtype) for t in a], {t.data_ptr() for t in a}
    del a
    fresh = [torch.empty(n, device=gen.device, dtype=t) for n, t in sizes]
    busy = not s.query()
    again = was & {t.data_ptr() for t in fresh}
    torch.cuda.synchronize()
    del out
    assert busy and not again


def test_outputs_that_a_caller_gives_count_as_written(gen):
    """autograd refuses a backward pass through a saved tensor that was overwritten: it goes by the tensor's version."""
    M, D, F = 40, 64, 72
    X, (Wg, Wu) = randn(gen, M, D), weights(gen, D, F)
    new = lambda *s, dt=F16: torch.zeros(s, device=gen.device, dtype=dt)  # noqa: E731
    H, G, U = new(M, F), new(M, F), new(M, F)
    dX, dWg, dWu = new(M, D), new(D, F, dt=F32), new(D, F, dt=F32)
    Q, s, C = new(M, D, dt=I8), new(M, dt=F32), new(M, F)
    B, sb = codes(gen, F, D), torch.ones(F, device=gen.device)
    saved = G.float().requires_grad_(True)
    for given, call in (((H, G, U), lambda: pax_b200.glu(X, Wg, Wu, out=H, G=G, U=U)),
                        ((G, U, dX, dWg, dWu), lambda: pax_b200.glu_backward(H, X, Wg, Wu, G, U, dG=G, dU=U, dX=dX, dWg=dWg, dWu=dWu, accumulate=True)),
                        ((Q, s), lambda: pax_b200.quantize_rows(X, out=Q, scale=s)), ((C,), lambda: pax_b200.gemm_i8(Q, B, s, sb, out=C))):
        was, inputs = [t._version for t in given], [t._version for t in (X, Wg, Wu, B, sb)]
        call()
        assert all(t._version > v for t, v in zip(given, was))
        assert [t._version for t in (X, Wg, Wu, B, sb)] == inputs
    y = (saved * G.float() * G.float()).sum()
    y2 = (torch.nn.functional.silu(saved.half()) * G).sum()
    pax_b200.glu(X, Wg, Wu, out=H, G=G, U=U)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y2.backward()
    y.backward()
    with torch.inference_mode():
        T = new(M, F)
        pax_b200.glu(X, Wg, Wu, out=T)
    assert torch.equal(pax_b200.glu(X, Wg, Wu, out=T), H)  # tensors without a version


@pytest.mark.parametrize("M", [7, 300])
def test_another_stream_inside_a_capture(gen, M):
    """A capture that forks to a second stream and joins it: the inputs and outputs of calls there are recorded for it."""
    D, F = 264, 520
    X, (Wg, Wu) = randn(gen, M, D), weights(gen, D, F)
    want = pax_b200.glu(X, Wg, Wu, save=True)
    grads = pax_b200.glu_backward(want[0], X, Wg, Wu, want[1], want[2])
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        a = X.clone()
        side.wait_stream(torch.cuda.current_stream())
        H, G, U = pax_b200.glu(a, Wg, Wu, save=True, stream=side)
        got = pax_b200.glu_backward(H, a, Wg, Wu, G, U, stream=side)
        del a
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for t, w in zip((H, G, U, *got), (*want, *grads)):
        assert torch.equal(t, w)
