"""The feed-forward products on the GPU against their 64-bit forms."""
from __future__ import annotations

import pytest
import torch

import pax_b200
from _feed_forward import ACTS, act, close, gemm_i8, glu, glu_grad, quantize

pytestmark = pytest.mark.gpu
F16, F32, I8 = torch.float16, torch.float32, torch.int8


@pytest.fixture
def gen(cuda):
    g = torch.Generator(device=cuda)
    g.manual_seed(1234)
    return g


def randn(g, *shape, scale=1.0, dtype=F16):
    return (torch.randn(shape, generator=g, device=g.device) * scale).to(dtype)


def padded(t, extra, fill=float("nan")):
    """t as a view of a wider buffer whose other columns hold `fill`."""
    b = torch.full((t.shape[0], t.shape[1] + extra), fill, device=t.device, dtype=t.dtype)
    b[:, : t.shape[1]] = t
    return b[:, : t.shape[1]]


def shifted(t, by=1):
    """t at a base that is `by` elements past an aligned one."""
    b = torch.zeros(t.numel() + by, device=t.device, dtype=t.dtype)[by:].view(t.shape)
    b.copy_(t)
    return b


def weights(g, D, F):
    s = max(D, 1) ** -0.5
    return randn(g, D, F, scale=s), randn(g, D, F, scale=s)


# tokens x width x feed-forward width: one token, the small kernel's edges, one
# tile, ragged tiles on every side, several tiles, and layouts without 16-byte rows
GLU_SHAPES = [(1, 8, 8), (1, 2048, 1000), (2, 64, 64), (8, 128, 72), (15, 200, 136), (16, 1024, 520), (17, 72, 2056), (33, 512, 64),
              (64, 4096, 256), (65, 264, 328), (100, 1032, 96), (128, 64, 128), (129, 192, 1160), (256, 256, 128), (257, 512, 264),
              (300, 8, 136), (520, 1096, 640), (1000, 640, 1408), (300, 4096, 136), (513, 2056, 264), (700, 1544, 296),
              (1, 9, 8), (7, 64, 33), (70, 65, 130), (200, 121, 77)]


@pytest.mark.parametrize("shape", GLU_SHAPES)
@pytest.mark.parametrize("save", [False, True])
def test_glu(gen, shape, save):
    M, D, F = shape
    name = ACTS[(M + D) % 3]
    X, (Wg, Wu) = randn(gen, M, D), weights(gen, D, F)
    got = pax_b200.glu(X, Wg, Wu, activation=name, save=save)
    ref = glu(X, Wg, Wu, name)
    for what, t in zip("HGU", got if save else (got,)):
        close(t, ref[what], what)


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("M", [5, 200])
def test_glu_activations_over_their_whole_range(gen, name, M):
    """Products from -60000 to 60000, with the steep part in between."""
    D, F = 64, 256
    X, Wu = torch.eye(D, device=gen.device, dtype=F16).repeat(4, 1)[:M].contiguous(), randn(gen, D, F, scale=1e-4)
    mags = torch.logspace(-7, 4.77, D * F // 2, device=gen.device).half()
    Wg = torch.cat([mags, -mags])[torch.randperm(D * F, generator=gen, device=gen.device)].view(D, F)
    H, G, U = pax_b200.glu(X, Wg, Wu, activation=name, save=True)
    ref = glu(X, Wg, Wu, name)
    close(G, ref["G"], "G")
    # one term a sum: G and U are exact, H is the activation's value rounded once
    g, u = G.double(), U.double()
    h = act(g, name) * u
    close(H, (h, 2.0 ** -11 * h.abs() + 2.0 ** -25 + 3e-6 * g.abs().clamp_min(1e-3) * u.abs()), "H")


@pytest.mark.parametrize("M", [3, 64, 150])
def test_glu_strided_operands_and_outputs(gen, M):
    D, F = 136, 264
    X, (Wg, Wu) = padded(randn(gen, M, D), 24), (padded(w, 40) for w in weights(gen, D, F))
    bufs = [torch.full((M + 2, F + 56), 7.0, device=gen.device, dtype=F16) for _ in range(3)]
    H, G, U = pax_b200.glu(X, Wg, Wu, out=bufs[0][1:-1, :F], G=bufs[1][1:-1, :F], U=bufs[2][1:-1, :F])
    for what, t, b in zip("HGU", (H, G, U), bufs):
        close(t, glu(X, Wg, Wu, "silu")[what], what)
        assert (b[:, F:] == 7).all() and (b[0] == 7).all() and (b[-1] == 7).all()


@pytest.mark.parametrize("M", [3, 150])
def test_sums_that_end_inside_a_16_byte_unit(gen, M):
    """Aligned row pitches with odd lengths: what follows a row's end is NaN or a code, and must not be read into the sum."""
    for D, F in ((133, 264), (70, 137)):
        X, (Wg, Wu) = padded(randn(gen, M, D), 200 - D), (padded(w, 280 - F) for w in weights(gen, D, F))
        buf = torch.full((M, 280), 7.0, device=gen.device, dtype=F16)
        close(pax_b200.glu(X, Wg, Wu, out=buf[:, :F]), glu(X, Wg, Wu, "silu")["H"], "H")
        assert (buf[:, F:] == 7).all()
        a = [padded(t, 280 - t.shape[1]) for t in back_inputs(gen, M, D, F)]
        ref = glu_grad(*a, "silu")
        for got, what in zip(pax_b200.glu_backward(*a), ("dX", "dWg", "dWu")):
            close(got, ref[what], what)
    A, B = padded(codes(gen, M, 137), 160 - 137, 55), padded(codes(gen, 40, 137), 176 - 137, 55)
    sa, sb = torch.rand(M, generator=gen, device=gen.device) * 1e-2, torch.rand(40, generator=gen, device=gen.device) * 1e-2
    close(pax_b200.gemm_i8(A, B, sa, sb), gemm_i8(A, B, sa, sb, None, True), "C")


@pytest.mark.parametrize("M", [2, 100])
def test_glu_unaligned_bases(gen, M):
    D, F = 64, 128
    X, (Wg, Wu) = shifted(randn(gen, M, D)), weights(gen, D, F)
    ref = glu(X, Wg, Wu, "silu")["H"]
    close(pax_b200.glu(X, Wg, Wu), ref, "X")
    close(pax_b200.glu(X, shifted(Wg, 3), Wu), ref, "W")
    out = shifted(torch.zeros(M, F, device=gen.device, dtype=F16))
    close(pax_b200.glu(X.clone(), Wg, Wu, out=out), ref, "out")


@pytest.mark.parametrize("M", [1, 64, 90])
def test_glu_empty_sum_is_zero(gen, M):
    X, W = randn(gen, M, 0), randn(gen, 0, 40)
    H, G, U = pax_b200.glu(X, W, W.clone(), save=True, out=torch.ones(M, 40, device=gen.device, dtype=F16))
    assert (H == 0).all() and (G == 0).all() and (U == 0).all()
    assert pax_b200.glu(randn(gen, 0, 8), *weights(gen, 8, 16)).shape == (0, 16)
    assert pax_b200.glu(randn(gen, 4, 8), *weights(gen, 8, 0)).shape == (4, 0)


@pytest.mark.parametrize("M", [4, 130])
def test_glu_keeps_nan_in_its_row_and_overflows_to_infinity(gen, M):
    D, F = 256, 136
    X, (Wg, Wu) = randn(gen, M, D), weights(gen, D, F)
    X[1, 3] = float("nan")
    H = pax_b200.glu(X, Wg, Wu)
    assert H[1].isnan().all()
    keep = [i for i in range(M) if i != 1]
    assert H[keep].isfinite().all()
    big = pax_b200.glu(torch.full((M, D), 60.0, device=gen.device, dtype=F16), Wg.abs() + 1, Wu.abs() + 1)
    assert (big == float("inf")).all()


# ------------------------------------------------------------------ backward
BACK_SHAPES = [(1, 64, 64), (3, 8, 8), (31, 136, 72), (64, 256, 128), (130, 768, 520), (257, 264, 1032), (512, 512, 256), (700, 1096, 328),
               (600, 264, 2056), (2500, 136, 264), (1100, 520, 1032), (4100, 72, 72),
               (5, 33, 64), (40, 64, 71), (90, 65, 130)]


def back_inputs(gen, M, D, F):
    X, (Wg, Wu) = randn(gen, M, D), weights(gen, D, F)
    return randn(gen, M, F, scale=0.5), X, Wg, Wu, randn(gen, M, F, scale=1.5), randn(gen, M, F)


@pytest.mark.parametrize("shape", BACK_SHAPES)
@pytest.mark.parametrize("dw", [F16, F32])
def test_glu_backward(gen, shape, dw):
    M, D, F = shape
    name = ACTS[(M + F) % 3]
    a = back_inputs(gen, M, D, F)
    dG, dU = torch.empty_like(a[0]), torch.empty_like(a[0])
    dX, dWg, dWu = pax_b200.glu_backward(*a, activation=name, dW_dtype=dw, dG=dG, dU=dU)
    assert dX.dtype == F16 and dWg.dtype == dWu.dtype == dw
    ref = glu_grad(*a, name, dw_f16=dw == F16)
    for what, t in (("dG", dG), ("dU", dU), ("dX", dX), ("dWg", dWg), ("dWu", dWu)):
        close(t, ref[what], what)


@pytest.mark.parametrize("name", ACTS)
def test_glu_gradients_agree_with_differences(gen, name):
    """d/dt sum(H . dH) along random directions, by central differences in 64 bits of the formula, for the gradients that
    the whole chain glu -> glu_backward returns."""
    M, D, F = 48, 64, 96
    X, (Wg, Wu) = randn(gen, M, D), weights(gen, D, F)
    dH = randn(gen, M, F)
    _, G, U = pax_b200.glu(X, Wg, Wu, activation=name, save=True)
    grads = pax_b200.glu_backward(dH, X, Wg, Wu, G, U, activation=name, dW_dtype=F32)
    leaves = [X.double(), Wg.double(), Wu.double()]

    def loss(ls):
        return (act(ls[0] @ ls[1], name) * (ls[0] @ ls[2]) * dH.double()).sum()

    for i in range(3):
        v = torch.randn(leaves[i].shape, generator=gen, device=gen.device, dtype=torch.float64)
        e = 1e-5
        up, dn = [list(leaves), list(leaves)]
        up[i], dn[i] = leaves[i] + e * v, leaves[i] - e * v
        want = (loss(up) - loss(dn)) / (2 * e)
        got = (grads[i].double() * v).sum()
        # roundings of G, U, dG, dU and the result: each 2^-11 of an element, met with random signs of v
        bound = 8 * 2.0 ** -11 * (grads[i].double() * v).norm() + 1e-6 * want.abs() + 1e-3
        assert (got - want).abs() <= bound, (i, got.item(), want.item(), bound.item())


@pytest.mark.parametrize("shape", [(130, 72, 136), (40, 33, 65), (600, 264, 2056), (2500, 136, 264)])
def test_glu_backward_parts_accumulation_and_shared_buffers(gen, shape):
    M, D, F = shape
    a = back_inputs(gen, M, D, F)
    ref = glu_grad(*a, "silu", dw_f16=False)
    full = pax_b200.glu_backward(*a, dW_dtype=F32)
    only_x = pax_b200.glu_backward(*a, need_dW=False)
    only_w = pax_b200.glu_backward(*a, need_dX=False, dW_dtype=F32)
    assert only_x[1] is None and only_x[2] is None and only_w[0] is None
    assert torch.equal(only_x[0], full[0]) and torch.equal(only_w[1], full[1]) and torch.equal(only_w[2], full[2])
    base = [randn(gen, D, F, dtype=F32) for _ in range(2)]
    acc = [b.clone() for b in base]
    pax_b200.glu_backward(*a, dWg=acc[0], dWu=acc[1], accumulate=True)
    for got, b, what in zip(acc, base, ("dWg", "dWu")):
        v, t = ref[what]
        close(got, (v + b.double(), t + 2.0 ** -24 * (v.abs() + b.double().abs() + t)), what)
    G, U = a[4].clone(), a[5].clone()
    shared = pax_b200.glu_backward(*a[:4], G, U, dW_dtype=F32, dG=G, dU=U)
    for x, y in zip(shared, full):
        assert torch.equal(x, y)
    close(G, ref["dG"], "dG in G")


@pytest.mark.parametrize("M", [70, 200])
def test_glu_backward_strided(gen, M):
    D, F = 72, 136
    a = [padded(t, 8 * (i + 1)) for i, t in enumerate(back_inputs(gen, M, D, F))]
    bx = torch.full((M, D + 8), 7.0, device=gen.device, dtype=F16)
    bg, bu = (torch.full((D, F + 16), 7.0, device=gen.device, dtype=F32) for _ in range(2))
    dX, dWg, dWu = pax_b200.glu_backward(*a, dX=bx[:, :D], dWg=bg[:, :F], dWu=bu[:, :F])
    ref = glu_grad(*a, "silu", dw_f16=False)
    close(dX, ref["dX"], "dX"), close(dWg, ref["dWg"], "dWg"), close(dWu, ref["dWu"], "dWu")
    assert (bx[:, D:] == 7).all() and (bg[:, F:] == 7).all() and (bu[:, F:] == 7).all()


def test_glu_backward_empty(gen):
    a = back_inputs(gen, 0, 16, 24)
    dX, dWg, dWu = pax_b200.glu_backward(*a, dWg=torch.ones(16, 24, device=gen.device), dWu=torch.ones(16, 24, device=gen.device))
    assert dX.shape == (0, 16) and (dWg == 0).all() and (dWu == 0).all()
    keep = [torch.ones(16, 24, device=gen.device) for _ in range(2)]
    pax_b200.glu_backward(*a, dWg=keep[0], dWu=keep[1], accumulate=True)
    assert (keep[0] == 1).all() and (keep[1] == 1).all()
    a = back_inputs(gen, 9, 16, 0)
    dX, dWg, dWu = pax_b200.glu_backward(*a, dX=torch.ones(9, 16, device=gen.device, dtype=F16))
    assert (dX == 0).all() and dWg.shape == (16, 0)
    dX, dWg, dWu = pax_b200.glu_backward(*back_inputs(gen, 9, 0, 16))
    assert dX.shape == (9, 0) and dWu.shape == (0, 16)


# ------------------------------------------------------------------ rows to int8
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (3, 7), (5, 8), (2, 64), (300, 1000), (7, 2048), (4, 2056), (9, 8192), (3, 8200),
                                   (2, 16384), (2, 20000), (2, 33), (1000, 136)])
def test_quantize_rows(gen, shape):
    X = randn(gen, *shape, scale=3.0)
    if shape[0] > 2:
        X[1] = 0
    Q, s = pax_b200.quantize_rows(X)
    q, ref = quantize(X)
    assert torch.equal(Q, q)
    close(s, (ref, 2.0 ** -24 * ref.abs()), "scale")


def test_quantize_rows_ties_and_every_magnitude(gen):
    """Every finite fp16 value against several row maxima: exact ties (254 x an odd multiple of the maximum), the largest and the
    smallest magnitudes, subnormal rows."""
    every = torch.arange(0, 0x7C00, dtype=torch.int16, device=gen.device).view(F16)
    rows = []
    for m in (127.0, 254.0, 63.5, 65504.0, 1.0, 0.333, 2.0 ** -24, 127 * 2.0 ** -24, 2.0 ** -14, 1016.0, 1270.0):
        m = torch.tensor(m, device=gen.device, dtype=F16)
        row = torch.where(every <= m, every, torch.zeros_like(every))
        row[0] = m
        rows.append(torch.stack([row, -row]))
    X = torch.cat(rows)
    for x in (X, X[:, :8000].contiguous(), X[:, :2001].contiguous()):
        Q, s = pax_b200.quantize_rows(x)
        assert torch.equal(Q, quantize(x)[0])


def test_quantize_rows_not_finite(gen):
    X = randn(gen, 6, 264)
    X[1, 5], X[2, 263], X[4, 0] = float("inf"), float("-inf"), float("nan")
    for x in (X, X[:, :261]):
        Q, s = pax_b200.quantize_rows(x)
        bad = ~x.isfinite().all(dim=1)
        assert s[bad].isnan().all() and (Q[bad] == 0).all()
        assert torch.equal(Q[~bad], quantize(x[~bad])[0])


def test_quantize_rows_strided_and_empty(gen):
    X = padded(randn(gen, 50, 136), 24)
    buf = torch.full((50, 160), 99, device=gen.device, dtype=I8)
    Q, _ = pax_b200.quantize_rows(X, out=buf[:, :136])
    assert torch.equal(Q, quantize(X)[0]) and (buf[:, 136:] == 99).all()
    Q, s = pax_b200.quantize_rows(randn(gen, 4, 0), scale=torch.ones(4, device=gen.device))
    assert Q.shape == (4, 0) and (s == 0).all()
    assert pax_b200.quantize_rows(randn(gen, 0, 8))[1].shape == (0,)
    assert torch.equal(pax_b200.quantize_rows(shifted(X))[0], quantize(X)[0])


# ------------------------------------------------------------------ 8-bit product
I8_SHAPES = [(1, 16, 16), (1, 1000, 4096), (3, 128, 128), (16, 264, 144), (17, 8, 2064), (33, 129, 256), (64, 4096, 1024), (65, 300, 400),
             (128, 256, 128), (130, 333, 1040), (256, 256, 256), (300, 1030, 640), (1000, 515, 272), (500, 300, 4112), (300, 515, 8192), (1, 5, 7), (20, 33, 30), (90, 70, 129),
             (2, 64, 32768)]


def codes(gen, m, k):
    return torch.randint(-128, 128, (m, k), generator=gen, device=gen.device, dtype=torch.int32).to(I8)


@pytest.mark.parametrize("shape", I8_SHAPES)
@pytest.mark.parametrize("out", [F16, F32])
@pytest.mark.parametrize("with_bias", [False, True])
def test_gemm_i8(gen, shape, out, with_bias):
    M, N, K = shape
    A, B = codes(gen, M, K), codes(gen, N, K)
    sa, sb = (torch.rand(n, generator=gen, device=gen.device) * 0.02 / K ** 0.25 + 1e-4 for n in (M, N))
    bias = randn(gen, N) if with_bias else None
    C = pax_b200.gemm_i8(A, B, sa, sb, bias=bias, out_dtype=out)
    close(C, gemm_i8(A, B, sa, sb, bias, out == F16), "C")


@pytest.mark.parametrize("M", [2, 70])
def test_gemm_i8_largest_sums_are_exact(gen, M):
    """The longest sum of the largest products, 131071 * 2^14 = 2^31 - 2^14, in both signs."""
    K, N = 131071, 8
    A, B = torch.full((M, K), -128, device=gen.device, dtype=I8), torch.full((N, K), -128, device=gen.device, dtype=I8)
    B[::2] = 127
    one = lambda n: torch.ones(n, device=gen.device)  # noqa: E731
    C = pax_b200.gemm_i8(A, B, one(M), one(N), out_dtype=F32)
    assert (C[:, 1::2] == float(K << 14)).all() and (C[:, ::2] == float(-K * 127 * 128)).all()
    K16 = 131056  # a row pitch of whole 16-byte units
    C = pax_b200.gemm_i8(A[:, :K16].contiguous(), B[:, :K16].contiguous(), one(M), one(N), out_dtype=F32)
    assert (C[:, 1::2] == float(K16 << 14)).all() and (C[:, ::2] == float(-K16 * 127 * 128)).all()


@pytest.mark.parametrize("M", [4, 64, 200])
@pytest.mark.parametrize("out", [F16, F32])
def test_gemm_i8_strided(gen, M, out):
    N, K = 137, 144
    A, B = padded(codes(gen, M, K), 16, 55), padded(codes(gen, N, K), 32, 55)
    sa, sb = torch.rand(M, generator=gen, device=gen.device) * 1e-2, torch.rand(N, generator=gen, device=gen.device) * 1e-2
    for wide in (N + 7, N + 8):
        buf = torch.full((M, wide), 7.0, device=gen.device, dtype=out)
        C = pax_b200.gemm_i8(A, B, sa, sb, out=buf[:, :N])
        close(C, gemm_i8(A, B, sa, sb, None, out == F16), "C")
        assert (buf[:, N:] == 7).all()
    C = pax_b200.gemm_i8(shifted(A), B, sa, sb, out_dtype=out)
    close(C, gemm_i8(A, B, sa, sb, None, out == F16), "C")


@pytest.mark.parametrize("M,K", [(200, 144), (300, 2064)])
@pytest.mark.parametrize("N", [129, 130, 131, 201, 318])
@pytest.mark.parametrize("out", [F16, F32])
def test_gemm_i8_rows_on_2_4_and_8_bytes(gen, M, K, N, out):
    """Every alignment of the output's rows, their last element anywhere in a unit; what follows the rows stays."""
    A, B = codes(gen, M, K), codes(gen, N, K)
    sa, sb = torch.rand(M, generator=gen, device=gen.device) * 1e-2, torch.rand(N, generator=gen, device=gen.device) * 1e-2
    ref = gemm_i8(A, B, sa, sb, None, out == F16)
    for wide in (N + 1, N + 2, N + 3, N + 4):
        buf = torch.full((M + 1, wide), 7.0, device=gen.device, dtype=out)
        close(pax_b200.gemm_i8(A, B, sa, sb, out=buf[:M, :N]), ref, "C")
        assert (buf[:, N:] == 7).all() and (buf[M] == 7).all()


@pytest.mark.parametrize("M", [3, 80])
def test_gemm_i8_empty_sum_and_scales_that_are_not_finite(gen, M):
    one = lambda n: torch.ones(n, device=gen.device)  # noqa: E731
    b = randn(gen, 24)
    C = pax_b200.gemm_i8(codes(gen, M, 0), codes(gen, 24, 0), one(M), one(24), bias=b)
    assert torch.equal(C, b.expand(M, 24))
    assert pax_b200.gemm_i8(codes(gen, 0, 16), codes(gen, 24, 16), one(0), one(24)).shape == (0, 24)
    sa, sb = one(M), one(24)
    sa[1], sb[5] = float("nan"), 0.0
    C = pax_b200.gemm_i8(codes(gen, M, 16), codes(gen, 24, 16), sa, sb, out_dtype=F32)
    assert C[1].isnan().all() and (C[0, 5] == 0) and C[2].isfinite().all()


# ------------------------------------------------------------------ large
@pytest.mark.slow
@pytest.mark.parametrize("extra", [0, 1])
def test_offsets_beyond_32_bits(gen, extra):
    """More than 2^31 elements a matrix, in aligned rows and in rows that are not: the last rows are where a 32-bit offset
    would go astray."""
    M, F, D = 66000, 32768 + extra, 64
    last = slice(M - 130, M)
    X, (Wg, Wu) = randn(gen, M, D), weights(gen, D, F)
    H, G, U = pax_b200.glu(X, Wg, Wu, save=True)
    ref = glu(X[last], Wg, Wu, "silu")
    for what, t in (("H", H), ("G", G), ("U", U)):
        close(t[last], ref[what], what)
    dG, dU = torch.empty_like(G), torch.empty_like(G)
    dX, _, _ = pax_b200.glu_backward(H, X, Wg, Wu, G, U, dG=dG, dU=dU, need_dW=False)
    ref = glu_grad(H[last], X[last], Wg, Wu, G[last], U[last], "silu")
    for what, t in (("dX", dX), ("dG", dG), ("dU", dU)):
        close(t[last], ref[what], what)
    del dG, dU, U, G
    Q, s = pax_b200.quantize_rows(H)
    assert torch.equal(Q[last], quantize(H[last])[0])
    del H
    # the same for the 8-bit product's output and for its operand
    A, B = codes(gen, M, 80), codes(gen, F, 80)
    sa, sb = torch.rand(M, generator=gen, device=gen.device) * 1e-2, torch.rand(F, generator=gen, device=gen.device) * 1e-2
    C = pax_b200.gemm_i8(A, B, sa, sb)
    close(C[last], gemm_i8(A[last], B, sa[last], sb, None, True), "C")
    del C
    W = codes(gen, 40, F)
    C = pax_b200.gemm_i8(Q, W, s, sb[:40].contiguous(), out_dtype=F32)
    close(C[last], gemm_i8(Q[last], W, s[last], sb[:40], None, False), "C")


# ------------------------------------------------------------------ together
def test_training_step_of_a_gated_layer(gen):
    """glu, the framework's own product as down-projection, and the gradients back to the input and both weights."""
    M, D, F = 200, 136, 264
    X, (Wg, Wu) = randn(gen, M, D), weights(gen, D, F)
    Wd, dY = randn(gen, F, D, scale=F ** -0.5), randn(gen, M, D)
    H, G, U = pax_b200.glu(X, Wg, Wu, save=True)
    Y = pax_b200.gemm(H, Wd, out_dtype=F32)
    close(Y, (H.double() @ Wd.double(), F * 2.0 ** -23 * (H.double().abs() @ Wd.double().abs()) + 1e-6), "Y")
    dH = pax_b200.gemm(dY, Wd.T.contiguous())
    got = pax_b200.glu_backward(dH, X, Wg, Wu, G, U)
    ref = glu_grad(dH, X, Wg, Wu, G, U, "silu")
    for t, what in zip(got, ("dX", "dWg", "dWu")):
        close(t, ref[what], what)


@pytest.mark.parametrize("M", [1, 48, 300])
def test_serving_a_quantised_projection(gen, M):
    """Weights quantised once, tokens per call: within the two quantisation steps of the fp16 product."""
    D, N = 512, 264
    X, W = randn(gen, M, D), randn(gen, N, D, scale=D ** -0.5)
    Wq, sw = pax_b200.quantize_rows(W)
    Xq, sx = pax_b200.quantize_rows(X)
    Y = pax_b200.gemm_i8(Xq, Wq, sx, sw, out_dtype=F32)
    x, w = X.double(), W.double()
    ex, ew = 0.501 * sx.double()[:, None], 0.501 * sw.double()[:, None]  # half a step, and the scale's own rounding
    tol = ex * w.abs().sum(1)[None, :] + x.abs().sum(1)[:, None] * ew.T + D * ex * ew.T + 1e-5
    close(Y, (x @ w.T, tol), "Y")


def run_all(t):
    H, G, U = pax_b200.glu(t["X"], t["Wg"], t["Wu"], save=True)
    grads = pax_b200.glu_backward(t["dH"], t["X"], t["Wg"], t["Wu"], G, U)
    Q, s = pax_b200.quantize_rows(t["X"])
    return (H, G, U, *grads, Q, s, pax_b200.gemm_i8(Q, t["Wq"], s, t["sw"]))


def all_inputs(gen, M, D=264, F=520):
    t = {"X": randn(gen, M, D), "dH": randn(gen, M, F)}
    t["Wg"], t["Wu"] = weights(gen, D, F)
    t["Wq"], t["sw"] = pax_b200.quantize_rows(randn(gen, 136, D))
    return t


@pytest.mark.parametrize("M", [1, 40, 300])
def test_calls_repeat_bit_for_bit(gen, M):
    t = all_inputs(gen, M)
    first = run_all(t)
    for _ in range(5):
        for a, b in zip(first, run_all(t)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("M", [7, 300])
def test_captured_and_replayed(gen, M):
    """Two graphs captured from the same calls, replayed by turns and at once on two streams, with new inputs in place."""
    t = [all_inputs(gen, M) for _ in range(2)]
    want = [run_all(x) for x in t]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for x, s in zip(t, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run_all(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(run_all(x))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        for a, b in zip(w, o):
            assert torch.equal(a, b)
    t[0]["X"].copy_(t[1]["X"])
    graphs[0].replay()
    fresh = run_all(t[0])
    torch.cuda.synchronize()
    for a, b in zip(fresh, outs[0]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("M", [7, 300])
def test_other_stream_and_calls_at_once(gen, M):
    t = [all_inputs(gen, M) for _ in range(3)]
    want = [run_all(x) for x in t]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for x, s in zip(t, streams):
            H, G, U = pax_b200.glu(x["X"], x["Wg"], x["Wu"], save=True, stream=s)
            grads = pax_b200.glu_backward(x["dH"], x["X"], x["Wg"], x["Wu"], G, U, stream=s)
            Q, sc = pax_b200.quantize_rows(x["X"], stream=s)
            got.append((H, G, U, *grads, Q, sc, pax_b200.gemm_i8(Q, x["Wq"], sc, x["sw"], stream=s)))
        torch.cuda.synchronize()
        for w, o in zip(want, got):
            for a, b in zip(w, o):
                assert torch.equal(a, b)


@pytest.mark.parametrize("shape", [(40, 264, 520), (130, 768, 2048), (100, 512, 512)])
def test_backward_passes_in_a_row_with_inputs_that_change(gen, shape):
    """Passes queued without a pause, the inputs overwritten in place between them: each launch of a pass starts while the one
    before ends, and none may read what the last pass or the next one writes."""
    M, D, F = shape
    sets = [back_inputs(gen, M, D, F) for _ in range(3)]
    want = [pax_b200.glu_backward(*a) for a in sets]
    torch.cuda.synchronize()
    live = [t.clone() for t in sets[0]]
    wrong = torch.zeros((), device=gen.device, dtype=torch.int64)
    for i in range(150):
        for t, new in zip(live, sets[i % 3]):
            t.copy_(new)
        got = pax_b200.glu_backward(*live, dG=live[4], dU=live[5])
        for g, w in zip(got, want[i % 3]):
            wrong += (g != w).sum()
    assert wrong.item() == 0


def test_glu_backward_sums_over_more_tokens_than_a_bounded_wait_covers(gen):
    """One term in 2^20 tokens is not zero and every product of them is exact, so that the sums are too."""
    M = (1 << 26) + 72
    X, G, U, dH = (torch.zeros(M, 8, device=gen.device, dtype=F16) for _ in range(4))
    X[:: 1 << 20] = 2.0
    U[:: 1 << 20] = 1.0
    dH[:: 1 << 20] = 1.0
    W = torch.zeros(8, 8, device=gen.device, dtype=F16)
    _, dWg, dWu = pax_b200.glu_backward(dH, X, W, W.clone(), G, U, need_dX=False, dW_dtype=F32, dG=G, dU=U)
    # silu'(0) = 1/2 and silu(0) = 0: 65 tokens of 2 * 1/2
    assert (dWg == 65.0).all() and (dWu == 0).all()
    assert pax_b200.device_error() == pax_b200.Status.OK


@pytest.mark.parametrize("between", ["glu, few tokens", "glu, tiles", "glu, split", "gemm_i8, tiles", "gemm, tiles", "gemm, few rows"])
def test_constant_weights_written_by_the_kernel_before_the_one_just_before(gen, between):
    """Three kernels in a row: the first writes B, the second is small and leaves most of the GPU free, the third has b_const."""
    N = K = 8192
    W, A = randn(gen, N, K), codes(gen, 1, K)
    ones = torch.ones(N, device=gen.device)
    Q, s = pax_b200.quantize_rows(W)
    ref = pax_b200.gemm_i8(A, Q, ones[:1], ones, out_dtype=F32)
    M, D, F = {"glu, few tokens": (1, 64, 64), "glu, split": (256, 2048, 128)}.get(between, (256, 64, 128))
    X, Y = randn(gen, M, D), randn(gen, D, F)
    A2, B2, s2, C = codes(gen, M, D), codes(gen, F, D), ones[:M], torch.empty((M, F), device=gen.device, dtype=F32)
    second = {"glu": lambda: pax_b200.glu(X, Y, Y), "gemm_i8": lambda: pax_b200.gemm_i8(A2, B2, s2, ones[:F]),
              "gemm": lambda: pax_b200.gemm(X if "tiles" in between else X[:4], Y, out=C if "tiles" in between else C[:4])}
    second = second[between.split(",")[0]]
    for _ in range(10):
        Q.fill_(1)
        pax_b200.quantize_rows(W, out=Q, scale=s)
        second()
        assert torch.equal(pax_b200.gemm_i8(A, Q, ones[:1], ones, out_dtype=F32, b_const=True), ref)


@pytest.mark.parametrize("M", [1, 24, 64])
def test_decoding_chain_with_constant_weights(gen, M):
    """Layers in a row, each reading what the one before wrote, with their weights marked constant: the same bits as without."""
    D, F, L = 512, 1032, 6
    X = randn(gen, M, D)
    W = [(*weights(gen, D, F), *pax_b200.quantize_rows(randn(gen, D, F, scale=F ** -0.5))) for _ in range(L)]

    def chain(const):
        x = X
        for Wg, Wu, Wq, sw in W:
            H = pax_b200.glu(x, Wg, Wu, w_const=const)
            Q, s = pax_b200.quantize_rows(H)
            x = pax_b200.gemm_i8(Q, Wq, s, sw, b_const=const)
            x = x / x.float().std().clamp_min(1e-3).half()
            H2 = pax_b200.glu(x, Wg, Wu, w_const=const)  # weights loaded while the first product still runs
            x = pax_b200.gemm(H2, Wd[:F], b_const=const)
        return x

    Wd = randn(gen, F, D, scale=F ** -0.5)
    want = chain(False)
    for _ in range(20):
        assert torch.equal(chain(True), want)


CAPTURE_FIRST = """
import torch, pax_b200
g = torch.Generator(device="cuda"); g.manual_seed(3)
h = lambda *s: (torch.randn(s, generator=g, device="cuda") * 0.1).half()
for M in (7, 300):
    X, Wg, Wu, dH = h(M, 264), h(264, 520), h(264, 520), h(M, 520)
    Wq, sw = torch.randint(-9, 9, (136, 264), device="cuda", dtype=torch.int8), torch.rand(136, device="cuda")
    def run():
        H, G, U = pax_b200.glu(X, Wg, Wu, save=True)
        Q, s = pax_b200.quantize_rows(X)
        return (H, G, U, *pax_b200.glu_backward(dH, X, Wg, Wu, G, U), Q, s, pax_b200.gemm_i8(Q, Wq, s, sw))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, run()))
print("ok")
"""


def test_the_first_call_of_a_process_can_be_captured(cuda):
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CAPTURE_FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stderr[-2000:]


def test_no_device_error_was_recorded(cuda):
    assert pax_b200.device_error() == pax_b200.Status.OK
