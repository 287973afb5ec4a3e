"""Plain 64-bit forms of the feed-forward products, with bounds on what fp32
sums and the named roundings may change.

One fp32 sum of n products is off by at most n * 2^-23 * sum |a b| (n - 1
additions of up to 2^-24 each, doubled for sums that truncate); a rounding to
fp16 by 2^-11 of the value, or 2^-25 among the subnormals.
"""
from __future__ import annotations

import torch

E16, SUB16, E32 = 2.0 ** -11, 2.0 ** -25, 2.0 ** -23
ACTS = ("silu", "gelu_tanh", "gelu_erf")
# Absolute error of act and act' as evaluated in fp32, relative to 1 + |x|:
# exp and reciprocal are good to a few 2^-22, the erf formula to 3e-7.
ACT_ERR = 2e-6


def act(x, name):
    if name == "silu":
        return x * torch.sigmoid(x)
    if name == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)))
    return 0.5 * x * torch.special.erfc(-x / 2 ** 0.5)


def act_grad(x, name):
    x = x.detach().requires_grad_(True)
    (d,) = torch.autograd.grad(act(x, name).sum(), x)
    return d


def rounded16(tol, ref):
    """Bound after one more rounding to fp16 of values within tol of ref."""
    return tol + E16 * (ref.abs() + tol) + SUB16


def glu(X, Wg, Wu, name):
    """{output: (64-bit value, bound)}"""
    x, wg, wu = X.double(), Wg.double(), Wu.double()
    n = X.shape[1]
    g, u = x @ wg, x @ wu
    tg, tu = n * E32 * (x.abs() @ wg.abs()), n * E32 * (x.abs() @ wu.abs())
    a = act(g, name)
    # |act'| < 1.13; act evaluated with ACT_ERR
    ta = 1.13 * tg + ACT_ERR * (1 + g.abs())
    h = a * u
    th = ta * (u.abs() + tu) + a.abs() * tu + 2 * E32 * h.abs()
    return {"H": (h, rounded16(th, h)), "G": (g, rounded16(tg, g)), "U": (u, rounded16(tu, u))}


def glu_grad(dH, X, Wg, Wu, G, U, name, dw_f16=True):
    x, wg, wu = X.double(), Wg.double(), Wu.double()
    dh, g, u = dH.double(), G.double(), U.double()
    a, d = act(g, name), act_grad(g, name)
    dg, du = dh * u * d, dh * a
    # one rounding to fp16 of dG and dU, the operands of the two products
    err = ACT_ERR * (1 + g.abs())
    tg = rounded16((dh * u).abs() * err + 3 * E32 * dg.abs(), dg)
    tu = rounded16(dh.abs() * err + 3 * E32 * du.abs(), du)
    m, f = dH.shape
    dx = dg @ wg.T + du @ wu.T
    tx = tg @ wg.abs().T + tu @ wu.abs().T + 2 * f * E32 * ((dg.abs() + tg) @ wg.abs().T + (du.abs() + tu) @ wu.abs().T)
    out = {"dG": (dg, tg), "dU": (du, tu), "dX": (dx, rounded16(tx, dx))}
    for name_, v, t in (("dWg", dg, tg), ("dWu", du, tu)):
        dw = x.T @ v
        tw = x.abs().T @ t + m * E32 * (x.abs().T @ (v.abs() + t))
        out[name_] = (dw, rounded16(tw, dw) if dw_f16 else tw + E32 * dw.abs())
    return out


def quantize(X):
    """Codes and scales by exact integer arithmetic: fp16 values are integers
    over 2^24, and round-half-even of 127 |x| / m is decided on integers."""
    xi = (X.double() * 2 ** 24).to(torch.int64)
    m = xi.abs().amax(dim=1, keepdim=True) if X.shape[1] else torch.zeros((X.shape[0], 1), dtype=torch.int64, device=X.device)
    safe = m.clamp_min(1)
    n2 = 254 * xi.abs()  # twice 127 |x|
    q = (n2 + safe) // (2 * safe)  # floor(127|x|/m + 1/2)
    tie = (n2 + safe) % (2 * safe) == 0
    q = torch.where(tie & (q % 2 == 1), q - 1, q) * torch.sign(xi)
    return q.to(torch.int8), (m[:, 0].double() / 2 ** 24 / 127)


def gemm_i8(A, B, sa, sb, bias, f16):
    acc = A.double() @ B.double().T  # exact: below 2^53
    s = sa.double()[:, None] * sb.double()[None, :]
    c = acc * s
    t = 4 * 2.0 ** -24 * c.abs() + 2.0 ** -126  # int to fp32, two products, each half a step; subnormal scales
    if bias is not None:
        b = bias.double()[None, :]
        c = c + b
        t = t + 2.0 ** -24 * (c.abs() + t)
    return c, rounded16(t, c) if f16 else t


def close(got, ref_tol, what=""):
    ref, tol = ref_tol
    got = got.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    if got.numel() == 0:
        return
    # beyond fp16's largest value a correct result is an infinity
    bad = ~((got - ref).abs() <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, first at "
                                 f"{bad.nonzero()[0].tolist()}: {got[bad][0].item()} for {ref[bad][0].item()}, "
                                 f"bound {tol[bad][0].item():.3g}")
