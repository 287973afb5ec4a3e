"""Feed-forward products on torch CUDA tensors: the gated up-projection with
its backward pass in fp16, and the 8-bit integer product with scales per token
and output channel.  torch supplies device memory and the stream; the work
runs in libpax_b200.so (pax_glu_ex, pax_glu_backward_ex, pax_quantize_rows,
pax_gemm_i8_ex).

Every call is asynchronous on the current stream of the tensors' device, or on
``stream``, whatever device is current.  A new output belongs to that stream:
a caller that passes ``stream`` orders its own use of the output after it, and
that stream's work after what writes the inputs.  The inputs themselves may be
freed right after the call.
Outputs must not overlap inputs or each other, but for glu_backward's dG and dU.
autograd records none of the calls, whatever their inputs require:
glu_backward is called by hand.  It does see that a given output was written.
"""
from __future__ import annotations

from enum import IntEnum

import torch

from ._lib import LibraryNotBuilt
from .api import _DT


class Activation(IntEnum):
    SILU = 0
    GELU_TANH = 1
    GELU_ERF = 2


_ACT = {a.name.lower(): int(a) for a in Activation}


def _activation(a) -> int:
    if isinstance(a, str):
        if a not in _ACT:
            raise ValueError(f"activation must be one of {', '.join(_ACT)}")
        return _ACT[a]
    return int(Activation(a))


_MODULE = None


def _native():
    """The module that checks, allocates and launches (csrc/torch_feed_forward.cpp)."""
    global _MODULE
    if _MODULE is None:
        try:
            from . import _feed_forward
        except ImportError as e:
            raise LibraryNotBuilt("pax_b200/_feed_forward.so is missing or does not load: build it with "
                                  f"`python -m pax_b200.build` (nvcc, g++). There is no fallback. ({e})") from e
        _MODULE = _feed_forward
    return _MODULE


def glu(X: torch.Tensor, Wg: torch.Tensor, Wu: torch.Tensor, *, activation="silu", save: bool = False,
        out: torch.Tensor | None = None, G: torch.Tensor | None = None, U: torch.Tensor | None = None,
        stream: torch.cuda.Stream | None = None, w_const: bool = False):
    """H = act(X @ Wg) * (X @ Wu): both projections of a gated feed-forward
    layer, the activation and the product in one kernel.

    X [M, D], Wg and Wu [D, F] are float16 with unit column stride; H is
    float16 [M, F].  activation is one of silu, gelu_tanh, gelu_erf.  With
    ``save`` (or given G and U) the products X @ Wg and X @ Wu are kept for
    glu_backward, in float16, and (H, G, U) is returned instead of H.
    w_const: Wg and Wu are not written by the kernel launched just before on
    this stream (weights); with at most 64 tokens the kernel may then start
    reading them before that kernel ends (as gemm's b_const).
    """
    return _native().glu(X, Wg, Wu, _activation(activation), bool(save), out, G, U, stream, bool(w_const))


def glu_backward(dH: torch.Tensor, X: torch.Tensor, Wg: torch.Tensor, Wu: torch.Tensor, G: torch.Tensor, U: torch.Tensor,
                 *, activation="silu", need_dX: bool = True, need_dW: bool = True, dX: torch.Tensor | None = None,
                 dWg: torch.Tensor | None = None, dWu: torch.Tensor | None = None,
                 dW_dtype: torch.dtype = torch.float16, accumulate: bool = False, dG: torch.Tensor | None = None,
                 dU: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None):
    """(dX, dWg, dWu) of glu from dH and the G and U that glu kept.

    All inputs are float16; dX is float16 [M, D], dWg and dWu are dW_dtype
    (float16 or float32) [D, F].  ``need_dX`` / ``need_dW`` false leaves that
    part out (None in its place).  ``accumulate`` adds the weight gradients to
    the given float32 dWg and dWu.  dG and dU take the gradients of the two
    products and may be G and U themselves, which saves 2 M F values of
    scratch; by default they are scratch of the call.

    dG and dU are rounded to float16 between the two steps: beyond 65504 they
    become infinities, which reach dX and the weight gradients, and at 2^-25 or
    less zeros.  dH is scaled for that by the caller, as float16 gradients are.
    """
    if dW_dtype not in _DT:
        raise TypeError("weight gradients must be float32 or float16")
    return _native().glu_backward(dH, X, Wg, Wu, G, U, _activation(activation), bool(need_dX), bool(need_dW), dX, dWg, dWu,
                                  int(_DT[dW_dtype]), bool(accumulate), dG, dU, stream)


def quantize_rows(X: torch.Tensor, *, out: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                  stream: torch.cuda.Stream | None = None):
    """(Q, scale): rows of float16 X [M, K] as int8 codes and one float32 scale
    each, scale = max|x| / 127 and Q = round(127 x / max|x|), ties to even, so
    that X is about Q * scale[:, None].  Used for activations, one scale per
    token, and for weights [N, K], one scale per output channel.  A row of
    zeros has scale 0; one with an infinity or NaN has scale NaN and codes 0.
    """
    return _native().quantize_rows(X, out, scale, stream)


def gemm_i8(A: torch.Tensor, B: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor, *,
            bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
            out_dtype: torch.dtype = torch.float16, stream: torch.cuda.Stream | None = None,
            b_const: bool = False) -> torch.Tensor:
    """C = (A @ B.T) * a_scale[:, None] * b_scale[None, :] (+ bias).

    A [M, K] and B [N, K] are int8 with unit column stride (what quantize_rows
    gives for tokens and for the weight's output channels), the scales float32
    [M] and [N], bias float16 [N]; C is float16 or float32 [M, N].  The sums
    are exact 32-bit integers, for K up to 131071.  b_const: B is not written
    by the kernel launched just before on this stream, as in gemm.
    """
    if out_dtype not in _DT:
        raise TypeError("out_dtype must be float32 or float16")
    return _native().gemm_i8(A, B, a_scale, b_scale, bias, out, int(_DT[out_dtype]), stream, bool(b_const))
