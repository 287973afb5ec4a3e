"""Feed-forward products on torch CUDA tensors: the gated up-projection with
its backward pass in fp16, and the 8-bit integer product with scales per token
and output channel.  torch supplies device memory and the stream; the work
runs in libpax_b200.so (pax_glu_ex, pax_glu_backward_ex, pax_quantize_rows,
pax_gemm_i8_ex).

Every call is asynchronous on the current stream of the tensors' device, or on
``stream``, whatever device is current.  A new output belongs to that stream:
a caller that passes ``stream`` orders its own use of the output after it.
autograd records none of the calls: glu_backward is called by hand.
"""
from __future__ import annotations

import ctypes
from enum import IntEnum

import torch

from . import _lib
from .api import _DT, PaxError


class Activation(IntEnum):
    SILU = 0
    GELU_TANH = 1
    GELU_ERF = 2


_ACT_NAMES = {a.name.lower(): a for a in Activation}


def _activation(a) -> int:
    if isinstance(a, str):
        if a not in _ACT_NAMES:
            raise ValueError(f"activation must be one of {', '.join(_ACT_NAMES)}")
        return int(_ACT_NAMES[a])
    return int(Activation(a))


def _matrix(t: torch.Tensor, name: str, rows: int, cols: int, dtypes: tuple, device: torch.device) -> int:
    """Checks an operand and returns its leading dimension (elements)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d).removeprefix('torch.') for d in dtypes)}")
    if t.shape != (rows, cols):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {(rows, cols)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    s0, s1 = t.stride()
    if rows > 1 and s1 == 1 and s0 >= cols > 0:
        return s0
    if rows == 0 or cols == 0:
        return 0
    if cols > 1 and s1 != 1:
        raise ValueError(f"{name} must be a 2-D tensor with unit column stride")
    if rows == 1:  # the pitch of one row is never used
        return 0
    if s0 < cols:  # expanded or overlapping rows
        raise ValueError(f"{name} must have rows that do not overlap")
    return s0


def _vector(t: torch.Tensor, name: str, n: int, dtype: torch.dtype, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError(f"{name} must be a {str(dtype).removeprefix('torch.')} tensor")
    if t.shape != (n,):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected ({n},)")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")


def _dims(t, name: str) -> tuple:
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D tensor")
    return t.shape


class _Call:
    """The device and stream of one call.  Outputs are allocated on the
    call's stream, so that neither their memory's earlier use nor the reuse
    after them can overlap the call, and stay reserved for the caller's
    current stream as well."""

    __slots__ = ("device", "other", "raw")

    def __init__(self, device: torch.device, stream: torch.cuda.Stream | None):
        if device.type != "cuda":
            raise ValueError("tensors must be on a CUDA device")
        self.device = device
        self.other = None
        if stream is None:
            self.raw = torch._C._cuda_getCurrentRawStream(device.index)
        else:
            if stream.device != device:
                raise ValueError(f"stream is on {stream.device}, expected {device}")
            self.raw = stream.cuda_stream
            if stream != torch.cuda.current_stream(device):
                self.other = stream

    def empty(self, like: torch.Tensor, shape, dtype=None, scratch=False) -> torch.Tensor:
        if dtype is None:
            dtype = like.dtype
        if self.other is None:
            return like.new_empty(shape, dtype=dtype)
        with torch.cuda.stream(self.other):
            t = like.new_empty(shape, dtype=dtype)
        if not scratch:
            t.record_stream(torch.cuda.current_stream(self.device))
        return t

    def run(self, name: str, *args) -> None:
        fn = getattr(_lib.get(), name)
        if torch.cuda.current_device() == self.device.index:
            st = fn(*args, self.raw)
        else:
            with torch.cuda.device(self.device):
                st = fn(*args, self.raw)
        if st != 0:
            raise PaxError(st, name)


_F16, _I8, _OUT = (torch.float16,), (torch.int8,), tuple(_DT)


def glu(X: torch.Tensor, Wg: torch.Tensor, Wu: torch.Tensor, *, activation="silu", save: bool = False,
        out: torch.Tensor | None = None, G: torch.Tensor | None = None, U: torch.Tensor | None = None,
        stream: torch.cuda.Stream | None = None):
    """H = act(X @ Wg) * (X @ Wu): both projections of a gated feed-forward
    layer, the activation and the product in one kernel.

    X [M, D], Wg and Wu [D, F] are float16 with unit column stride; H is
    float16 [M, F].  activation is one of silu, gelu_tanh, gelu_erf.  With
    ``save`` (or given G and U) the products X @ Wg and X @ Wu are kept for
    glu_backward, and (H, G, U) is returned instead of H.
    """
    M, D = _dims(X, "X")
    _, F = _dims(Wg, "Wg")
    act = _activation(activation)
    if (G is None) != (U is None):
        raise ValueError("G and U go together")
    dev = X.device
    ldx = _matrix(X, "X", M, D, _F16, dev)
    ldwg, ldwu = _matrix(Wg, "Wg", D, F, _F16, dev), _matrix(Wu, "Wu", D, F, _F16, dev)
    ldh = _matrix(out, "out", M, F, _F16, dev) if out is not None else F
    ldg = ldu = F
    if G is not None:
        ldg, ldu = _matrix(G, "G", M, F, _F16, dev), _matrix(U, "U", M, F, _F16, dev)
    call = _Call(dev, stream)
    H = out if out is not None else call.empty(X, (M, F))
    if save and G is None:
        G, U = call.empty(X, (M, F)), call.empty(X, (M, F))
    g, u = (0, 0) if G is None else (G.data_ptr(), U.data_ptr())
    d = _lib.GluDesc(X.data_ptr(), Wg.data_ptr(), Wu.data_ptr(), H.data_ptr(), g, u, M, D, F, ldx, ldwg, ldwu, ldh, ldg,
                     ldu, act)
    call.run("pax_glu_ex", ctypes.byref(d))
    return H if G is None else (H, G, U)


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
    """
    M, D = _dims(X, "X")
    _, F = _dims(Wg, "Wg")
    dev = X.device
    act = _activation(activation)
    if (dWg is None) != (dWu is None):
        raise ValueError("dWg and dWu go together")
    if dWg is not None:
        if not need_dW:
            raise ValueError("dWg and dWu are given, but need_dW is false")
        dW_dtype = dWg.dtype
    if dX is not None and not need_dX:
        raise ValueError("dX is given, but need_dX is false")
    if dW_dtype not in _DT:
        raise TypeError("weight gradients must be float32 or float16")
    if accumulate and (dWg is None or dW_dtype != torch.float32):
        raise ValueError("accumulate needs given float32 dWg and dWu")
    lds = [_matrix(dH, "dH", M, F, _F16, dev), _matrix(X, "X", M, D, _F16, dev), _matrix(Wg, "Wg", D, F, _F16, dev),
           _matrix(Wu, "Wu", D, F, _F16, dev), _matrix(G, "G", M, F, _F16, dev), _matrix(U, "U", M, F, _F16, dev)]
    lds += (F if dG is None else _matrix(dG, "dG", M, F, _F16, dev), F if dU is None else _matrix(dU, "dU", M, F, _F16, dev),
            D if dX is None else _matrix(dX, "dX", M, D, _F16, dev))
    if dWg is None:
        lds += (F, F)
    else:
        lds += (_matrix(dWg, "dWg", D, F, (dW_dtype,), dev), _matrix(dWu, "dWu", D, F, (dW_dtype,), dev))
    call = _Call(dev, stream)
    plain = call.other is None  # a contiguous input of the same kind is the quickest model of an output
    if need_dX and dX is None:
        dX = torch.empty_like(X) if plain and lds[1] == D else call.empty(X, (M, D))
    if need_dW and dWg is None:
        if plain and lds[2] == F and dW_dtype is torch.float16:
            dWg, dWu = torch.empty_like(Wg), torch.empty_like(Wg)
        else:
            dWg, dWu = call.empty(Wg, (D, F), dW_dtype), call.empty(Wg, (D, F), dW_dtype)
    if dG is None and dU is None:
        scratch = call.empty(X, (2, M, F), scratch=True)  # freed on the call's stream, after the call
        dg = scratch.data_ptr()
        du = dg + 2 * M * F
    else:
        dG = dG if dG is not None else call.empty(X, (M, F), scratch=True)
        dU = dU if dU is not None else call.empty(X, (M, F), scratch=True)
        dg, du = dG.data_ptr(), dU.data_ptr()
    d = _lib.GluGradDesc(dH.data_ptr(), X.data_ptr(), Wg.data_ptr(), Wu.data_ptr(), G.data_ptr(), U.data_ptr(), dg, du,
                         *(0 if t is None else t.data_ptr() for t in (dX, dWg, dWu)), M, D, F, *lds, _DT[dW_dtype],
                         accumulate, act)
    call.run("pax_glu_backward_ex", ctypes.byref(d))
    return dX, dWg, dWu


def quantize_rows(X: torch.Tensor, *, out: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                  stream: torch.cuda.Stream | None = None):
    """(Q, scale): rows of float16 X [M, K] as int8 codes and one float32 scale
    each, scale = max|x| / 127 and Q = round(127 x / max|x|), ties to even, so
    that X is about Q * scale[:, None].  Used for activations, one scale per
    token, and for weights [N, K], one scale per output channel.  A row of
    zeros has scale 0; one with an infinity or NaN has scale NaN and codes 0.
    """
    M, K = _dims(X, "X")
    dev = X.device
    ldx = _matrix(X, "X", M, K, _F16, dev)
    ldq = _matrix(out, "out", M, K, _I8, dev) if out is not None else K
    if scale is not None:
        _vector(scale, "scale", M, torch.float32, dev)
    call = _Call(dev, stream)
    Q = out if out is not None else call.empty(X, (M, K), torch.int8)
    s = scale if scale is not None else call.empty(X, (M,), torch.float32)
    call.run("pax_quantize_rows", X.data_ptr(), ldx, Q.data_ptr(), ldq, s.data_ptr(), M, K)
    return Q, s


def gemm_i8(A: torch.Tensor, B: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor, *,
            bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
            out_dtype: torch.dtype = torch.float16, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """C = (A @ B.T) * a_scale[:, None] * b_scale[None, :] (+ bias).

    A [M, K] and B [N, K] are int8 with unit column stride (what quantize_rows
    gives for tokens and for the weight's output channels), the scales float32
    [M] and [N], bias float16 [N]; C is float16 or float32 [M, N].  The sums
    are exact 32-bit integers, for K up to 131071.
    """
    M, K = _dims(A, "A")
    N, _ = _dims(B, "B")
    dev = A.device
    lda, ldb = _matrix(A, "A", M, K, _I8, dev), _matrix(B, "B", N, K, _I8, dev)
    _vector(a_scale, "a_scale", M, torch.float32, dev)
    _vector(b_scale, "b_scale", N, torch.float32, dev)
    if bias is not None:
        _vector(bias, "bias", N, torch.float16, dev)
    ldc = N
    if out is not None:
        ldc = _matrix(out, "out", M, N, _OUT, dev)
        out_dtype = out.dtype
    elif out_dtype not in _DT:
        raise TypeError("out_dtype must be float32 or float16")
    call = _Call(dev, stream)
    C = out if out is not None else call.empty(A, (M, N), out_dtype)
    d = _lib.GemmI8Desc(A.data_ptr(), B.data_ptr(), C.data_ptr(), a_scale.data_ptr(), b_scale.data_ptr(),
                        0 if bias is None else bias.data_ptr(), M, N, K, lda, ldb, ldc, _DT[out_dtype])
    call.run("pax_gemm_i8_ex", ctypes.byref(d))
    return C
