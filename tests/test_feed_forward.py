"""The feed-forward products' argument checks, on the CPU: nothing here
launches a kernel."""
from __future__ import annotations

import ctypes

import pytest
import torch

import pax_b200
from pax_b200 import _lib

F16, F32, I8 = torch.float16, torch.float32, torch.int8
INVALID, OK = 1, 0


def h(*shape, dtype=F16):
    return torch.zeros(shape, dtype=dtype)


def glu_args(M=4, D=16, F=8):
    return [h(M, D), h(D, F), h(D, F)]


def back_args(M=4, D=16, F=8):
    return [h(M, F), h(M, D), h(D, F), h(D, F), h(M, F), h(M, F)]


def test_cpu_tensors_are_refused():
    for call in (lambda: pax_b200.glu(*glu_args()), lambda: pax_b200.glu_backward(*back_args()),
                 lambda: pax_b200.quantize_rows(h(4, 8)),
                 lambda: pax_b200.gemm_i8(h(4, 16, dtype=I8), h(8, 16, dtype=I8), h(4, dtype=F32), h(8, dtype=F32))):
        with pytest.raises(ValueError, match="CUDA device"):
            call()


@pytest.mark.parametrize("i", range(3))
def test_glu_refuses_types_shapes_and_strides(i):
    a = glu_args()
    for bad, err in ((a[i].float(), TypeError), (a[i][:, :-1], ValueError), (a[i][:-1], ValueError),
                     (a[i].T.contiguous().T, ValueError), (a[i][:1].expand(a[i].shape), ValueError), (a[i][0], ValueError)):
        with pytest.raises(err):
            pax_b200.glu(*[bad if j == i else t for j, t in enumerate(a)])


def test_what_is_not_a_tensor_is_refused():
    for call in (lambda: pax_b200.glu(None, *glu_args()[1:]), lambda: pax_b200.glu(*glu_args()[:2], [1.0]),
                 lambda: pax_b200.glu_backward(*back_args(), dX=3), lambda: pax_b200.quantize_rows("x"),
                 lambda: pax_b200.gemm_i8(h(4, 16, dtype=I8), h(8, 16, dtype=I8), 0.5, h(8, dtype=F32))):
        with pytest.raises((TypeError, ValueError), match="tensor"):
            call()


def test_glu_refuses_half_of_the_kept_products_and_unknown_activations():
    with pytest.raises(ValueError, match="together"):
        pax_b200.glu(*glu_args(), G=h(4, 8))
    with pytest.raises(ValueError):
        pax_b200.glu(*glu_args(), activation="relu")
    with pytest.raises(ValueError):
        pax_b200.glu(*glu_args(), activation=7)
    with pytest.raises(TypeError):
        pax_b200.glu(*glu_args(), out=h(4, 8, dtype=F32))


@pytest.mark.parametrize("i", range(6))
def test_glu_backward_refuses_types_shapes_and_strides(i):
    a = back_args()
    for bad, err in ((a[i].float(), TypeError), (a[i][:, :-1], ValueError), (a[i].T.contiguous().T, ValueError)):
        with pytest.raises(err):
            pax_b200.glu_backward(*[bad if j == i else t for j, t in enumerate(a)])


def test_glu_backward_refuses_contradictions():
    w = lambda dt=F32: h(16, 8, dtype=dt)  # noqa: E731
    for kw, err in (({"dWg": w()}, ValueError), ({"accumulate": True}, ValueError),
                    ({"accumulate": True, "dWg": w(F16), "dWu": w(F16)}, ValueError),
                    ({"dWg": w(), "dWu": w(F16)}, TypeError), ({"dWg": w(), "dWu": w(), "need_dW": False}, ValueError),
                    ({"dX": h(4, 16), "need_dX": False}, ValueError), ({"dX": h(4, 16, dtype=F32)}, TypeError),
                    ({"dW_dtype": torch.bfloat16}, TypeError), ({"dG": h(4, 16)}, ValueError)):
        with pytest.raises(err):
            pax_b200.glu_backward(*back_args(), **kw)


def test_quantize_rows_refusals():
    for kw, err in (({"out": h(4, 8)}, TypeError), ({"out": h(4, 7, dtype=I8)}, ValueError),
                    ({"scale": h(4)}, TypeError), ({"scale": h(5, dtype=F32)}, ValueError),
                    ({"scale": h(8, dtype=F32)[::2]}, ValueError)):
        with pytest.raises(err):
            pax_b200.quantize_rows(h(4, 8), **kw)
    with pytest.raises(TypeError):
        pax_b200.quantize_rows(h(4, 8, dtype=F32))
    with pytest.raises(ValueError):
        pax_b200.quantize_rows(h(8))


def test_gemm_i8_refusals():
    A, B, sa, sb = h(4, 16, dtype=I8), h(8, 16, dtype=I8), h(4, dtype=F32), h(8, dtype=F32)
    for args, kw, err in (((A.half(), B, sa, sb), {}, TypeError), ((A, B[:, :-1], sa, sb), {}, ValueError),
                          ((A, B, sa[:-1], sb), {}, ValueError), ((A, B, sa, sb.half()), {}, TypeError),
                          ((A, B, sa, sb), {"bias": h(4)}, ValueError), ((A, B, sa, sb), {"bias": h(8, dtype=F32)}, TypeError),
                          ((A, B, sa, sb), {"out_dtype": I8}, TypeError), ((A, B, sa, sb), {"out": h(8, 4)}, ValueError)):
        with pytest.raises(err):
            pax_b200.gemm_i8(*args, **kw)


# ------------------------------------------------------------------ C entries
def filled(cls, ptr=64, **kw):
    """A descriptor whose pointers all hold `ptr` (never read: every call here is refused or empty)."""
    d = cls()
    for name, t in cls._fields_:
        if t is ctypes.c_void_p:
            setattr(d, name, ptr)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def call(fn, d):
    return getattr(pax_b200.lib, fn)(ctypes.byref(d), None)


def test_null_descriptors():
    for fn in ("pax_glu_ex", "pax_glu_backward_ex", "pax_gemm_i8_ex"):
        assert getattr(pax_b200.lib, fn)(None, None) == INVALID
        assert pax_b200.last_error() == pax_b200.Status.INVALID


@pytest.mark.parametrize("bad", [{"M": -1}, {"D": -1}, {"F": 1 << 31}, {"act": 3}, {"act": -1}, {"X": None}, {"Wg": None}, {"Wu": None},
                                 {"H": None}, {"G": None}, {"U": None}, {"ldx": 15}, {"ldwg": 7}, {"ldh": -8}, {"X": 65}])
def test_pax_glu_ex_refusals(bad):
    assert call("pax_glu_ex", filled(_lib.GluDesc, **{"M": 4, "D": 16, "F": 8, **bad})) == INVALID


GRAD_PTRS = {"dU": 128, "dX": 192, "dWg": 256, "dWu": 320}


@pytest.mark.parametrize("bad", [{"dG": 128}, {"lddg": 16}, {"dG": 192, "dU": 64, "ldg": 16}, {"M": -1}, {"act": 3}, {"dH": None}, {"X": None}, {"Wg": None}, {"G": None}, {"dG": None}, {"dU": None},
                                 {"dWg": None}, {"dWu": None}, {"dw_dtype": 2}, {"dw_dtype": 1, "accumulate": 1}, {"lddh": 7},
                                 {"lddwg": 7}, {"dWg": 66}])
def test_pax_glu_backward_ex_refusals(bad):
    assert call("pax_glu_backward_ex", filled(_lib.GluGradDesc, **{"M": 4, "D": 16, "F": 8, **GRAD_PTRS, **bad})) == INVALID


@pytest.mark.parametrize("bad", [{"M": -1}, {"K": 131072}, {"A": None}, {"B": None}, {"C": None}, {"a_scale": None}, {"b_scale": None},
                                 {"lda": 15}, {"ldc": 7}, {"c_dtype": 5}, {"C": 66}, {"a_scale": 66}, {"bias": 65}])
def test_pax_gemm_i8_ex_refusals(bad):
    assert call("pax_gemm_i8_ex", filled(_lib.GemmI8Desc, **{"M": 4, "N": 8, "K": 16, **bad})) == INVALID


def test_pax_quantize_rows_refusals():
    f = pax_b200.lib.pax_quantize_rows
    assert f(64, 0, 64, 0, 64, -1, 8, None) == INVALID
    assert f(None, 0, 64, 0, 64, 4, 8, None) == INVALID
    assert f(64, 0, None, 0, 64, 4, 8, None) == INVALID
    assert f(64, 0, 64, 0, None, 4, 8, None) == INVALID
    assert f(64, 7, 64, 0, 64, 4, 8, None) == INVALID
    assert f(65, 0, 64, 0, 64, 4, 8, None) == INVALID


def test_empty_problems_launch_nothing():
    assert call("pax_glu_ex", filled(_lib.GluDesc, ptr=None, M=0, D=16, F=8)) == OK
    assert call("pax_glu_ex", filled(_lib.GluDesc, ptr=None, M=4, D=16, F=0)) == OK
    assert call("pax_glu_backward_ex", filled(_lib.GluGradDesc, ptr=None, M=0, D=16, F=8)) == OK
    assert call("pax_gemm_i8_ex", filled(_lib.GemmI8Desc, ptr=None, M=0, N=8, K=16)) == OK
    assert pax_b200.lib.pax_quantize_rows(None, 0, None, 0, None, 0, 8, None) == OK
