"""Refusals of the product with an epilogue and of the activations' backward, without a GPU."""
import ctypes

import pytest

from easyllm_amd import _lib

A = 1 << 20  # an aligned address nobody reads


def refused(code, text, name, *args):
    _lib.load()
    with pytest.raises(RuntimeError, match=r"\(%d\).*%s" % (code, text)):
        _lib.call(name, *args)


def call(a=A, b=A, c=A, M=16, N=64, K=64, lda=64, ldb=64, ldc=64, bias=None, residual=None, pre=None, ldr=64, ldp=64, act=1, ws=None, size=0, epilogue=True):
    e = ctypes.byref(_lib.Epilogue(bias, residual, pre, ldr, ldp, act)) if epilogue else None
    return "ezl_gemm_bf16_epilogue", a, b, c, M, N, K, lda, ldb, ldc, e, ws, size, None


def test_the_product_refuses():
    for args in (dict(M=-1), dict(N=-8), dict(K=0), dict(K=-64), dict(epilogue=False)):
        refused(-1, "negative size, empty reduction or no epilogue", *call(**args))
    for act in (-1, 3):
        refused(-1, "act must be", *call(act=act))
    for args in (dict(a=None), dict(b=None), dict(c=None)):
        refused(-1, "null", *call(**args))
    for args in (dict(N=60, ldc=64), dict(ldc=68), dict(residual=A, ldr=68), dict(pre=A, ldp=68), dict(ldc=1 << 21), dict(residual=A, ldr=1 << 21), dict(pre=A, ldp=1 << 21)):
        refused(-2, "multiples of 8", *call(**args))
    for args in (dict(ldc=56), dict(lda=56), dict(ldb=56), dict(residual=A, ldr=56), dict(pre=A, ldp=56)):
        refused(-1, "leading dimension", *call(**args))
    for args in (dict(a=A + 2), dict(b=A + 8), dict(c=A + 4), dict(bias=A + 2), dict(residual=A + 8), dict(pre=A + 2), dict(ws=A + 8, size=64)):
        refused(-1, "aligned", *call(**args))
    refused(-2, "contiguous extent of A", *call(K=60))
    assert _lib.call(*call(M=0)) is None and _lib.call(*call(N=0)) is None


def test_the_activations_backward_refuses():
    def bwd(act=1, dy=A, pre=A, out=A, g=None, ws=None, size=0, rows=2, n=64):
        return "ezl_act_bwd", act, dy, pre, out, g, ws, size, rows, n, None
    for act in (0, 3):
        refused(-1, "act must be", *bwd(act=act))
    for args in (dict(n=60), dict(n=0), dict(rows=-1), dict(rows=2 ** 31)):
        refused(-2, "n % 8", *bwd(**args))
    for args in (dict(dy=None), dict(pre=None), dict(out=None)):
        refused(-1, "null", *bwd(**args))
    for args in (dict(dy=A + 2), dict(pre=A + 8), dict(out=A + 4)):
        refused(-1, "aligned", *bwd(**args))
    g = ctypes.byref(_lib.LayerGrad(A, None, 0))
    refused(-1, "workspace", *bwd(g=g))
    refused(-1, "workspace", *bwd(g=g, ws=A, size=_lib.column_sum_workspace_bytes(2, 64) - 1))
