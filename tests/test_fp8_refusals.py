"""CPU checks of the fp8 entry points: sizes are host arithmetic, and bad
arguments are refused before any CUDA call (the pointers here are host
addresses that nothing may follow). No kernel runs."""
import ctypes as C

import numpy as np
import pytest

import fp8_util as F
from u15b200 import _lib as L

A = 1 << 20          # a 16-byte aligned address
I = C.c_int


def ints(*v):
    return (I * len(v))(*v)


@pytest.fixture(scope="module")
def lib():
    return L.lib()


@pytest.mark.parametrize("rows,cols", [(1, 16), (128, 512), (129, 528), (4096, 12288), (0, 128)])
def test_scale_bytes(lib, rows, cols):
    assert lib.u15c_fp8_scale_bytes(rows, cols) == F.scale_bytes(rows, cols)


def test_scale_places_are_a_bijection():
    p = F.places(256, 1024)
    assert sorted(p.ravel()) == list(range(F.scale_bytes(256, 1024)))


def test_workspace_holds_its_parts(lib):
    for rows, h, i in [(1, 16, 128), (333, 4096, 12288)]:
        need = rows * h + rows * i + F.scale_bytes(rows, h) + F.scale_bytes(rows, i)
        assert need <= lib.u15c_ffn_fp8_workspace_bytes(rows, h, i) < need + 1024
    assert lib.u15c_ffn_fp8_workspace_bytes(0, 4096, 12288) == 0


def refused(rc, word):
    assert rc == L.EINVAL and word in L.last_error(), (rc, L.last_error())


def test_quantisers(lib):
    refused(lib.u15c_quant_rows_fp8(None, None, A, A, 4, 128), "null")
    refused(lib.u15c_quant_rows_fp8(None, A, A, A, 4, 24), "multiple of 16")
    refused(lib.u15c_quant_rows_fp8(None, A + 8, A, A, 4, 128), "unaligned")
    refused(lib.u15c_quant_rows_fp8(None, A, A, A, -1, 128), "negative")
    refused(lib.u15c_quant_weight_fp8(None, A, A, A, 0, 4, 128), "out of")
    refused(lib.u15c_quant_weight_fp8(None, A, A, A, 2, 4, 40), "multiple of 16")
    refused(lib.u15c_dequant_fp8(None, A, A, A + 2, 1, 4, 128), "unaligned")
    refused(lib.u15c_dequant_fp8(None, A, A, A, 1, 4, 0), "cols")
    refused(lib.u15c_quant_rows_fp8(None, A, A, A, 1 << 30, 16), "2^30")
    refused(lib.u15c_quant_rows_fp8(None, A, A, A, 4, 1 << 30), "2^30")
    refused(lib.u15c_quant_weight_fp8(None, A, A, A, 1, 1 << 24, 16), "range")
    refused(lib.u15c_dequant_fp8(None, A, A, A, 1, 1 << 30, 16), "range")


def norm(lib, x=A, delta=None, w=A, ne=2, off=None, ex=None, ns=0, out=None, q=A, s=A, rows=4,
         dim=128):
    return lib.u15c_mot_add_rms_norm_quant_fp8(None, x, delta, w, ne, off, ex, ns, out, q, s,
                                               rows, dim, 1e-6)


def test_norm(lib):
    refused(norm(lib, w=None), "null")
    refused(norm(lib, delta=A + 4), "unaligned")
    refused(norm(lib, out=A + 1), "unaligned")
    refused(norm(lib, dim=120), "multiple of 16")
    refused(norm(lib, ne=0), "out of")
    refused(norm(lib, rows=1 << 30), "out of")
    refused(norm(lib, dim=1 << 30), "out of")
    refused(norm(lib, off=ints(0, 2, 3), ex=ints(0, 1), ns=2), "cover")
    refused(norm(lib, off=ints(0, 2, 4), ex=ints(0, 2), ns=2), "expert")


def linear(lib, xq=A, sx=A, wq=A, sw=A, ne=2, off=None, ex=None, ns=0, epi=0, bias=None,
           resid=None, y=A, M=4, K=128, N=256):
    return lib.u15c_mot_linear_fp8(None, xq, sx, wq, sw, ne, off, ex, ns, epi, bias, resid, y, M,
                                   K, N)


def test_linear(lib):
    refused(linear(lib, epi=4), "epilogue")
    refused(linear(lib, epi=-1), "epilogue")
    refused(linear(lib, epi=1), "residual")
    refused(linear(lib, epi=2, N=384), "256")
    refused(linear(lib, epi=2, bias=A), "bias")
    refused(linear(lib, K=100), "multiple of 16")
    refused(linear(lib, N=0), "positive")
    refused(linear(lib, M=-1), "not negative")
    refused(linear(lib, ne=40, N=1 << 27), "2^31")
    for k in ("M", "K", "N"):
        refused(linear(lib, **{k: 1 << 30}), "2^30")
    for k in ("xq", "sx", "wq", "sw", "y"):
        refused(linear(lib, **{k: None}), "null")
    for k in ("xq", "sx", "wq", "sw"):
        refused(linear(lib, **{k: A + 8}), "aligned")
    refused(linear(lib, y=A + 1), "aligned")
    refused(linear(lib, epi=3, y=A + 2), "aligned")
    refused(linear(lib, off=ints(0, 3, 2, 4), ex=ints(0, 1, 0), ns=3), "non-decreasing")
    refused(linear(lib, off=ints(*range(10)), ex=ints(*[0] * 9), ns=9, M=9), "8 routing")


def test_swiglu_and_ffn(lib):
    def swiglu(yq=A, sy=A, N=256):
        return lib.u15c_mot_swiglu_fp8(None, A, A, A, A, 1, None, None, 0, yq, sy, 4, 128, N)
    refused(swiglu(N=128), "256")
    refused(swiglu(sy=None), "null")
    refused(swiglu(yq=A + 4), "aligned")

    def ffn(x=A, delta=None, w=A, guq=A, dq=A, y=A, ws=A, rows=4, h=128, i=256, off=None, ex=None,
            ns=0):
        return lib.u15c_mot_ffn_fp8(None, x, delta, w, guq, A, dq, A, 2, off, ex, ns, y, ws, rows,
                                    h, i, 1e-6)
    refused(ffn(ws=None), "null")
    refused(ffn(ws=A + 8), "unaligned")
    refused(ffn(i=192), "128")
    refused(ffn(h=72), "16")
    refused(ffn(rows=-3), "negative")
    refused(ffn(guq=None), "null")
    refused(ffn(dq=A + 1), "aligned")
    refused(ffn(off=ints(0, 5), ex=ints(0), ns=1), "cover")


def test_no_rows_is_no_work(lib):
    """Zero rows return at once: an empty tensor has no address."""
    assert lib.u15c_quant_rows_fp8(None, None, None, None, 0, 128) == L.OK
    assert lib.u15c_dequant_fp8(None, None, None, None, 1, 0, 128) == L.OK
    assert norm(lib, x=None, q=None, s=None, rows=0) == L.OK
    assert linear(lib, xq=None, sx=None, y=None, M=0) == L.OK
    assert lib.u15c_mot_ffn_fp8(None, None, None, A, A, A, A, A, 1, None, None, 0, None, None, 0,
                                128, 256, 1e-6) == L.OK


def test_rule_restated():
    """The restatement the GPU tests use: rounding, ties, and no saturation."""
    assert list(F.codes(np.array([448.0, -448.0, 0.0, 1.0, 1.0625, 1.1875, 2.0 ** -10,
                                  3 * 2.0 ** -10]))) == [0x7E, 0xFE, 0, 0x38, 0x38, 0x3A, 0, 2]
    a = np.random.default_rng(0).lognormal(0, 20, 20000)
    s = F.scale_byte(a)
    assert (a <= 448 * 2.0 ** (s - 127)).all()
    assert ((a > 448 * 2.0 ** (s - 128)) | (s == 0)).all()
