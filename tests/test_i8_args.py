"""Refusals of the int8 operators (llamini_b200.h): every bad argument fails
with a message before any device work, so this runs without a GPU."""
from __future__ import annotations

import pytest

NAN = float("nan")
D = 0x10000                       # a made-up address: no call below gets as far as reading it


def _weights(L, type=8, blocks=D, rows=4, cols=64, q=D, ld=64, scale=D):
    return L.llamini_weights_i8_device(type, blocks, rows, cols, q, ld, scale, None)


def _norm(L, type=0, x=D, ldx=64, r=None, ldr=64, s=None, lds=64, w=D, eps=1e-5, rows=4, cols=64, q=D, ldq=64, scale=D):
    return L.llamini_rms_norm_i8_device(type, x, ldx, r, ldr, s, lds, w, eps, rows, cols, q, ldq, scale, None)


def _glu(L, type=0, g=D, ldg=64, u=D, ldu=64, act=0, rows=4, cols=64, q=D, ldq=64, scale=D):
    return L.llamini_glu_i8_device(type, g, ldg, u, ldu, act, rows, cols, q, ldq, scale, None)


def _gemm(L, a=D, lda=64, sa=D, rows=4, w=D, ldw=64, sw=D, n=8, cols=64, bias=None, out_type=0, out=D, ldo=8):
    return L.llamini_gemm_i8_device(a, lda, sa, rows, w, ldw, sw, n, cols, bias, out_type, out, ldo, None)


BAD = [
    (_weights, dict(type=7), "unsupported type 7"),
    (_weights, dict(type=30), "unsupported type 30"),
    (_weights, dict(cols=48, ld=48), "not whole blocks"),
    (_weights, dict(type=12, cols=128, ld=128), "not whole blocks"),
    (_weights, dict(cols=0), "0 columns"),
    (_weights, dict(cols=131104, ld=131104), "131104 columns"),
    (_weights, dict(ld=63), "pitch 63"),
    (_weights, dict(rows=1 << 31), "rows"),
    (_weights, dict(blocks=None), "null pointer"),
    (_weights, dict(q=None), "null pointer"),
    (_weights, dict(scale=None), "null pointer"),
    (_weights, dict(blocks=D + 1), "not aligned"),
    (_weights, dict(type=0, blocks=D + 2), "not aligned"),
    (_weights, dict(scale=D + 2), "not aligned"),
    (_norm, dict(type=8), "element type 8"),
    (_norm, dict(type=2), "element type 2"),
    (_norm, dict(cols=0), "0 columns"),
    (_norm, dict(cols=131072, ldx=131072, ldq=131072), "131072 columns"),
    (_norm, dict(ldx=63), "pitch 63 of x"),
    (_norm, dict(r=D, ldr=63), "pitch 63 of the residual"),
    (_norm, dict(s=D + 4096, lds=63), "pitch 63 of the sum"),
    (_norm, dict(ldq=63), "pitch 63 of q"),
    (_norm, dict(ldx=(1 << 40) + 1), "of x"),
    (_norm, dict(eps=-1.0), "eps"),
    (_norm, dict(eps=NAN), "eps"),
    (_norm, dict(s=D, lds=65), "needs that input's pitch"),
    (_norm, dict(r=D + 4096, s=D + 4096, lds=65), "needs that input's pitch"),
    (_norm, dict(x=None), "null pointer"),
    (_norm, dict(w=None), "null pointer"),
    (_norm, dict(q=None), "null pointer"),
    (_norm, dict(scale=None), "null pointer"),
    (_norm, dict(x=D + 2), "not aligned"),
    (_norm, dict(type=1, x=D + 1), "not aligned"),
    (_norm, dict(type=30, r=D + 1), "not aligned"),
    (_norm, dict(w=D + 2), "not aligned"),
    (_glu, dict(type=3), "element type 3"),
    (_glu, dict(act=3), "unknown activation 3"),
    (_glu, dict(cols=0), "0 columns"),
    (_glu, dict(ldg=63), "pitch 63 of gate"),
    (_glu, dict(ldu=63), "pitch 63 of up"),
    (_glu, dict(ldq=63), "pitch 63 of q"),
    (_glu, dict(g=None), "null pointer"),
    (_glu, dict(q=None), "null pointer"),
    (_glu, dict(u=D + 2), "not aligned"),
    (_glu, dict(rows=0x80000000), "rows"),
    (_gemm, dict(out_type=8), "output type 8"),
    (_gemm, dict(cols=0), "0 columns"),
    (_gemm, dict(cols=131072, lda=131072, ldw=131072), "131072 columns"),
    (_gemm, dict(lda=63), "pitch"),
    (_gemm, dict(ldw=63), "pitch"),
    (_gemm, dict(ldo=7), "pitch"),
    (_gemm, dict(rows=0x80000000), "outputs"),
    (_gemm, dict(a=None), "null pointer"),
    (_gemm, dict(sa=None), "null pointer"),
    (_gemm, dict(w=None), "null pointer"),
    (_gemm, dict(sw=None), "null pointer"),
    (_gemm, dict(out=None), "null pointer"),
    (_gemm, dict(sa=D + 2), "not aligned"),
    (_gemm, dict(sw=D + 1), "not aligned"),
    (_gemm, dict(bias=D + 2), "not aligned"),
    (_gemm, dict(out=D + 2), "not aligned"),
    (_gemm, dict(out_type=1, out=D + 1), "not aligned"),
]


@pytest.mark.parametrize("i", range(len(BAD)))
def test_bad_arguments_are_refused(lm, i):
    fn, kw, message = BAD[i]
    L = lm.lib()
    L.llamini_clear_error()
    assert fn(L, **kw) == -1
    assert message in lm.last_error()
    L.llamini_clear_error()


@pytest.mark.parametrize("fn", [_weights, _norm, _glu, _gemm])
def test_no_rows_is_no_work(lm, fn):
    L = lm.lib()
    L.llamini_clear_error()
    assert fn(L, rows=0) == 0
    assert lm.last_error() == ""
    if fn is _gemm:
        assert fn(L, n=0, ldo=0) == 0


@pytest.mark.parametrize("fn", [_weights, _norm, _glu, _gemm])
def test_memory_that_no_kernel_may_use_is_refused(lm, fn):
    """Addresses that are not the current device's memory: refused by the
    library with a GPU, and without one there is no CPU path."""
    L = lm.lib()
    L.llamini_clear_error()
    assert fn(L) == -1
    want = "not memory of the current device" if L.llamini_device_count() > 0 else "no usable CUDA device"
    assert want in lm.last_error()
    L.llamini_clear_error()


def test_status_without_a_device(lm):
    L = lm.lib()
    if L.llamini_device_count() > 0:
        pytest.skip("a GPU is present")
    assert L.llamini_i8_status(None) == -1
    assert "no usable CUDA device" in lm.last_error()
    L.llamini_clear_error()


def test_wait_bound_is_limited(lm):
    L = lm.lib()
    L.llamini_clear_error()
    assert L.llamini_set_i8_wait_ns(60_000_000_001) == -1
    assert "at most 60000000000" in lm.last_error()
    L.llamini_clear_error()
    assert L.llamini_set_i8_wait_ns(60_000_000_000) == 0
    assert L.llamini_set_i8_wait_ns(2_000_000_000) == 0
