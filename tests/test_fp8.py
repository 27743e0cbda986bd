"""Argument checks of the 8-bit linear layers that need no GPU, and the plain forms they are tested with."""
import ctypes

import numpy as np
import pytest
import torch

from rngd_pd import _lib, fp8
from tests import fp8_ref as ref


def test_tensors_off_the_gpu_are_refused():
    x, w = torch.zeros(4, 256), torch.ones(256)
    q, s = torch.zeros(4, 256, dtype=torch.float8_e4m3fn), torch.zeros(4, 2)
    for f in (lambda: fp8.quantize(x), lambda: fp8.quantize_weight(x), lambda: fp8.rms_norm(x, w, 1e-5),
              lambda: fp8.matmul(q, s, q, s[:1]), lambda: fp8.matmul_swiglu(q, s, q, s[:1], q, s[:1])):
        with pytest.raises(ValueError):
            f()


def test_c_entries_refuse_bad_arguments():
    """Refused on the host, with a message, before anything is launched."""
    lib, p = _lib.lib, ctypes.c_void_p(4096)
    odd = ctypes.c_void_p(4097)
    st2 = (ctypes.c_int64 * 2)(2, 1)

    def mm(a=p, lda=256, sa=p, b=p, ldb=256, M=4, N=4, K=256, add=None, y=p, ldy=4, dt=0, ss=st2):
        return lib.rngd_f8_matmul(a, lda, sa, ss, b, ldb, p, ss, M, N, K, add, 4, y, ldy, dt, None)

    def sw(q=p, ldq=16, K=256, N=4):
        return lib.rngd_f8_swiglu(p, 256, p, st2, p, 256, p, st2, p, 256, p, st2, 4, N, K, q, ldq, p, None)

    bad = [
        (lambda: lib.rngd_f8_rows(p, 3, 8, 1, 8, p, 16, p, None), "data type 3"),
        (lambda: lib.rngd_f8_rows(p, 0, 8, 2, 8, p, 8, p, None), "16 bytes"),
        (lambda: lib.rngd_f8_rows(p, 0, 8, 2, 32, p, 16, p, None), "16 bytes"),
        (lambda: lib.rngd_f8_rows(odd, 0, 8, 1, 8, p, 16, p, None), "misaligned"),
        (lambda: lib.rngd_f8_rows(p, 0, 8, -1, 8, p, 16, p, None), "-1 rows"),
        (lambda: lib.rngd_f8_rows(p, 0, 8, 1, 8, p, 16, None, None), "null"),
        (lambda: lib.rngd_f8_weight(p, 0, 8, 2, 8, odd, 16, p, None), "16 bytes"),
        (lambda: lib.rngd_f8_weight(p, -1, 8, 2, 8, p, 16, p, None), "data type"),
        (lambda: lib.rngd_f8_rms_norm(p, 8, None, 0, p, 0, 1, 1, 8, 1e-5, None, 0, p, 16, p, None), "weights of data type 1"),
        (lambda: lib.rngd_f8_rms_norm(p, 8, p, 8, p, 0, 0, 1, 8, 1e-5, None, 0, p, 16, p, None), "place for the sum"),
        (lambda: lib.rngd_f8_rms_norm(p, 8, p, 8, p, 0, 0, 1, 8, 1e-5, p, 8, p, 16, p, None), "place of its own"),
        (lambda: lib.rngd_f8_rms_norm(p, 8, None, 0, None, 0, 0, 1, 8, 1e-5, None, 0, p, 16, p, None), "null"),
        (lambda: mm(dt=5), "data type 5"), (lambda: mm(K=0), "x 0"), (lambda: mm(M=-1), "-1 x"),
        (lambda: mm(K=2 ** 31 - 2), "too much"), (lambda: mm(N=2 ** 31 - 2), "too much"), (lambda: sw(K=2 ** 30 + 1), "too much"),
        (lambda: lib.rngd_f8_rows(p, 0, 8, 1, 2 ** 30 + 1, p, 16, p, None), "1073741825"),
        (lambda: lib.rngd_f8_rows(p, 0, 8, 2 ** 33, 8, p, 16, p, None), "8589934592 rows"), (lambda: mm(a=odd), "misaligned"), (lambda: mm(lda=250), "250 apart"),
        (lambda: mm(ldb=128), "128 apart"), (lambda: mm(b=None), "null"), (lambda: mm(sa=None), "null"),
        (lambda: mm(y=None), "null"), (lambda: mm(y=odd), "misaligned"), (lambda: mm(add=odd), "misaligned"),
        (lambda: mm(ldy=3), "lie on one another"), (lambda: mm(ss=None), "null"),
        (lambda: sw(q=odd), "16 bytes"), (lambda: sw(ldq=8), "16 bytes"), (lambda: sw(K=0), "x 0"),
        (lambda: sw(N=-4), "-4"), (lambda: sw(q=None), "null"),
    ]
    for f, words in bad:
        assert f() == _lib.RNGD_ERR_ARG, words
        assert words in _lib.last_error(), (words, _lib.last_error())


def test_empty_calls_do_nothing():
    lib, p = _lib.lib, ctypes.c_void_p(4096)
    st2 = (ctypes.c_int64 * 2)(2, 1)
    assert lib.rngd_f8_rows(None, 0, 0, 0, 8, None, 0, None, None) == 0
    assert lib.rngd_f8_weight(None, 0, 0, 4, 0, None, 0, None, None) == 0
    assert lib.rngd_f8_rms_norm(None, 0, None, 0, None, 0, 0, 0, 8, 1e-5, None, 0, None, 0, None, None) == 0
    assert lib.rngd_f8_matmul(None, 0, None, st2, p, 256, p, st2, 0, 4, 256, None, 0, None, 0, 0, None) == 0


def test_plain_forms_on_small_cases():
    assert ref.e4m3([448.0, 500.0, 0.0, 17.0, 19.0, 18.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, -240.0]).tolist() == \
        [448, 448, 0, 16, 20, 18, 2.0 ** -9, 0, 2.0 ** -8, -240]
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    codes = codes[~codes.isnan()].numpy()
    assert np.array_equal(ref.e4m3(codes), codes)
    x = np.linspace(-450, 450, 9001)
    near = codes[np.abs(x[:, None] - codes).argmin(1)]
    got = ref.e4m3(x)
    assert np.all(np.abs(got - x) <= np.abs(near - x))
    y = np.arange(300.0).reshape(1, 300) - 280
    assert ref.limits(y).tolist() == [[280, 152, 24]]
    assert ref.block_limits(np.arange(260.0).reshape(130, 2)).tolist() == [[255.0], [259.0]]
    a, b = np.ones((2, 130)), np.ones((129, 130))
    sa, sb = np.array([[1.0, 2.0], [3.0, 4.0]]), np.array([[1.0, 1.0], [0.5, 2.0]])
    y, mag = ref.product(a, sa, b, sb)
    assert y[0, 0] == 128 + 4 and y[1, 128] == 128 * 1.5 + 2 * 8 and np.array_equal(y, mag)


def _huge(shape, dtype=torch.bfloat16, ld=None):
    """A tensor on the GPU by its shape and type alone: nothing is allocated, any launch would fail here."""
    return torch.empty_strided(shape, (ld or shape[1], 1), dtype=dtype, device="cuda")


@pytest.mark.parametrize("n", [2 ** 30 + 1, 2 ** 32, 2 ** 32 + 8])
def test_widths_that_32_bits_do_not_hold_are_refused(n):
    """Not cut to their lowest 32 bits: 2^32 values a row would pass for none, 2^32 + 8 for eight."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    e4m3, f32, G = torch.float8_e4m3fn, torch.float32, -(-n // 128)
    with FakeTensorMode(allow_non_fake_inputs=True):
        x, w, v = _huge((1, n)), _huge((2, n)), torch.empty(n, dtype=torch.bfloat16, device="cuda")
        q, s = _huge((1, n), e4m3, n + -n % 16), _huge((1, G), f32)
        for f in (lambda: fp8.quantize(x), lambda: fp8.quantize_weight(w), lambda: fp8.rms_norm(x, v, 1e-5),
                  lambda: fp8.rms_norm(x, v, 1e-5, residual=x), lambda: fp8.matmul(q, s, q, s),
                  lambda: fp8.matmul_swiglu(q, s, q, s, q, s)):
            with pytest.raises(ValueError, match=str(n)):
                f()


@pytest.mark.parametrize("n", [2 ** 31 - 255, 2 ** 32, 2 ** 32 + 8])
def test_rows_that_32_bits_do_not_hold_are_refused(n):
    from torch._subclasses.fake_tensor import FakeTensorMode
    e4m3, f32, NB = torch.float8_e4m3fn, torch.float32, -(-n // 128)
    with FakeTensorMode(allow_non_fake_inputs=True):
        w = _huge((n, 1))
        many, one, block = (_huge((n, 1), e4m3, 16), _huge((n, 1), f32)), (_huge((1, 1), e4m3, 16), _huge((1, 1), f32)), \
            _huge((NB, 1), f32)
        for f in (lambda: fp8.quantize_weight(w), lambda: fp8.matmul(*many, *one), lambda: fp8.matmul(*one, many[0], block),
                  lambda: fp8.matmul_swiglu(*many, *one, *one),
                  lambda: fp8.matmul_swiglu(*one, many[0], block, many[0], block)):
            with pytest.raises(ValueError, match=str(n)):
                f()


def test_the_greatest_sizes_pass_the_checks():
    """2^30 values a row and 2^31 - 256 rows."""
    dev, e4m3, f32 = torch.device("cuda", 0), torch.float8_e4m3fn, torch.float32
    n = 2 ** 30
    assert fp8._source("x", (1, n), (n, 1), torch.bfloat16, dev)[2:4] == (1, n)
    n = 2 ** 31 - 256
    assert fp8._operand("b", ((n, 1), (16, 1), e4m3, dev), ((n // 128, 1), (1, 1), f32, dev), True)[0] == n


def _tile_rows(M, N, K, gated=0):
    n = ctypes.c_int(0)
    assert _lib.lib.rngd_f8_tile_rows(M, N, K, gated, ctypes.byref(n)) == 0
    return n.value


def test_few_rows_take_the_kernel_for_few_rows():
    """Also where K is too short to be cut, so that either kernel has one wave."""
    for N in (1, 128, 896, 4864, 18944):
        for K in (1, 128, 512, 896, 1100, 4096):
            assert [_tile_rows(M, N, K) for M in (1, 16, 17, 32, 33, 64)] == [16, 16, 32, 32, 64, 64]
            assert [_tile_rows(M, N, K, 1) for M in (1, 16)] == [16, 16]
    assert _tile_rows(128, 4096, 4096) == 128 and _tile_rows(33, 14336, 4096, 1) == 64
    assert _tile_rows(333, 6144, 4096) == 256 and _tile_rows(8192, 4096, 14336) == 256
    n = ctypes.c_int(0)
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 2 ** 30 + 1)):
        assert _lib.lib.rngd_f8_tile_rows(*bad, 0, ctypes.byref(n)) == _lib.RNGD_ERR_ARG
    assert _lib.lib.rngd_f8_tile_rows(1, 1, 1, 0, None) == _lib.RNGD_ERR_ARG and "null" in _lib.last_error()


def test_status_entries_refuse_null():
    assert _lib.lib.rngd_f8_status(None, 1) == _lib.RNGD_ERR_ARG and "null" in _lib.last_error()
