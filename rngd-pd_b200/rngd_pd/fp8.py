"""Linear layers in 8 bits: rows and weights held in e4m3 with fp32 scales, and the products of such operands.

The reference's projections are bf16 (src/rngd_pd/kernels/decode_batch.py:73-109).  Held in 8 bits, weights take
half the bytes, which is what a decode step's time goes by, and the tensor cores run at twice the rate, which is
what a prompt's goes by.

  rows    float8_e4m3fn [T, K], scale float32 [T, G]: one for each 128 values from the left, G = ceil(K / 128)
  weight  float8_e4m3fn [N, K], scale float32 [ceil(N / 128), G]: one for each block of 128 x 128

With m = max(amax, 2^-100) of a group, scale = m / 448 and a value x is held as e4m3(x * (448 / m)).  A group with a
NaN or an infinity reads as NaN.  The products hold a row's scale times a block's in fp32: but for groups of zeros the two
should multiply to one of its normal numbers (magnitudes of a and b to between 1e-32 and 1e43).  Rows start on 16 bytes:
where K is no multiple of 16, the tensors that quantize, quantize_weight, rms_norm and matmul_swiglu return are views of
wider ones, and operands that a caller brings have to be laid out like that too.

Everything lives on the tensors' GPU; calls are queued on the current stream and wait for nothing, so they can
be captured into a CUDA graph.  As with torch's own operators, a tensor made on another stream has to be
ordered before the call by the caller (and kept alive with record_stream).  Nothing falls back to the CPU.

The products' kernels wait for their own copies, 2 s at most.  Where such a wait runs out the call's results are NaN and
device_status() says so, whatever the engines' own status (BeamDecodeEngine.result) reads and clears.
"""
import ctypes
import functools

import torch

from rngd_pd import _lib

GROUP = 128  # values that share a scale

_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_E4M3 = torch.float8_e4m3fn
_F32 = torch.float32
_empty = torch.empty_strided  # half of torch.empty's time on the host
# what the library counts with 32 bits; ctypes would cut greater numbers to their lowest 32
_MOST_K = 2 ** 30
_MOST_ROWS = 2 ** 31 - 256  # of a weight, and of a product's operands
_check, _stream = _lib.check, torch._C._cuda_getCurrentRawStream
_current = torch._C._cuda_getDevice  # the calls start over with the tensors' GPU where another is current
_rows, _weight, _norm = _lib.lib.rngd_f8_rows, _lib.lib.rngd_f8_weight, _lib.lib.rngd_f8_rms_norm
_matmul, _swiglu = _lib.lib.rngd_f8_matmul, _lib.lib.rngd_f8_swiglu


# The operators are called hundreds of times a step, and small ones take less time on the GPU than a call's checks on
# the host.  So what depends on shapes, strides and types alone is checked once for each set of them.

def _key(t):
    return t.shape, t.stride(), t.dtype, t.device


def _matrix(name, shape, strides, dtype, dev):
    """Row stride of a matrix of bfloat16, float16 or float32 whose rows are contiguous."""
    if len(shape) != 2 or dtype not in _DT or dev.type != "cuda" or (shape[1] > 1 and strides[1] != 1):
        raise ValueError(f"{name} must be a CUDA matrix of bfloat16, float16 or float32 with contiguous rows, got "
                         f"{tuple(shape)} {dtype} strides {strides} on {dev}")
    return strides[0]


def _like(name, shape, strides, dtype, dev, want, want_dtype, want_dev):
    """Row stride of a matrix that has to be of this shape and type."""
    if shape != want or dtype is not want_dtype or dev != want_dev:
        raise ValueError(f"{name} must be {tuple(want)} {want_dtype} on {want_dev}, got {tuple(shape)} {dtype} on {dev}")
    return _matrix(name, shape, strides, dtype, dev)


def _groups(n):
    return (n + GROUP - 1) // GROUP


@functools.lru_cache(maxsize=4096)
def _source(name, shape, strides, dtype, dev):
    """What the quantisers take from their input: (row stride, type's number, sizes, strides of the 8-bit rows and of
    the scales, their number a row).  name: "w" of a weight, whose rows are counted with 32 bits too."""
    ld = _matrix(name, shape, strides, dtype, dev)
    T, K = shape
    if K > _MOST_K or (name == "w" and T > _MOST_ROWS):
        raise ValueError(f"{name} {tuple(shape)} is too much: {_MOST_ROWS} rows of a weight, {_MOST_K} values a row")
    return ld, _DT[dtype], T, K, ((K + 15) // 16 * 16, 1), (_groups(K), 1), _groups(K)


def _operand(name, q, scale, blocks):
    """(n, k, row stride, strides of the scales) of 8-bit rows or, with `blocks`, of a weight, given as _key()s."""
    shape, strides, dtype, dev = q
    if len(shape) != 2 or dtype is not _E4M3 or dev.type != "cuda":
        raise ValueError(f"{name} must be a float8_e4m3fn CUDA matrix, got {tuple(shape)} {dtype} on {dev}")
    n, k = shape
    ld = strides[0]
    if (k > 1 and strides[1] != 1) or (n > 1 and (ld % 16 or ld < k)):
        raise ValueError(f"{name} {tuple(shape)} strides {strides}: rows must be contiguous, start on 16 bytes and not "
                         "overlap")
    if k == 0 or k > _MOST_K or n > _MOST_ROWS:
        raise ValueError(f"{name} {tuple(shape)}: nothing to sum, or too much ({_MOST_ROWS} rows of {_MOST_K} values)")
    want = (_groups(n) if blocks else n, _groups(k))
    if scale[0] != want or scale[2] is not _F32 or scale[3] != dev:
        raise ValueError(f"{name}'s scale must be float32 {want} on {dev}, got {tuple(scale[0])} {scale[2]} on {scale[3]}")
    return n, k, ld, _lib.i64_array(scale[1])


def _against(name, a, b, b_scale):
    """_operand() of a weight that rows `a` (a _key()) are multiplied with."""
    n, k, ld, st = _operand(name, b, b_scale, True)
    if k != a[0][1] or b[3] != a[3]:
        raise ValueError(f"{name} {tuple(b[0])} on {b[3]}: rows of {a[0][1]} values on {a[3]} are needed")
    return n, ld, st


@functools.lru_cache(maxsize=4096)
def _product(dtype, a, a_scale, b, b_scale, add, out):
    M, K, lda, ast = _operand("a", a, a_scale, False)
    N, ldb, bst = _against("b", a, b, b_scale)
    if dtype not in _DT:
        raise ValueError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    dev, shape = a[3], (M, N)
    ldadd = 0 if add is None else _like("add", *add, shape, dtype, dev)
    ldo = N if out is None else _like("out", *out, shape, dtype, dev)
    if M > 1 and ldo < N:
        raise ValueError(f"out {shape} strides {out[1]}: rows lie on one another")
    return M, N, K, lda, ast, ldb, bst, ldadd, ldo, _DT[dtype], shape, (N, 1)


@functools.lru_cache(maxsize=4096)
def _gated(a, a_scale, gate, gate_scale, up, up_scale):
    M, K, lda, ast = _operand("a", a, a_scale, False)
    N, ldg, gst = _against("gate", a, gate, gate_scale)
    n, ldu, ust = _against("up", a, up, up_scale)
    if n != N:
        raise ValueError(f"gate {tuple(gate[0])} and up {tuple(up[0])} must be of one shape")
    return M, N, K, lda, ast, ldg, gst, ldu, ust, (M, N), ((N + 15) // 16 * 16, 1), (M, _groups(N)), (_groups(N), 1)


def _start(name, q):
    p = q.data_ptr()
    if p % 16:
        raise ValueError(f"{name} must start on 16 bytes")
    return p


def quantize(x):
    """Rows in 8 bits: x [T, K] bfloat16, float16 or float32 (rows contiguous) -> (q [T, K], scale [T, G])."""
    dev = x.device
    ld, dt, T, K, st, s_st, G = _source("x", x.shape, x.stride(), x.dtype, dev)
    if dev.index != _current():
        with torch.cuda.device(dev):
            return quantize(x)
    q = _empty((T, K), st, dtype=_E4M3, device=dev)
    scale = _empty((T, G), s_st, dtype=_F32, device=dev)
    _check(_rows(x.data_ptr(), dt, ld, T, K, q.data_ptr(), st[0], scale.data_ptr(), _stream(dev.index)))
    return q, scale


def quantize_weight(w):
    """A weight in 8 bits: w [N, K] bfloat16, float16 or float32 (rows contiguous) -> (q [N, K], scale
    [ceil(N / 128), G])."""
    dev = w.device
    ld, dt, N, K, st, s_st, G = _source("w", w.shape, w.stride(), w.dtype, dev)
    if dev.index != _current():
        with torch.cuda.device(dev):
            return quantize_weight(w)
    q = _empty((N, K), st, dtype=_E4M3, device=dev)
    scale = _empty((_groups(N), G), s_st, dtype=_F32, device=dev)
    _check(_weight(w.data_ptr(), dt, ld, N, K, q.data_ptr(), st[0], scale.data_ptr(), _stream(dev.index)))
    return q, scale


def rms_norm(x, weight, eps, residual=None):
    """The RMS norm of x + residual in 8 bits, and that sum: (q [T, K], scale [T, G], total).

    x, residual: [T, K] of one type (rows contiguous); weight: [K] of that type or float32.  total = x + residual
    rounded to their type, the residual stream as it goes on (None without a residual); the norm is of the rounded
    sum, total / sqrt(mean(total^2) + eps) * weight, worked out in fp32 (rows whose squares leave its range by values times
    a power of two) and rounded to 8 bits alone."""
    dev, dtype = x.device, x.dtype
    ld, dt, T, K, st, s_st, G = _source("x", x.shape, x.stride(), dtype, dev)
    wt = weight.dtype
    if weight.shape != (K,) or (wt is not dtype and wt is not _F32) or weight.device != dev or not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous {dtype} or float32 [{K}] tensor on {dev}, got "
                         f"{tuple(weight.shape)} {wt} on {weight.device}")
    if residual is not None:
        if residual.shape != x.shape or residual.dtype is not dtype or residual.device != dev:
            raise ValueError(f"residual must be {tuple(x.shape)} {dtype} on {dev}, got {tuple(residual.shape)} "
                             f"{residual.dtype} on {residual.device}")
        ldr = _source("residual", x.shape, residual.stride(), dtype, dev)[0]
    if dev.index != _current():
        with torch.cuda.device(dev):
            return rms_norm(x, weight, eps, residual)
    q = _empty((T, K), st, dtype=_E4M3, device=dev)
    scale = _empty((T, G), s_st, dtype=_F32, device=dev)
    if residual is None:
        total, r, t, ldr = None, None, None, 0
    else:
        total = _empty((T, K), (K, 1), dtype=dtype, device=dev)
        r, t = residual.data_ptr(), total.data_ptr()
    _check(_norm(x.data_ptr(), ld, r, ldr, weight.data_ptr(), dt, _DT[wt], T, K, eps, t, K, q.data_ptr(), st[0],
                 scale.data_ptr(), _stream(dev.index)))
    return q, scale, total


def matmul(a, a_scale, b, b_scale, dtype=torch.bfloat16, add=None, out=None):
    """a b^T of 8-bit rows a [M, K] and an 8-bit weight b [N, K], plus `add`: [M, N] of `dtype`, in `out` where given.

    Sums are held in fp32, `add` ([M, N] of `dtype`, rows contiguous) is added there, and the result is rounded once
    to `dtype` (bfloat16, float16 or float32).  out: [M, N] of `dtype`, rows contiguous; it may be `add` itself, but
    must not overlap it in part, nor the operands."""
    M, N, K, lda, ast, ldb, bst, ldadd, ldo, dt, shape, st = _product(
        dtype, _key(a), _key(a_scale), _key(b), _key(b_scale), None if add is None else _key(add),
        None if out is None else _key(out))
    ap, bp, dev = _start("a", a), _start("b", b), a.device
    if dev.index != _current():
        with torch.cuda.device(dev):
            return matmul(a, a_scale, b, b_scale, dtype, add, out)
    if out is None:
        out = _empty(shape, st, dtype=dtype, device=dev)
    _check(_matmul(ap, lda, a_scale.data_ptr(), ast, bp, ldb, b_scale.data_ptr(), bst, M, N, K,
                   None if add is None else add.data_ptr(), ldadd, out.data_ptr(), ldo, dt, _stream(dev.index)))
    return out


def matmul_swiglu(a, a_scale, gate, gate_scale, up, up_scale):
    """silu(a gate^T) * (a up^T) of 8-bit rows a [M, K] and 8-bit weights gate, up [N, K], in 8 bits again:
    (q [M, N], scale [M, ceil(N / 128)]), what the down projection takes.  Nothing is rounded in between."""
    M, N, K, lda, ast, ldg, gst, ldu, ust, shape, st, s_shape, s_st = _gated(
        _key(a), _key(a_scale), _key(gate), _key(gate_scale), _key(up), _key(up_scale))
    ap, gp, up_, dev = _start("a", a), _start("gate", gate), _start("up", up), a.device
    if dev.index != _current():
        with torch.cuda.device(dev):
            return matmul_swiglu(a, a_scale, gate, gate_scale, up, up_scale)
    q = _empty(shape, st, dtype=_E4M3, device=dev)
    scale = _empty(s_shape, s_st, dtype=_F32, device=dev)
    _check(_swiglu(ap, lda, a_scale.data_ptr(), ast, gp, ldg, gate_scale.data_ptr(), gst, up_, ldu, up_scale.data_ptr(),
                   ust, M, N, K, q.data_ptr(), st[0], scale.data_ptr(), _stream(dev.index)))
    return q, scale


def device_status(reset=True):
    """Status word of the products' device waits on the current GPU: 0, or the code of the first one that ran out since it
    was last cleared (reset: by this call).  Waits for the GPU; not for use under graph capture."""
    st = ctypes.c_int(0)
    torch.cuda.synchronize()
    _lib.call("rngd_f8_status", ctypes.byref(st), 1 if reset else 0)
    return st.value
