"""Linear layers in 8 bits: rows and weights held in e4m3 with fp32 scales, and the products of such operands.

The reference's projections are bf16 (src/rngd_pd/kernels/decode_batch.py:73-109).  Held in 8 bits, weights take
half the bytes, which is what a decode step's time goes by, and the tensor cores run at twice the rate, which is
what a prompt's goes by.

  rows    float8_e4m3fn [T, K], scale float32 [T, G]: one for each 128 values from the left, G = ceil(K / 128)
  weight  float8_e4m3fn [N, K], scale float32 [ceil(N / 128), G]: one for each block of 128 x 128

With m = max(amax, 2^-100) of a group, scale = m / 448 and a value x is held as e4m3(x * (448 / m)).  A group with a
NaN or an infinity reads as NaN.  Rows start on 16 bytes: where K is no multiple of 16, the tensors that quantize,
quantize_weight, rms_norm and matmul_swiglu return are views of wider ones, and operands that a caller brings have to
be laid out like that too.

Everything lives on the tensors' GPU; calls are queued on the current stream and wait for nothing, so they can
be captured into a CUDA graph.  As with torch's own operators, a tensor made on another stream has to be
ordered before the call by the caller (and kept alive with record_stream).  Nothing falls back to the CPU.
"""
import torch

from rngd_pd import _lib

GROUP = 128  # values that share a scale

_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_E4M3 = torch.float8_e4m3fn
_F32 = torch.float32
_INT_MAX = 2 ** 31 - GROUP
_check = _lib.check
_rows, _weight, _norm = _lib.lib.rngd_f8_rows, _lib.lib.rngd_f8_weight, _lib.lib.rngd_f8_rms_norm
_matmul, _swiglu = _lib.lib.rngd_f8_matmul, _lib.lib.rngd_f8_swiglu


def _elsewhere(dev):
    """Whether another GPU than the tensors' is current (the calls below then start over with theirs)."""
    return dev.index != torch.cuda.current_device()


def _matrix(name, x, dev=None, shape=None, dtype=None):
    """Row stride of a matrix of bfloat16, float16 or float32 whose rows are contiguous."""
    if x.dim() != 2 or x.dtype not in _DT or not x.is_cuda or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError(f"{name} must be a CUDA matrix of bfloat16, float16 or float32 with contiguous rows, got "
                         f"{tuple(x.shape)} {x.dtype} strides {x.stride()} on {x.device}")
    if dev is not None and (x.device != dev or x.shape != shape or x.dtype is not dtype):
        raise ValueError(f"{name} must be {tuple(shape)} {dtype} on {dev}, got {tuple(x.shape)} {x.dtype} on {x.device}")
    return x.stride(0)


def _held(rows, K, dev):
    """Room for rows of K 8-bit values that start on 16 bytes, and the bytes between them."""
    if K % 16 == 0:
        return torch.empty((rows, K), dtype=_E4M3, device=dev), K
    wide = (K + 15) // 16 * 16
    return torch.empty((rows, wide), dtype=_E4M3, device=dev)[:, :K], wide


def _operand(name, q, scale, blocks, dev=None, K=None):
    """(pointer, row stride, pointer of the scales, their strides) of 8-bit rows or, with `blocks`, of a weight."""
    if q.dim() != 2 or q.dtype is not _E4M3 or not q.is_cuda or (dev is not None and q.device != dev):
        raise ValueError(f"{name} must be a float8_e4m3fn matrix on {dev or 'a GPU'}, got {tuple(q.shape)} {q.dtype} on "
                         f"{q.device}")
    n, k = q.shape
    if K is not None and k != K:
        raise ValueError(f"{name} {tuple(q.shape)}: rows of {K} values are needed")
    ld = q.stride(0)
    if (k > 1 and q.stride(1) != 1) or q.data_ptr() % 16 or (n > 1 and (ld % 16 or ld < k)):
        raise ValueError(f"{name} {tuple(q.shape)} strides {q.stride()}: rows must be contiguous, start on 16 bytes and "
                         "not overlap")
    want = ((n + GROUP - 1) // GROUP if blocks else n, (k + GROUP - 1) // GROUP)
    if scale.shape != want or scale.dtype is not _F32 or scale.device != q.device:
        raise ValueError(f"{name}'s scale must be float32 {want} on {q.device}, got {tuple(scale.shape)} {scale.dtype} on "
                         f"{scale.device}")
    return q.data_ptr(), ld, scale.data_ptr(), _lib.i64_array(scale.stride())


def quantize(x):
    """Rows in 8 bits: x [T, K] bfloat16, float16 or float32 (rows contiguous) -> (q [T, K], scale [T, G])."""
    ld = _matrix("x", x)
    dev = x.device
    T, K = x.shape
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return quantize(x)
    q, ldq = _held(T, K, dev)
    scale = torch.empty((T, (K + GROUP - 1) // GROUP), dtype=_F32, device=dev)
    _check(_rows(x.data_ptr(), _DT[x.dtype], ld, T, K, q.data_ptr(), ldq, scale.data_ptr(), _lib.raw_stream(dev.index)))
    return q, scale


def quantize_weight(w):
    """A weight in 8 bits: w [N, K] bfloat16, float16 or float32 (rows contiguous) -> (q [N, K], scale
    [ceil(N / 128), G])."""
    ld = _matrix("w", w)
    dev = w.device
    N, K = w.shape
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return quantize_weight(w)
    q, ldq = _held(N, K, dev)
    scale = torch.empty(((N + GROUP - 1) // GROUP, (K + GROUP - 1) // GROUP), dtype=_F32, device=dev)
    _check(_weight(w.data_ptr(), _DT[w.dtype], ld, N, K, q.data_ptr(), ldq, scale.data_ptr(), _lib.raw_stream(dev.index)))
    return q, scale


def rms_norm(x, weight, eps, residual=None):
    """The RMS norm of x + residual in 8 bits, and that sum: (q [T, K], scale [T, G], total).

    x, residual: [T, K] of one type (rows contiguous); weight: [K] of that type or float32.  total = x + residual
    rounded to their type, the residual stream as it goes on (None without a residual); the norm is of the rounded
    sum, total / sqrt(mean(total^2) + eps) * weight, worked out in fp32 and rounded to 8 bits alone."""
    ld = _matrix("x", x)
    dev, dt = x.device, x.dtype
    T, K = x.shape
    if weight.shape != (K,) or (weight.dtype is not dt and weight.dtype is not _F32) or weight.device != dev or \
            not weight.is_contiguous():
        raise ValueError(f"weight must be a contiguous {dt} or float32 [{K}] tensor on {dev}, got {tuple(weight.shape)} "
                         f"{weight.dtype} on {weight.device}")
    if residual is not None:
        ldr = _matrix("residual", residual, dev, x.shape, dt)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return rms_norm(x, weight, eps, residual)
    q, ldq = _held(T, K, dev)
    scale = torch.empty((T, (K + GROUP - 1) // GROUP), dtype=_F32, device=dev)
    if residual is None:
        total, r, t, ldr = None, None, None, 0
    else:
        total = torch.empty((T, K), dtype=dt, device=dev)
        r, t = residual.data_ptr(), total.data_ptr()
    _check(_norm(x.data_ptr(), ld, r, ldr, weight.data_ptr(), _DT[dt], _DT[weight.dtype], T, K, eps, t, K,
                 q.data_ptr(), ldq, scale.data_ptr(), _lib.raw_stream(dev.index)))
    return q, scale, total


def matmul(a, a_scale, b, b_scale, dtype=torch.bfloat16, add=None, out=None):
    """a b^T of 8-bit rows a [M, K] and an 8-bit weight b [N, K], plus `add`: [M, N] of `dtype`, in `out` where given.

    Sums are held in fp32, `add` ([M, N] of `dtype`, rows contiguous) is added there, and the result is rounded once
    to `dtype` (bfloat16, float16 or float32).  out: [M, N] of `dtype`, rows contiguous; it may be `add` itself, but
    must not overlap it in part, nor the operands."""
    ap, lda, sp, ss = _operand("a", a, a_scale, False)
    dev = a.device
    M, K = a.shape
    bp, ldb, tp, ts = _operand("b", b, b_scale, True, dev, K)
    N = b.shape[0]
    if dtype not in _DT:
        raise ValueError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    if K == 0 or K > _INT_MAX:
        raise ValueError(f"a {tuple(a.shape)}: nothing to sum, or too much")
    p, lda_ = (None, 0) if add is None else (add.data_ptr(), _matrix("add", add, dev, (M, N), dtype))
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return matmul(a, a_scale, b, b_scale, dtype, add, out)
    if out is None:
        out, ldo = torch.empty((M, N), dtype=dtype, device=dev), N
    else:
        ldo = _matrix("out", out, dev, (M, N), dtype)
        if M > 1 and ldo < N:
            raise ValueError(f"out {tuple(out.shape)} strides {out.stride()}: rows lie on one another")
    _check(_matmul(ap, lda, sp, ss, bp, ldb, tp, ts, M, N, K, p, lda_, out.data_ptr(), ldo, _DT[dtype],
                   _lib.raw_stream(dev.index)))
    return out


def matmul_swiglu(a, a_scale, gate, gate_scale, up, up_scale):
    """silu(a gate^T) * (a up^T) of 8-bit rows a [M, K] and 8-bit weights gate, up [N, K], in 8 bits again:
    (q [M, N], scale [M, ceil(N / 128)]), what the down projection takes.  Nothing is rounded in between."""
    ap, lda, sp, ss = _operand("a", a, a_scale, False)
    dev = a.device
    M, K = a.shape
    gp, ldg, tp, ts = _operand("gate", gate, gate_scale, True, dev, K)
    up_, ldu, vp, vs = _operand("up", up, up_scale, True, dev, K)
    N = gate.shape[0]
    if up.shape[0] != N:
        raise ValueError(f"gate {tuple(gate.shape)} and up {tuple(up.shape)} must be of one shape")
    if K == 0 or K > _INT_MAX:
        raise ValueError(f"a {tuple(a.shape)}: nothing to sum, or too much")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return matmul_swiglu(a, a_scale, gate, gate_scale, up, up_scale)
    q, ldq = _held(M, N, dev)
    scale = torch.empty((M, (N + GROUP - 1) // GROUP), dtype=_F32, device=dev)
    _check(_swiglu(ap, lda, sp, ss, gp, ldg, tp, ts, up_, ldu, vp, vs, M, N, K, q.data_ptr(), ldq, scale.data_ptr(),
                   _lib.raw_stream(dev.index)))
    return q, scale
