"""Plain numpy forms, in 64 bits, of the 8-bit linear layers."""
import numpy as np


def e4m3(x):
    """Round to the nearest number of e4m3 (ties to even), held to 448."""
    x = np.asarray(x, np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.clip(np.floor(np.log2(np.abs(x))), -6, 8)
    step = 2.0 ** (np.where(np.isfinite(e), e, -6) - 3)
    return np.clip(np.rint(x / step) * step, -448, 448)


def groups(n):
    return -(-n // 128)


def limits(y):
    """m = max(amax, 2^-100) of each group of 128 along the last dimension (NaN where it holds one)."""
    K = y.shape[-1]
    a = np.abs(y)
    m = np.stack([a[..., g * 128:(g + 1) * 128].max(-1) for g in range(groups(K))], -1)
    return np.maximum(m, 2.0 ** -100)


def block_limits(w):
    """The same of each block of 128 x 128."""
    m = limits(w)
    return np.stack([m[n * 128:(n + 1) * 128].max(0) for n in range(groups(w.shape[0]))])


def spread(s, K):
    """Scales of groups, one for each value."""
    return np.repeat(s, 128, -1)[..., :K]


def spread_blocks(s, N, K):
    return spread(np.repeat(s, 128, 0)[:N], K)


def quantise(y, m):
    """What fp32 makes of values y (exact in fp32) under limits m of their shape: one quotient, one product."""
    y, m = y.astype(np.float32), m.astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        return e4m3((y * (np.float32(448) / m)).astype(np.float64)), m / np.float32(448)


def norm(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def product(a, sa, b, sb):
    """(y, sum of the magnitudes) of rows a [M, K], sa [M, G] and a weight b [N, K], sb [NB, G]."""
    x, w = a * spread(sa, a.shape[1]), b * spread_blocks(sb, *b.shape)
    return x @ w.T, np.abs(x) @ np.abs(w).T


def swiglu(g, u):
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g)) * u
