"""The 8-bit products' kernel for few rows, each of its tiles: results, where they go, scales, lost groups.  Every case
asks the library which kernel it takes, so that none comes to test the other one."""
import ctypes

import numpy as np
import pytest
import torch

from tests import fp8_ref as ref
from tests.test_fp8_gpu import DT, _held, _np, _scales, _simple, _tol

pytestmark = pytest.mark.gpu

# a's rows, the weight's, K -> rows of a tile: K in one run and cut over clusters of 2, 4 and 8, a last run and a last tile
# that are not full, K that ends inside a group, one value short of a group and of a vector, several tiles of a's rows
CASES = [(1, 1, 1, 16), (3, 333, 17, 16), (16, 1111, 500, 16), (2, 130, 1100, 16), (5, 1000, 2303, 16), (13, 333, 4100, 16),
         (7, 37001, 1025, 16), (17, 129, 300, 32), (32, 1111, 896, 32), (20, 333, 1100, 32), (31, 515, 4100, 32),
         (33, 300, 777, 64), (64, 640, 128, 64), (40, 1111, 1100, 64), (63, 333, 4099, 64),
         (65, 333, 1100, 128), (90, 1111, 2100, 128), (128, 257, 4100, 128), (200, 4095, 4096, 128), (129, 515, 1100, 128)]
GATED = [(1, 1, 1, 16), (2, 130, 500, 16), (16, 1111, 1100, 16), (3, 333, 4100, 16), (9, 19001, 1025, 16), (20, 333, 1100, 32),
         (32, 1111, 4100, 32), (25, 140, 2303, 32), (40, 333, 1100, 64), (64, 1001, 4100, 64), (90, 260, 2100, 64), (150, 333, 4099, 64)]


def _takes(M, N, K, rows, gated=0):
    from rngd_pd import _lib
    n = ctypes.c_int(0)
    _lib.call("rngd_f8_tile_rows", M, N, K, gated, ctypes.byref(n))
    assert n.value == rows, (M, N, K, n.value)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M,N,K,rows", CASES)
def test_products(M, N, K, rows, dt):
    from rngd_pd import fp8
    _takes(M, N, K, rows)
    ops, y, mag = _simple(M, N, K, seed=M)
    got = fp8.matmul(*ops, dtype=DT[dt])
    assert np.all(np.abs(_np(got) - y) <= _tol(y, mag, K, dt))
    add = torch.randn(M, N, generator=torch.Generator().manual_seed(9)).to(DT[dt]) * 5
    y, mag = y + _np(add), mag + np.abs(_np(add))
    got = fp8.matmul(*ops, dtype=DT[dt], add=add.cuda())
    assert np.all(np.abs(_np(got) - y) <= _tol(y, mag, K, dt))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M,N,K,rows", [c for c in CASES if c[1] < 5000 and c[0] > 1])
def test_results_lie_where_they_are_asked_for(M, N, K, rows, dt):
    """Rows apart and off 16 bytes; what lies between and behind them stays; add and out may be one tensor."""
    from rngd_pd import fp8
    _takes(M, N, K, rows)
    ops, y, mag = _simple(M, N, K)
    for at, ld in ((0, N), (0, N + 24), (3, N + 9), (8, (N + 31) // 8 * 8)):
        room = torch.full((M + 2, ld), 7.0, dtype=DT[dt], device="cuda")
        flat = room.view(-1)
        out = flat.as_strided((M, N), (ld, 1), at)
        left = torch.ones(flat.shape, dtype=torch.bool, device="cuda")
        left.as_strided((M, N), (ld, 1), at).fill_(False)
        assert fp8.matmul(*ops, dtype=DT[dt], out=out) is out
        assert np.all(np.abs(_np(out) - y) <= _tol(y, mag, K, dt))
        assert torch.all(flat[left] == 7.0)
        fp8.matmul(*ops, dtype=DT[dt], out=out.fill_(2.5), add=out)
        assert np.all(np.abs(_np(out) - (y + 2.5)) <= _tol(y + 2.5, mag + 2.5, K, dt))
        assert torch.all(flat[left] == 7.0)
    for one in (torch.randn(1, N).to(DT[dt]).cuda().expand(M, N), torch.randn(M, N + 5).to(DT[dt]).cuda()[:, 5:]):
        got = fp8.matmul(*ops, dtype=DT[dt], add=one)
        z = y + _np(one)
        assert np.all(np.abs(_np(got) - z) <= _tol(z, mag + np.abs(_np(one)), K, dt))


@pytest.mark.parametrize("M,N,K,rows", [(5, 300, 700, 16), (5, 300, 4300, 16), (30, 333, 1100, 32), (50, 333, 4300, 64),
                                        (100, 300, 2100, 128)])
def test_scales_of_any_strides(M, N, K, rows):
    from rngd_pd import fp8
    _takes(M, N, K, rows)
    (a, sa, b, sb), y, mag = _simple(M, N, K)
    want = fp8.matmul(a, sa, b, sb)
    assert np.all(np.abs(_np(want) - y) <= _tol(y, mag, K, "bf16"))
    for f in (lambda s: s.t().contiguous().t(), lambda s: torch.stack((s, s * 0), 2)[:, :, 0],
              lambda s: torch.cat((s, s), 1)[:, :s.shape[1]]):
        assert torch.equal(want, fp8.matmul(a, f(sa), b, f(sb)))
    got = fp8.matmul(a, sa[:1].expand(M, -1), b, sb)
    assert torch.equal(got, fp8.matmul(a, sa[:1].expand(M, -1).contiguous(), b, sb))


@pytest.mark.parametrize("M,K,rows", [(2, 520, 16), (16, 4100, 16), (20, 1100, 32), (40, 777, 64), (60, 2100, 64), (90, 1100, 128)])
def test_lost_groups_spoil_their_rows_alone(M, K, rows):
    from rngd_pd import fp8
    N = 260
    _takes(M, N, K, rows)
    x, w = torch.randn(M, K), torch.randn(N, K) * 0.02
    x[1, 300] = float("nan")
    x[0, K - 1] = float("inf")
    w[130, 40] = float("nan")
    a, sa = fp8.quantize(x.cuda())
    b, sb = fp8.quantize_weight(w.cuda())
    y = _np(fp8.matmul(a, sa, b, sb, dtype=torch.float32))
    assert np.all(np.isnan(y[:2])) and np.all(np.isnan(y[:, 128:256]))
    assert np.all(np.isfinite(y[2:, :128])) and np.all(np.isfinite(y[2:, 256:]))
    z = fp8.matmul(*fp8.quantize(torch.zeros(M, K).cuda()), b[:128], sb[:1], dtype=torch.float32)
    assert torch.all(z == 0)


@pytest.mark.parametrize("M,N,K,rows", GATED)
def test_gate_and_up(M, N, K, rows):
    from rngd_pd import fp8
    _takes(M, N, K, rows, 1)
    a, av = _held(M, K, M)
    g, gv = _held(N, K, N)
    u, uv = _held(N, K, K, wide=2)
    G, NB = ref.groups(K), ref.groups(N)
    sa, sg, su = _scales((M, G), 1), _scales((NB, G), 2) / K ** 0.5 * 0.1, _scales((NB, G), 3) * 0.1
    q, s = fp8.matmul_swiglu(a, sa.cuda(), g, sg.cuda(), u, su.cuda())
    assert q.shape == (M, N) and s.shape == (M, NB) and q.stride(0) % 16 == 0
    gy, gm = ref.product(av, sa.double().numpy(), gv, sg.double().numpy())
    uy, um = ref.product(av, sa.double().numpy(), uv, su.double().numpy())
    y = ref.swiglu(gy, uy)
    # the errors of both sums through silu (its slope is under 1.1, silu(g) / g under 1), then exp to 2 + 1.2 |g| ulp,
    # quotient, product and the scale's: 8 more
    eg, eu = _tol(0 * gy, gm, K, "fp32"), _tol(0 * uy, um, K, "fp32")
    err = 1.1 * eg * np.abs(uy) + np.abs(gy) * eu + 1.1 * eg * eu + (8 + 2 * np.abs(gy)) * 2.0 ** -23 * np.abs(y)
    m = ref.limits(y)
    sn, wide = _np(s), ref.spread(_np(s), N)
    most = ref.limits(err + 2.0 ** -22 * np.abs(y))
    assert np.all(np.abs(sn * 448 - m) <= most)
    slack = err + (ref.spread(most / m, N) + 2.0 ** -22) * np.abs(y)
    assert np.all(np.abs(_np(q) * wide - y) <= (np.abs(y) + slack) * 2.0 ** -4 + slack + 2.0 ** -10 * wide)
    # scales of other strides, and bytes behind a row's values: the same
    t = lambda x: x.t().contiguous().t()
    again = fp8.matmul_swiglu(a, t(sa.cuda()), g, t(sg.cuda()), u, t(su.cuda()))
    assert torch.equal(q.float(), again[0].float()) and torch.equal(s, again[1])


@pytest.mark.parametrize("M,K,rows", [(3, 300, 16), (16, 4100, 16), (20, 1100, 32), (40, 2100, 64)])
def test_gate_and_up_of_lost_and_zero_rows(M, K, rows):
    from rngd_pd import fp8
    _takes(M, 130, K, rows, 1)
    x = torch.randn(M, K)
    x[0] = 0
    x[1, 7] = float("nan")
    x[2, K - 1] = float("inf")
    w = torch.randn(130, K)
    q, s = fp8.matmul_swiglu(*fp8.quantize(x.cuda()), *fp8.quantize_weight(w.cuda()), *fp8.quantize_weight(w.cuda()))
    q, s = _np(q), _np(s)
    assert np.all(q[0] == 0) and np.all(np.isnan(q[1:3])) and np.all(np.isnan(s[1:3])) and np.all(np.isfinite(q[3:]))
    w[5, 9] = float("nan")  # the weight's first 128 rows are lost, and with them the result's first group of every row
    q, s = fp8.matmul_swiglu(*fp8.quantize(x.cuda()), *fp8.quantize_weight(w.cuda()), *fp8.quantize_weight(torch.ones(130, K).cuda()))
    q, s = _np(q), _np(s)
    assert np.all(np.isnan(s[:, 0])) and np.all(np.isnan(q[3:, :128])) and np.all(np.isfinite(q[3:, 128:]))


@pytest.mark.parametrize("M,N,K,rows", [(16, 128, 500, 16), (30, 515, 896, 32), (64, 333, 260, 64)])
def test_uncut_products_have_the_pairs_bits(M, N, K, rows):
    """Either kernel adds the groups in their order: rows by themselves are the rows of a call of many."""
    from rngd_pd import fp8
    _takes(M, N, K, rows)
    _takes(2000, N, K, 256)
    (a, sa, b, sb), _, _ = _simple(2000, N, K)
    many = fp8.matmul(a, sa, b, sb, dtype=torch.float32)
    assert torch.equal(fp8.matmul(a[:M], sa[:M], b, sb, dtype=torch.float32), many[:M])
