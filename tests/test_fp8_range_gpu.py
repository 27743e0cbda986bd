"""The 8-bit RMS norm of rows whose squares leave fp32: the 64-bit definition has an ordinary answer."""
import numpy as np
import pytest
import torch

from tests.test_fp8_gpu import DT, _check_norm, _np, _rows

pytestmark = pytest.mark.gpu

# rows as whole vectors and not; in registers (one and two runs of them, the sum's row in shared memory or not) and read twice
WIDTHS = [1, 300, 1000, 4096, 6145, 8200, 12287, 16384, 16500, 33001]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("K", WIDTHS)
@pytest.mark.parametrize("size", [1e17, 1e20, 1e30, 2e37])
def test_rows_beyond_the_root_of_fp32(dt, K, size):
    """Their squares times 2^-160 are exact but for a rounding each, so that the tolerance of ordinary rows holds."""
    from rngd_pd import fp8
    x, r = (_rows(4, K, dt, K + i).clamp(-8, 8) for i in (1, 2))
    w = 1 + 0.3 * torch.randn(K, generator=torch.Generator().manual_seed(K))
    x, r = x * size, r * size
    x[3], r[3] = x[3] / size, r[3] / size  # an ordinary row among them
    assert torch.isfinite(x.float() + r.float()).all()
    _check_norm(x, w, 1e-5, None, fp8.rms_norm(x.cuda(), w.cuda(), 1e-5))
    _check_norm(x, w, 1e-5, r, fp8.rms_norm(x.cuda(), w.cuda(), 1e-5, r.cuda()))


@pytest.mark.parametrize("K", WIDTHS)
def test_one_value_of_fp32s_largest(K):
    from rngd_pd import fp8
    x = _rows(3, K, "fp32", K)
    x[0, K // 2] = -3.4e38
    x[1] = 3.4e38
    w = torch.rand(K) + 0.5
    _check_norm(x, w, 1e-6, None, fp8.rms_norm(x.cuda(), w.cuda(), 1e-6))


@pytest.mark.parametrize("K", WIDTHS)
@pytest.mark.parametrize("size", [1e-19, 1e-22, 1e-30])
@pytest.mark.parametrize("eps", [0.0, 1e-42, 1e-10])
def test_rows_below_the_root_of_fp32(K, size, eps):
    """With an eps as small as their squares, tiny rows are rows like others.  (1e-42 is no number of fp32's normal ones:
    it is 714 steps of 2^-149, off by less than one of them.)"""
    from rngd_pd import fp8
    x = (_rows(3, K, "fp32", K).abs() + 0.1) * size
    w = torch.rand(K) + 0.5
    _check_norm(x, w, float(np.float32(eps)), None, fp8.rms_norm(x.cuda(), w.cuda(), eps))


def test_rows_of_zeros_and_lost_ones_stay_what_they_were():
    from rngd_pd import fp8
    for K in (300, 4096, 16384, 33001):
        x = torch.randn(4, K)
        x[0] = 0
        x[1, K // 2] = float("nan")
        x[2] = 1e30
        x[2, K // 2] = -float("inf")
        q, s, _ = fp8.rms_norm(x.cuda(), torch.ones(K).cuda(), 1e-5)
        q, s = _np(q), _np(s)
        assert np.all(q[0] == 0) and np.all(np.isfinite(s[0])) and np.all(np.isnan(q[1]))
        g = K // 2 // 128
        with np.errstate(invalid="ignore"):
            lost = np.isnan(q[2] * np.repeat(s[2], 128)[:K])
        assert np.all(lost[g * 128:g * 128 + 128]) and not lost[:g * 128].any() and not lost[g * 128 + 128:].any()
        q, s, _ = fp8.rms_norm(torch.zeros(2, K).cuda(), torch.ones(K).cuda(), 1e-38)
        assert np.all(_np(q) == 0) and np.all(_np(s) == np.float32(2.0 ** -100) / np.float32(448))
