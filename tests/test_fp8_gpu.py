"""The 8-bit linear layers on the GPU against plain numpy forms in 64 bits."""
import numpy as np
import pytest
import torch

from tests import fp8_ref as ref

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}  # half a step of the type, relative
E4M3 = torch.float8_e4m3fn


def _np(t):
    return t.detach().cpu().double().numpy()


def _rows(T, K, dt, seed, spread=1.0):
    """Rows of sizes of their own, a few large channels, a group of zeros and one far below the others."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g) * (0.3 + torch.rand(T, 1, generator=g)) * spread
    x[:, ::61] *= 9
    if K > 256:
        x[T // 2, 128:256] = 0
        x[T // 3, :128] *= 1e-3
    return x.to(DT[dt])


def _held(T, K, seed, wide=0):
    """Random 8-bit rows with garbage (NaN) behind each row's values: q [T, K], its values."""
    ld = (K + 15) // 16 * 16 + 16 * wide
    g = torch.Generator().manual_seed(seed)
    v = (torch.randn(T, K, generator=g) * 100).clamp(-448, 448).to(E4M3)
    held = torch.full((T, ld), 0x7F, dtype=torch.uint8)
    held[:, :K] = v.view(torch.uint8)
    return held.cuda().view(E4M3)[:, :K], v.double().numpy()


def _scales(shape, seed):
    return torch.rand(*shape, generator=torch.Generator().manual_seed(seed)) * 0.02 + 0.001


# ------------------------------------------------------------------------------------------ quantisers
SIZES = [(1, 1), (1, 128), (3, 7), (16, 4096), (5, 200), (130, 136), (7, 1001), (33, 640), (2, 16500)]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,K", SIZES)
def test_rows_follow_the_definition(dt, T, K):
    from rngd_pd import fp8
    x = _rows(T, K, dt, T + K)
    q, s = fp8.quantize(x.cuda())
    m = ref.limits(_np(x))
    want, scale = ref.quantise(_np(x), ref.spread(m, K))
    assert q.dtype == E4M3 and q.shape == (T, K) and s.shape == (T, ref.groups(K)) and q.stride(0) % 16 == 0
    assert np.array_equal(_np(s), (m.astype(np.float32) / np.float32(448)).astype(np.float64))
    assert np.array_equal(_np(q), want)
    # half a step of e4m3 (2^-4 of the value, 2^-10 of the scale below its normal numbers), two roundings of fp32 before
    err = np.abs(_np(q) * scale - _np(x))
    assert np.all(err <= np.abs(_np(x)) * (2.0 ** -4 + 2.0 ** -22) + 2.0 ** -10 * scale)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (129, 130), (300, 520), (64, 1000), (257, 4096)])
def test_weights_follow_the_definition(dt, N, K):
    from rngd_pd import fp8
    w = _rows(N, K, dt, N * 3 + K, spread=0.02)
    q, s = fp8.quantize_weight(w.cuda())
    m = ref.block_limits(_np(w))
    want, _ = ref.quantise(_np(w), ref.spread_blocks(m, N, K))
    assert q.shape == (N, K) and s.shape == (ref.groups(N), ref.groups(K))
    assert np.array_equal(_np(s), (m.astype(np.float32) / np.float32(448)).astype(np.float64))
    assert np.array_equal(_np(q), want)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_groups_of_zeros_tiny_and_lost_ones(dt):
    from rngd_pd import fp8
    x = torch.zeros(5, 400)
    x[1, 130] = 1e-35                                  # below 2^-100: held to that
    x[2, 5], x[2, 6] = float("nan"), 3.0
    x[3, 300], x[3, 301] = float("inf"), 3.0
    x[4] = -3e38 if dt == "fp32" else 3e38
    x = x.to(DT[dt])
    for f in (fp8.quantize, fp8.quantize_weight):
        q, s = f(x.cuda()) if f is fp8.quantize else f(x[:2].cuda())
        q, s = _np(q), _np(s)
        # 1e-35 * 448 / 2^-100 = 0.00568, 2.9 of e4m3's smallest steps of 2^-9
        assert q[1, 130] == 3 * 2.0 ** -9 and np.all(np.delete(q[:2].ravel(), 530) == 0)
        assert np.all(s[0] == np.float32(2.0 ** -100) / np.float32(448))
    q, s = (_np(t) for t in fp8.quantize(x.cuda()))
    with np.errstate(invalid="ignore"):
        v = q * ref.spread(s, 400)
    assert np.all(np.isnan(v[2, :128])) and np.all(v[2, 128:] == 0)
    assert np.all(np.isnan(v[3, 256:384])) and np.all(np.delete(v[3], range(256, 384)) == 0)  # the group of 128
    assert np.all(np.abs(q[4]) == 448) and np.all(np.isfinite(v[4]))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_strides_and_places_that_no_vector_load_takes(dt):
    """Rows apart, rows that start off 16 bytes, one row given many times: the same numbers."""
    from rngd_pd import fp8
    x = _rows(9, 264, dt, 5)
    want = fp8.quantize(x.cuda())
    room = torch.zeros(9, 300, dtype=DT[dt], device="cuda")
    for at in (0, 1, 8, 13):
        view = room[:, at:at + 264]
        view.copy_(x)
        for a, b in zip(fp8.quantize(view), want):
            assert torch.equal(a.float(), b.float())
        for a, b in zip(fp8.quantize_weight(view), fp8.quantize_weight(x.cuda())):
            assert torch.equal(a.float(), b.float())
    q, s = fp8.quantize(x.cuda()[2:3].expand(6, 264))
    assert torch.equal(q.float(), want[0][2:3].float().expand(6, 264)) and torch.equal(s, want[1][2:3].expand(6, 3))


# ------------------------------------------------------------------------------------------------ norm
def _check_norm(x, w, eps, residual, got):
    q, s, total = got
    h = _np(x)
    if residual is not None:
        want = (x.float() + residual.float()).to(x.dtype)
        assert torch.equal(total.cpu(), want)
        h = _np(want)
    else:
        assert total is None
    y = ref.norm(h, _np(w), eps)
    m = ref.limits(y)
    K = y.shape[1]
    # squares summed by a thread (8 a vector, few of them), 5 shuffles, at most 32 warps: under 100 additions of
    # positive numbers, halved by the root; rsqrt to 2 ulp, three products, the quotient: 64 roundings of 2^-24
    tol = 64 * 2.0 ** -24
    sg = _np(s)
    assert np.all(np.abs(sg - m / 448) <= tol * m / 448)
    wide = ref.spread(sg, K)
    assert np.all(np.abs(_np(q) * wide - y) <= np.abs(y) * (2.0 ** -4 + 2 * tol) + 2.0 ** -10 * wide)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,K", SIZES + [(2, 33001), (3, 40960)])
def test_norm_follows_the_definition(dt, T, K):
    from rngd_pd import fp8
    x, r = _rows(T, K, dt, T + 2 * K), _rows(T, K, dt, T + 3 * K, spread=3.0)
    w = 1 + 0.3 * torch.randn(K, generator=torch.Generator().manual_seed(K))
    for weight in (w, w.to(DT[dt])):
        for res in (None, r):
            got = fp8.rms_norm(x.cuda(), weight.cuda(), 1e-5, None if res is None else res.cuda())
            _check_norm(x, weight, 1e-5, res, got)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("K", [6143, 6145, 12159, 12161, 12287, 12289, 16383, 16384])
def test_norm_at_the_widths_where_its_layout_changes(dt, K):
    """Rows that one, two and no registers' worth of groups hold, the sum's row in shared memory and not."""
    from rngd_pd import fp8
    x, r, w = _rows(3, K, dt, K), _rows(3, K, dt, K + 1, spread=3.0), torch.rand(K) + 0.5
    _check_norm(x, w, 1e-5, r, fp8.rms_norm(x.cuda(), w.cuda(), 1e-5, r.cuda()))


def test_norm_of_zero_rows_and_lost_ones():
    from rngd_pd import fp8
    x = torch.randn(4, 300)
    x[0] = 0
    x[1, 140] = float("nan")
    x[2, 140] = float("inf")
    q, s, _ = fp8.rms_norm(x.cuda(), torch.ones(300).cuda(), 1e-5)
    q, s = _np(q), _np(s)
    assert np.all(q[0] == 0) and np.all(s[0] > 0)
    assert np.all(np.isnan(q[1])) and np.all(np.isnan(s[1]))
    with np.errstate(invalid="ignore"):
        v = q[2] * ref.spread(s[2:3], 300)[0]
    assert np.all(np.isnan(v[128:256])) and np.all(v[:128] == 0) and np.all(v[256:] == 0)
    _check_norm(x[3:], torch.ones(300), 1e-5, None, fp8.rms_norm(x[3:].cuda(), torch.ones(300).cuda(), 1e-5))


def test_norm_of_rows_apart_and_off_16_bytes():
    from rngd_pd import fp8
    x, r = _rows(6, 520, "bf16", 1), _rows(6, 520, "bf16", 2)
    w = torch.rand(521).cuda()
    room = torch.zeros(6, 1100, dtype=torch.bfloat16, device="cuda")
    for at, wo in ((0, 0), (8, 0), (3, 0), (8, 1)):
        a, b = room[:, at:at + 520], room[:, 560 + at:1080 + at]
        a.copy_(x)
        b.copy_(r)
        _check_norm(x, w[wo:wo + 520].cpu(), 1e-6, r, fp8.rms_norm(a, w[wo:wo + 520], 1e-6, b))
        _check_norm(x, w[wo:wo + 520].cpu(), 1e-6, x, fp8.rms_norm(a, w[wo:wo + 520], 1e-6, a))


# --------------------------------------------------------------------------------------------- products
def _tol(y, mag, K, dt):
    """Products are exact.  A group's four steps of 32 are summed in fp32 by the tensor cores (8 roundings of 2^-24 of
    the magnitudes a step at most), then the scales (2), the groups' sum (one each) and the type's half step."""
    return (32 + 2 + ref.groups(K)) * 2.0 ** -24 * mag + HALF[dt] * np.abs(y) + 1e-30


MM = [(1, 1, 1), (1, 128, 128), (2, 3, 17), (16, 256, 512), (5, 130, 1000), (17, 64, 129), (33, 300, 257),
      (64, 128, 640), (65, 129, 384), (100, 520, 144), (128, 128, 2048), (129, 257, 136), (255, 1000, 400),
      (300, 264, 1536), (513, 770, 272), (1, 4096, 4096), (7, 2000, 5000), (1030, 1290, 300), (700, 2304, 900)]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M,N,K", MM)
def test_products_follow_the_definition(dt, M, N, K):
    from rngd_pd import fp8
    a, av = _held(M, K, M + K, wide=1)
    b, bv = _held(N, K, N + 2 * K, wide=0)
    sa, sb = _scales((M, ref.groups(K)), 1), _scales((ref.groups(N), ref.groups(K)), 2) * 0.1
    y, mag = ref.product(av, sa.double().numpy(), bv, sb.double().numpy())
    got = fp8.matmul(a, sa.cuda(), b, sb.cuda(), dtype=DT[dt])
    assert got.dtype == DT[dt] and got.shape == (M, N)
    assert np.all(np.abs(_np(got) - y) <= _tol(y, mag, K, dt))
    add = torch.randn(M, N, generator=torch.Generator().manual_seed(9)).to(DT[dt]) * 5
    y = y + _np(add)
    got = fp8.matmul(a, sa.cuda(), b, sb.cuda(), dtype=DT[dt], add=add.cuda())
    assert np.all(np.abs(_np(got) - y) <= _tol(y, mag + np.abs(_np(add)), K, dt))


# K cut over clusters of 2, 4 and 8, more than 32 groups in one run, several tiles a block
WIDE = [(1, 900, 2100), (16, 4096, 4096), (30, 1000, 4096), (60, 2000, 2048), (128, 1000, 8192), (100, 640, 1536),
        (7, 39000, 4300), (40, 19100, 4352), (16, 60000, 260), (4100, 5000, 300), (2048, 4096, 512)]


@pytest.mark.parametrize("M,N,K", WIDE)
def test_products_cut_and_tiled_in_every_way(M, N, K):
    from rngd_pd import fp8
    ops, y, mag = _simple(M, N, K)
    add = torch.randn(M, N, generator=torch.Generator().manual_seed(9)).bfloat16()
    got = fp8.matmul(*ops, dtype=torch.float32)
    assert np.all(np.abs(_np(got) - y) <= _tol(y, mag, K, "fp32"))
    got = fp8.matmul(*ops, dtype=torch.bfloat16, add=add.cuda())
    y, mag = y + _np(add), mag + np.abs(_np(add))
    assert np.all(np.abs(_np(got) - y) <= _tol(y, mag, K, "bf16"))


def _simple(M, N, K, seed=0):
    a, av = _held(M, K, seed + 1)
    b, bv = _held(N, K, seed + 2)
    sa, sb = _scales((M, ref.groups(K)), seed + 3), _scales((ref.groups(N), ref.groups(K)), seed + 4) * 0.1
    y, mag = ref.product(av, sa.double().numpy(), bv, sb.double().numpy())
    return (a, sa.cuda(), b, sb.cuda()), y, mag


@pytest.mark.parametrize("M,N,K", [(3, 200, 500), (150, 333, 300), (40, 1111, 777), (600, 515, 260)])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_results_lie_where_they_are_asked_for(M, N, K, dt):
    """Rows apart and off 16 bytes; what lies between and behind them stays; add and out may be one tensor."""
    from rngd_pd import fp8
    ops, y, mag = _simple(M, N, K)
    for at, ld in ((0, N), (0, N + 24), (3, N + 9), (8, (N + 31) // 8 * 8)):
        room = torch.full((M + 2, ld), 7.0, dtype=DT[dt], device="cuda")
        flat = room.view(-1)
        out = flat[at:].as_strided((M, N), (ld, 1), at)
        assert fp8.matmul(*ops, dtype=DT[dt], out=out) is out
        assert np.all(np.abs(_np(out) - y) <= _tol(y, mag, K, dt))
        left = torch.ones(flat.shape, dtype=torch.bool, device="cuda")
        left.as_strided((M, N), (ld, 1), at).fill_(False)
        assert torch.all(flat[left] == 7.0)
        fp8.matmul(*ops, dtype=DT[dt], out=out.fill_(2.5), add=out)
        assert np.all(np.abs(_np(out) - (y + 2.5)) <= _tol(y + 2.5, mag + 2.5, K, dt))
    one = torch.randn(1, N, device="cuda").to(DT[dt])
    got = fp8.matmul(*ops, dtype=DT[dt], add=one.expand(M, N))
    assert np.all(np.abs(_np(got) - (y + _np(one))) <= _tol(y + _np(one), mag + np.abs(_np(one)), K, dt))


def test_scales_of_any_strides():
    from rngd_pd import fp8
    for M in (5, 300):
        (a, sa, b, sb), y, mag = _simple(M, 300, 700)
        want = fp8.matmul(a, sa, b, sb)
        for f in (lambda s: s.t().contiguous().t(), lambda s: torch.stack((s, s * 0), 2)[:, :, 0],
                  lambda s: torch.cat((s, s), 1)[:, :s.shape[1]]):
            assert torch.equal(want, fp8.matmul(a, f(sa), b, f(sb)))
        got = fp8.matmul(a, sa[:1].expand(M, -1), b, sb)
        assert torch.equal(got, fp8.matmul(a, sa[:1].expand(M, -1).contiguous(), b, sb))


@pytest.mark.parametrize("M", [2, 20, 90, 400])
def test_lost_groups_spoil_their_rows_alone(M):
    from rngd_pd import fp8
    N, K = 260, 520
    x, w = torch.randn(M, K), torch.randn(N, K) * 0.02
    x[1, 300] = float("nan")
    x[0, 519] = float("inf")
    w[130, 40] = float("nan")
    a, sa = fp8.quantize(x.cuda())
    b, sb = fp8.quantize_weight(w.cuda())
    y = _np(fp8.matmul(a, sa, b, sb, dtype=torch.float32))
    assert np.all(np.isnan(y[:2])) and np.all(np.isnan(y[:, 128:256]))
    assert np.all(np.isfinite(y[2:, :128])) and np.all(np.isfinite(y[2:, 256:]))
    z = fp8.matmul(*fp8.quantize(torch.zeros(M, K).cuda()), b[:128], sb[:1], dtype=torch.float32)
    assert torch.all(z == 0)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 128, 256), (16, 512, 1024), (5, 100, 300), (3, 129, 17), (33, 260, 640),
                                   (70, 384, 200), (128, 256, 128), (200, 330, 1000), (520, 640, 384), (1030, 200, 260),
                                   (260, 1100, 500), (16, 1000, 4096), (30, 1000, 4096), (64, 500, 4096), (3, 19100, 4352),
                                   (2100, 3001, 260), (700, 5000, 140)])
def test_gate_and_up_follow_the_definition(M, N, K):
    from rngd_pd import fp8
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


def test_gate_and_up_of_lost_and_zero_rows():
    from rngd_pd import fp8
    for M in (3, 200):
        x = torch.randn(M, 300)
        x[0] = 0
        x[1, 7] = float("nan")
        w = fp8.quantize_weight(torch.randn(130, 300).cuda())
        q, s = fp8.matmul_swiglu(*fp8.quantize(x.cuda()), *w, *w)
        q, s = _np(q), _np(s)
        assert np.all(q[0] == 0) and np.all(np.isnan(q[1])) and np.all(np.isnan(s[1])) and np.all(np.isfinite(q[2:]))


# ------------------------------------------------------------------------------------ used as in a model
def _mlp(x, r, norm_w, w):
    from rngd_pd import fp8
    q, s, total = fp8.rms_norm(x, norm_w, 1e-5, r)
    h, hs = fp8.matmul_swiglu(q, s, *w["gate"], *w["up"])
    return (q, s, total, h, hs, fp8.matmul(h, hs, *w["down"], dtype=x.dtype, add=total))


@pytest.mark.parametrize("T", [1, 16, 100, 300])
def test_a_layers_mlp(T):
    """Norm, gate and up, down onto the residual: each from what the step before gave."""
    from rngd_pd import fp8
    H, M = 512, 1408
    g = torch.Generator().manual_seed(T)
    w = {n: fp8.quantize_weight((torch.randn(*d, generator=g) * 0.05).bfloat16().cuda())
         for n, d in (("gate", (M, H)), ("up", (M, H)), ("down", (H, M)))}
    x, r = (torch.randn(T, H, generator=g).bfloat16() for _ in (0, 1))
    nw = (1 + 0.1 * torch.randn(H, generator=g)).bfloat16()
    q, s, total, h, hs, y = _mlp(x.cuda(), r.cuda(), nw.cuda(), w)
    _check_norm(x, nw, 1e-5, r, (q, s, total))
    gy, uy = (ref.product(_np(q), _np(s), *map(_np, w[n]))[0] for n in ("gate", "up"))
    act = ref.swiglu(gy, uy)
    wide = ref.spread(_np(hs), M)
    # sums of 4 groups are exact to 2^-18 of their magnitudes, far below half a step of e4m3
    assert np.all(np.abs(_np(h) * wide - act) <= np.abs(act) * (2.0 ** -4 + 2.0 ** -12) + 2.0 ** -10 * wide * 1.01)
    z, mag = ref.product(_np(h), _np(hs), *map(_np, w["down"]))
    z = z + _np(total)
    assert np.all(np.abs(_np(y) - z) <= _tol(z, mag + np.abs(_np(total)), M, "bf16"))


def test_graph_replays_and_other_streams_give_the_same():
    """Captured once, replayed on new inputs, next to eager calls of the same operators on another stream."""
    from rngd_pd import fp8
    H, M = 512, 1408
    w = {n: fp8.quantize_weight((torch.randn(*d) * 0.05).bfloat16().cuda())
         for n, d in (("gate", (M, H)), ("up", (M, H)), ("down", (H, M)))}
    nw = torch.ones(H, dtype=torch.bfloat16, device="cuda")
    for T in (16, 260):
        xs = [torch.randn(2, T, H).bfloat16().cuda() for _ in range(4)]
        want = [[t.float().clone() for t in _mlp(x[0], x[1], nw, w)] for x in xs]
        x = xs[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _mlp(x[0], x[1], nw, w)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _mlp(x[0], x[1], nw, w)
        for i in (1, 2, 3, 1):
            x.copy_(xs[i])
            side.wait_stream(torch.cuda.current_stream())
            graph.replay()
            with torch.cuda.stream(side):
                other = _mlp(xs[0][0], xs[0][1], nw, w)
            torch.cuda.synchronize()
            assert all(torch.equal(a.float(), b) for a, b in zip(got, want[i]))
            assert all(torch.equal(a.float(), b) for a, b in zip(other, want[0]))


def test_weights_written_by_the_launch_before():
    """A weight quantised into memory that held another one, and multiplied with at once, over and over."""
    from rngd_pd import fp8
    g = torch.Generator().manual_seed(4)
    a = fp8.quantize(torch.randn(5, 4096, generator=g).cuda())
    ws = [(torch.randn(2048, 4096, generator=g) * 0.02).cuda() for _ in range(3)]
    want = []
    for w in ws:
        b = fp8.quantize_weight(w)
        torch.cuda.synchronize()
        want.append((fp8.matmul(*a, *b, dtype=torch.float32), fp8.matmul_swiglu(*a, *b, *b)[0].float()))
        torch.cuda.synchronize()
    got = []
    for i in range(60):
        b = fp8.quantize_weight(ws[i % 3])
        got.append((fp8.matmul(*a, *b, dtype=torch.float32), fp8.matmul_swiglu(*a, *b, *b)[0]))
        del b  # the next one gets its memory
    for i, (y, q) in enumerate(got):
        assert torch.equal(y, want[i % 3][0]) and torch.equal(q.float(), want[i % 3][1])


def test_calls_on_two_streams_at_once():
    from rngd_pd import fp8
    cases = [_simple(*d)[0] for d in ((3, 3000, 4096), (300, 1500, 2048), (40, 2000, 1000), (1000, 2000, 512))]
    want = [fp8.matmul(*c, dtype=torch.float32) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            got.append((i * 3 % 4, fp8.matmul(*cases[i * 3 % 4], dtype=torch.float32)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[c]) for c, y in got)


def test_the_same_call_twice_gives_the_same_bits():
    from rngd_pd import fp8
    for M, N, K in ((1, 4096, 4096), (16, 1024, 14336), (60, 4096, 2048), (300, 1500, 4096), (2000, 600, 1000)):
        ops, _, _ = _simple_gpu(M, N, K)
        first = fp8.matmul(*ops, dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(first, fp8.matmul(*ops, dtype=torch.float32))


def _simple_gpu(M, N, K):
    a, sa = _held(M, K, 1)[0], _scales((M, ref.groups(K)), 3).cuda()
    b, sb = _held(N, K, 2)[0], _scales((ref.groups(N), ref.groups(K)), 4).cuda()
    return (a, sa, b, sb), None, None


def test_no_wait_ran_out():
    from rngd_pd import _lib
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


# ------------------------------------------------------------------------------------------- refusals
def test_refusals():
    from rngd_pd import fp8
    x = torch.zeros(4, 256, device="cuda")
    w = torch.ones(256, device="cuda")
    q, s = fp8.quantize(x)
    b, t = fp8.quantize_weight(torch.zeros(130, 256, device="cuda"))
    held = torch.zeros(4, 300, dtype=torch.uint8, device="cuda").view(E4M3)
    bad = [
        lambda: fp8.quantize(x.double()), lambda: fp8.quantize(x[0]), lambda: fp8.quantize(x.t()),
        lambda: fp8.quantize_weight(x.int()), lambda: fp8.quantize_weight(x[:, ::2]),
        lambda: fp8.rms_norm(x, w.half(), 1e-5), lambda: fp8.rms_norm(x, w[:255], 1e-5),
        lambda: fp8.rms_norm(x, w, 1e-5, residual=x.bfloat16()), lambda: fp8.rms_norm(x, w, 1e-5, residual=x[:2]),
        lambda: fp8.rms_norm(x, w.cpu(), 1e-5), lambda: fp8.rms_norm(x, torch.ones(512, device="cuda")[::2], 1e-5),
        lambda: fp8.matmul(x, s, b, t), lambda: fp8.matmul(q, s, b[:, :128], t[:, :1]),
        lambda: fp8.matmul(q, s[:, :1], b, t), lambda: fp8.matmul(q, s, b, t[:1]), lambda: fp8.matmul(q, s.half(), b, t),
        lambda: fp8.matmul(q, s.cpu(), b, t), lambda: fp8.matmul(q, s, b, t, dtype=torch.float64),
        lambda: fp8.matmul(held[:, :256], s, b, t), lambda: fp8.matmul(held[:1, 1:257], s[:1], b, t),
        lambda: fp8.matmul(q[:, ::2], s[:, :1], b[:, :128], t[:, :1]),
        lambda: fp8.matmul(q[:1].expand(4, 256), s, b, t),
        lambda: fp8.matmul(q, s, b, t, add=torch.zeros(4, 130, device="cuda")),
        lambda: fp8.matmul(q, s, b, t, add=torch.zeros(4, 129, device="cuda", dtype=torch.bfloat16)),
        lambda: fp8.matmul(q, s, b, t, out=torch.zeros(4, 130, device="cuda")),
        lambda: fp8.matmul(q, s, b, t, out=torch.zeros(1, 130, device="cuda", dtype=torch.bfloat16).expand(4, 130)),
        lambda: fp8.matmul(q[:, :0], s[:, :0], b[:, :0], t[:, :0]),
        lambda: fp8.matmul_swiglu(q, s, b, t, b[:129], t), lambda: fp8.matmul_swiglu(q, s, b, t, b, t[:, :1]),
        lambda: fp8.matmul_swiglu(q[:, :128], s[:, :1], b, t, b, t),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            raise AssertionError(f"call {i} was not refused")


def test_empty_calls():
    from rngd_pd import fp8
    b, t = fp8.quantize_weight(torch.zeros(130, 256, device="cuda"))
    q, s = fp8.quantize(torch.zeros(0, 256, device="cuda"))
    assert q.shape == (0, 256) and s.shape == (0, 2)
    assert fp8.matmul(q, s, b, t).shape == (0, 130)
    assert fp8.matmul_swiglu(q, s, b, t, b, t)[0].shape == (0, 130)
    q, s, h = fp8.rms_norm(torch.zeros(0, 256, device="cuda"), torch.ones(256, device="cuda"), 1e-5,
                           torch.zeros(0, 256, device="cuda"))
    assert q.shape == h.shape == (0, 256)
    assert fp8.quantize(torch.zeros(3, 0, device="cuda"))[1].shape == (3, 0)
    e, f = fp8.quantize_weight(torch.zeros(0, 256, device="cuda"))
    assert fp8.matmul(*fp8.quantize(torch.zeros(3, 256, device="cuda")), e, f).shape == (3, 0)
