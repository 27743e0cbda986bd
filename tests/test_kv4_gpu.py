"""The paged 4-bit KV cache on the GPU against plain numpy forms in 64 bits: what is stored and read back,
the attention over it (masks, lengths, types, layouts), and the pages of its sequences."""
import numpy as np
import pytest
import torch

from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -10, "fp32": 2.0 ** -23}  # one rounding to the type, and its half again


def _np(t):
    return t.detach().cpu().double().numpy()


def _pool_of(L, P, NKV, HD, fill=255):
    """A pool whose bytes are all `fill`: 255 makes every scale a NaN."""
    return torch.full((L, P, NKV, 4, 20 * HD), fill, dtype=torch.uint8, device="cuda")


def _cache(B, width, NKV, HD, lens, seed, spread=1.0, P=None):
    """Pages with lens[b] positions stored, everything else NaN: pool [P, ...], table, K, V as stored."""
    from rngd_pd import kv4
    g = torch.Generator().manual_seed(seed)
    P = P or B * width + 3
    table = torch.randperm(P, generator=g)[:B * width].view(B, width).to(torch.int32).cuda()
    pool = _pool_of(1, P, NKV, HD)
    T = max(max(lens), 1)
    k = torch.randn(1, B, T, NKV, HD, generator=g) * spread + torch.randn(1, 1, 1, NKV, HD, generator=g)
    v = torch.randn(1, B, T, NKV, HD, generator=g) * spread
    kv4.store(pool, table, torch.zeros(B, dtype=torch.int32, device="cuda"), k.cuda(), v.cuda(),
              count=torch.tensor(lens, dtype=torch.int32).cuda())
    return pool[0], table


# ------------------------------------------------------------------------------------ store and load
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("HD,NKV,L,T", [(128, 3, 2, 37), (64, 2, 1, 70), (64, 1, 3, 1), (128, 8, 1, 1)])
def test_store_and_load_follow_the_definition(dt, HD, NKV, L, T):
    from rngd_pd import kv4
    g = torch.Generator().manual_seed(HD + T)
    B, width = 4, 4
    P = B * width + 2
    table = torch.randperm(P, generator=g)[:B * width].view(B, width).to(torch.int32)
    table[2, 1] = -1                       # no page for positions 64..127 of stream 2
    table[3, 0] = P + 7                    # an id that is none
    start = torch.tensor([0, 13, 50, 61], dtype=torch.int32)
    count = torch.tensor([T, max(T - 5, 0), T, T], dtype=torch.int32)
    k = (torch.randn(L, B, T, NKV, HD, generator=g) * 3 + 1).to(DT[dt])
    v = torch.randn(L, B, T, NKV, HD, generator=g).to(DT[dt])
    pool = _pool_of(L, P, NKV, HD, fill=171)
    before = pool.clone()
    kv4.store(pool, table.cuda(), start.cuda(), k.cuda(), v.cuda(), count=count.cuda())
    got = kv4.load(pool, table.cuda(), start.cuda(), T, count=count.cuda(), dtype=torch.float32)
    pos = start.view(B, 1) + torch.arange(T)
    page = table.gather(1, (pos // 64).long())
    there = ((torch.arange(T) < count.view(B, 1)) & (page >= 0) & (page < P)).numpy()
    for x, y in ((k, got[0]), (v, got[1])):
        u, s, c, tie = ref.encode(_np(x))
        want = ref.values(u, s, c) * there[None, :, :, None, None]
        y = _np(y)
        # fp32 decides a code as 64 bits do, but for quotients within 2^-16 of a tie; there either neighbour will do
        keep = there[None, :, :, None, None]
        step, base = np.repeat(s, 32, -1) * keep, np.repeat(np.abs(c), 32, -1) * keep
        assert np.all((y == want) | ((tie < 2.0 ** -16) & (np.abs(y - want) <= 1.01 * step)))
        # half a step, and at the ends of the range the roundings of s (31 times), c and the value to 11 bits
        assert np.all(np.abs(y - _np(x) * keep) <= step * (0.5 + 31 * 2.0 ** -11) + 2.0 ** -11 * (base + np.abs(y)) + 1e-7)
    # the pages hold that in the documented layout, and nothing else was touched
    K, V = ref.decode_pool(pool.cpu().numpy())
    mine = torch.zeros(L, P, 64, dtype=torch.bool)
    for b in range(B):
        for t in range(T):
            if there[b, t]:
                pg, o = int(page[b, t]), int(pos[b, t]) % 64
                mine[:, pg, o] = True
                for l in range(L):
                    assert np.array_equal(K[l, pg, :, o], _np(got[0])[l, b, t])
                    assert np.array_equal(V[l, pg, :, o], _np(got[1])[l, b, t])
    K0, V0 = ref.decode_pool(before.cpu().numpy())
    keep = ~mine.numpy()
    for a, o in ((K, K0), (V, V0)):
        assert np.array_equal(a.swapaxes(2, 3)[keep], o.swapaxes(2, 3)[keep], equal_nan=True)


def test_load_types_and_default_count():
    from rngd_pd import kv4
    pool, table = _cache(2, 2, 2, 64, [70, 70], 3)
    start = torch.tensor([3, 5], dtype=torch.int32, device="cuda")
    a = kv4.load(pool, table, start, 60, dtype=torch.float32)
    for dt in (torch.float16, torch.bfloat16):
        b = kv4.load(pool, table, start, 60, dtype=dt)
        assert a[0].shape == b[0].shape == (2, 60, 2, 64)
        assert torch.equal(a[0].to(dt), b[0]) and torch.equal(a[1].to(dt), b[1])


@pytest.mark.parametrize("HD", [64, 128])
def test_store_of_special_values(HD):
    """Constant groups are exact, magnitudes are held to 16384, a NaN spoils its own group of 32 alone."""
    from rngd_pd import kv4
    x = torch.randn(1, 1, 5, 1, HD, generator=torch.Generator().manual_seed(1))
    x[0, 0, 0, 0, :32] = 0.75
    x[0, 0, 1, 0, 3], x[0, 0, 1, 0, 4] = float("inf"), -1e30
    x[0, 0, 2, 0, 33] = float("nan")
    x[0, 0, 3, 0, :32] = 1e-7 * torch.arange(32)
    x[0, 0, 4, 0, :32] = 0.0
    pool = _pool_of(1, 1, 1, HD, 0)
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv4.store(pool, z.view(1, 1), z, x.cuda(), x.cuda())
    for y in kv4.load(pool, z.view(1, 1), z, 5, dtype=torch.float32):
        y = _np(y)[0, 0, :, 0]
        u, s, c, _ = ref.encode(_np(x)[0, 0, :, 0])
        assert np.array_equal(y, ref.values(u, s, c), equal_nan=True)
        assert np.all(y[0, :32] == 0.75) and np.all(y[4, :32] == 0.0)
        assert abs(y[1, 3] - 16384) < 32 and abs(y[1, 4] + 16384) < 32
        assert np.isnan(y[2, 32:64]).all() and np.isfinite(np.delete(y[2], np.arange(32, 64))).all()


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("HD", [64, 128])
def test_store_of_groups_far_from_zero(dt, HD):
    """Means of 0 to 2^13 steps: c's rounding comes to count for more than a step, and codes are held to 0..15."""
    from rngd_pd import kv4
    far = [0.0, 10.0, 100.0, 400.0, 520.0, 700.0, 2000.0, 8192.0]
    x = 15 * torch.rand(len(far), 2, HD, generator=torch.Generator().manual_seed(HD))
    x += torch.tensor(far).view(-1, 1, 1)
    x[:, 1] *= -0.03                                        # and small steps below zero
    x = x.to(DT[dt])
    pool, z = _pool_of(1, 1, 2, HD, 0), torch.zeros(1, dtype=torch.int32, device="cuda")
    rows = x.view(1, 1, len(far), 2, HD).cuda()
    kv4.store(pool, z.view(1, 1), z, rows, rows)
    X = _np(x)
    u, s, c, tie = ref.encode(X)
    want, step, base = ref.values(u, s, c), np.repeat(s, 32, -1), np.repeat(np.abs(c), 32, -1)
    for y in kv4.load(pool, z.view(1, 1), z, len(far), dtype=torch.float32):
        y = _np(y)[0, 0]
        # the quotient in fp32 is off by 2^-18 of a step at most (two roundings of up to 32 steps)
        assert np.all((y == want) | ((tie < 2.0 ** -16) & (np.abs(y - want) <= 1.01 * step)))
        # half a step, s rounded (31 times), c and the value rounded to 11 bits
        assert np.all(np.abs(y - X) <= step * (0.5 + 31 * 2.0 ** -11) + 2.0 ** -11 * (base + np.abs(y)))
    # the scales themselves against 64 bits: s to a place of fp16, c the nearest to min - 16 s but for fp32's rounding
    raw = pool[0, 0].cpu().numpy()[:, 0, 16 * HD:18 * HD]   # first block, K's scales [heads][16 keys][HD / 32][s, c]
    sc = np.ascontiguousarray(raw).view(np.float16).astype(np.float64).reshape(2, 16, HD // 32, 2)
    g = X.reshape(len(far), 2, -1, 32)
    for i in range(len(far)):
        s64 = (g[i].max(-1) - g[i].min(-1)) / 15
        assert np.all(np.abs(sc[:, i, :, 0] - s64) <= 2.0 ** -10 * s64)
        c64 = g[i].min(-1) - 16 * sc[:, i, :, 0]
        assert np.all(np.abs(sc[:, i, :, 1] - c64) <= 2.0 ** -11 * np.abs(c64) * (1 + 2.0 ** -10) + 2.0 ** -24)


def test_store_takes_any_strides():
    """The prefill engine's layout [L][2][NKV][S][HD], odd strides and odd addresses store the same bytes."""
    from rngd_pd import kv4
    L, NKV, S, HD, T = 2, 3, 40, 128, 33
    g = torch.Generator().manual_seed(5)
    kv = torch.randn(L, 2, NKV, S, HD, generator=g).to(torch.bfloat16).cuda()
    k, v = (kv[:, i, :, :T].permute(0, 2, 1, 3)[:, None] for i in (0, 1))
    odd = torch.zeros(L * T * NKV * (HD + 3) + 1, dtype=torch.bfloat16, device="cuda")[1:]
    odd = odd.view(L, 1, T, NKV, HD + 3)[..., :HD]
    odd.copy_(k)
    start = torch.tensor([9], dtype=torch.int32, device="cuda")
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    pools = [_pool_of(L, 3, NKV, HD, 0) for _ in range(3)]
    kv4.store(pools[0], table, start, k.contiguous(), v.contiguous())
    kv4.store(pools[1], table, start, k, v)
    kv4.store(pools[2], table, start, odd, v)
    assert torch.equal(pools[0], pools[1]) and torch.equal(pools[0], pools[2])
    # one layer at a time, through one layer's pool
    one = _pool_of(L, 3, NKV, HD, 0)
    for l in range(L):
        kv4.store(one[l], table, start, k[l], v[l])
    assert torch.equal(one, pools[0])


# ---------------------------------------------------------------------------------------- attention
def _check(q, pool, table, lens, dt, window=0, sinks=0, scale=None, out=None):
    from rngd_pd import kv4
    B, T, NH, HD = q.shape
    got = kv4.attention(q, pool, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), window=window,
                        sinks=sinks, scale=scale, out=out)
    assert got.dtype == q.dtype and got.shape == q.shape
    K, V = ref.decode_pool(pool.cpu().numpy())
    want, bound = ref.attend(_np(q), K, V, table.cpu().numpy(), lens, window, sinks, HD ** -0.5 if scale is None else scale)
    got = _np(got)
    assert np.isfinite(got).all()
    over = np.abs(got - want) - (bound + EPS[dt] * np.abs(want))
    assert over.max() <= 0, f"off by {np.abs(got - want).max()}, {over.max()} over the bound"
    return got


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("HD", [64, 128])
@pytest.mark.parametrize("NH,NKV", [(8, 2), (4, 4), (14, 2), (16, 2), (6, 2)])
def test_attention_over_lengths(dt, HD, NH, NKV):
    lens = [0, 1, 15, 16, 17, 63, 64, 65, 130, 200]
    pool, table = _cache(len(lens), 4, NKV, HD, lens, 11)
    q = torch.randn(len(lens), 1, NH, HD, generator=torch.Generator().manual_seed(2)).to(DT[dt]).cuda()
    got = _check(q, pool, table, lens, dt)
    assert np.all(got[0] == 0)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("window,sinks", [(0, 5), (1, 0), (1, 4), (16, 0), (64, 1), (65, 64), (100, 70), (1000, 3),
                                          (2 ** 31 - 1, 0), (40, 2 ** 31 - 1)])
def test_attention_windows_and_sinks(dt, window, sinks):
    lens = [1, 2, 64, 129, 190, 256, 255]
    pool, table = _cache(len(lens), 4, 2, 128, lens, 12)
    for T in (1, 3):
        q = torch.randn(len(lens), T, 8, 128, generator=torch.Generator().manual_seed(T)).to(DT[dt]).cuda()
        _check(q, pool, table, lens, dt, window, sinks)


@pytest.mark.parametrize("HD", [64, 128])
@pytest.mark.parametrize("T", [2, 4, 5, 9, 16, 33])
def test_attention_of_several_tokens(HD, T):
    """Each token sees up to itself; where a sequence holds fewer positions than tokens the first see nothing."""
    lens = [0, 1, T - 1, T, T + 1, 64, 70, 191]
    pool, table = _cache(len(lens), 3, 2, HD, lens, 13)
    q = torch.randn(len(lens), T, 8, HD, generator=torch.Generator().manual_seed(T)).cuda()
    got = _check(q, pool, table, lens, "fp32")
    assert np.all(got[0] == 0) and np.all(got[1, :T - 1] == 0)
    _check(q, pool, table, lens, "fp32", window=T // 2 + 1, sinks=2)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("HD", [64, 128])
@pytest.mark.parametrize("T", [5, 6, 12])
def test_attention_of_many_streams_and_rows(dt, HD, T):
    """20, 24 and 48 query rows of a kv head, in enough streams to fill the GPU."""
    lens = [0, 1, T - 1, T, 63, 64, 65, 128] + [(37 * i) % 150 for i in range(32)]
    pool, table = _cache(len(lens), 3, 4, HD, lens, 31)
    q = torch.randn(len(lens), T, 16, HD, generator=torch.Generator().manual_seed(HD + T)).to(DT[dt]).cuda()
    got = _check(q, pool, table, lens, dt)
    assert np.all(got[0] == 0)
    _check(q, pool, table, lens, dt, window=33, sinks=3)


def test_attention_without_pages():
    """-1, ids outside the pool and a table too narrow for the length: those positions are not seen."""
    lens = [200, 200, 130, 64, 1000]
    pool, table = _cache(5, 4, 2, 128, [200, 200, 130, 64, 256], 14)
    P = pool.shape[0]
    table[0, 1], table[1, 0], table[1, 3], table[2, 2], table[3, 0] = -1, P, -5, 2 ** 31 - 1, -1
    q = torch.randn(5, 1, 8, 128, generator=torch.Generator().manual_seed(3)).cuda()
    got = _check(q, pool, table, lens, "fp32")
    assert np.all(got[3] == 0)
    narrow = torch.empty(5, 0, dtype=torch.int32, device="cuda")
    assert np.all(_check(q, pool, narrow, lens, "fp32") == 0)


@pytest.mark.parametrize("HD,NH", [(64, 4), (64, 16), (128, 4), (128, 16)])
def test_attention_keeps_unseen_nans_out(HD, NH):
    """NaN in keys or values outside the window, and in what a later token alone sees."""
    from rngd_pd import kv4
    g = torch.Generator().manual_seed(21)
    T, n, W = 3, 150, 60
    k, v = torch.randn(2, 1, 1, n, 2, HD, generator=g)
    k[0, 0, 7, 0, 3] = v[0, 0, 9, 1, 40] = v[0, 0, n - T - W, 0, 0] = float("nan")   # before any window
    v[0, 0, n - 1, 0, 5] = k[0, 0, n - 2, 1, 5] = float("nan")                       # the last tokens' own
    pool, table = _pool_of(1, 4, 2, HD), torch.tensor([[3, 1, 0]], dtype=torch.int32, device="cuda")
    kv4.store(pool, table, torch.zeros(1, dtype=torch.int32, device="cuda"), k.cuda(), v.cuda())
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = torch.randn(1, T, NH, HD, generator=g).cuda()
    got = _np(kv4.attention(q, pool[0], table, lens, window=W))[0]
    G = NH // 2
    assert np.isfinite(got[0]).all() and np.isfinite(got[1, :G]).all()
    assert np.isnan(got[1, G:]).all() and np.isnan(got[2, :G]).any() and np.isnan(got[2, G:]).all()
    # what is finite is what it would be without the NaNs
    clean = k.nan_to_num(1.0), v.nan_to_num(1.0)
    kv4.store(pool, table, torch.zeros(1, dtype=torch.int32, device="cuda"), clean[0].cuda(), clean[1].cuda())
    want = _np(kv4.attention(q, pool[0], table, lens, window=W))[0]
    np.testing.assert_allclose(got[0], want[0], rtol=0, atol=1e-6)


def test_attention_of_more_streams_than_a_launch_takes():
    B = 1030
    lens = [(7 * b) % 60 for b in range(B)]
    pool, table = _cache(B, 1, 1, 64, lens, 22)
    q = torch.randn(B, 1, 2, 64, generator=torch.Generator().manual_seed(9)).cuda()
    _check(q, pool, table, lens, "fp32")


def test_offsets_beyond_32_bits():
    """Pages, and layers of a pool, more than 4 GB apart."""
    from rngd_pd import kv4
    P, NKV, HD, n = 30000, 8, 128, 130
    g = torch.Generator().manual_seed(23)
    k, v = (torch.randn(2, 1, n, NKV, HD, generator=g).to(torch.bfloat16).cuda() for _ in (0, 1))
    q = torch.randn(1, 1, 32, HD, generator=g).cuda()
    zero, lens = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda")
    near, far = kv4.alloc_pool(2, 3, NKV, HD), kv4.alloc_pool(2, P, NKV, HD)
    tn = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    tf = torch.tensor([[P - 1, 3, P - 2]], dtype=torch.int32, device="cuda")
    kv4.store(near, tn, zero, k, v)
    kv4.store(far, tf, zero, k, v)
    for l in range(2):
        assert torch.equal(kv4.attention(q, near[l], tn, lens), kv4.attention(q, far[l], tf, lens))
    assert all(torch.equal(a, b) for a, b in zip(kv4.load(near, tn, zero, n), kv4.load(far, tf, zero, n)))
    ref0 = torch.zeros(P, dtype=torch.int32, device="cuda")
    ref0[tf[0].long()] = 1
    _, t2, live = kv4.compact(far, ref0, tf)
    assert live.item() == 3 and sorted(t2[0].tolist()) == [0, 1, 2]
    assert all(torch.equal(a, b) for a, b in zip(kv4.load(near, tn, zero, n), kv4.load(far, t2, zero, n)))


def test_attention_takes_any_strides_and_writes_into_out():
    lens = [77, 130]
    pool, table = _cache(2, 3, 2, 64, lens, 15)
    big = torch.randn(2, 5, 8, 3, 64 + 5, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    q = big[:, 1:4, :, 1, 5:]
    a = _check(q, pool, table, lens, "bf16")
    out = torch.zeros(2, 8, 3, 64, dtype=torch.bfloat16, device="cuda")
    b = _check(q, pool, table, lens, "bf16", out=out.transpose(1, 2))
    assert np.array_equal(a, b) and np.array_equal(_np(out.transpose(1, 2)), a)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("mag", [1e-4, 30.0, 3000.0])
def test_attention_of_small_and_large_queries(dt, mag):
    """Flat and one-hot softmaxes; q beyond what its products hold in fp16."""
    lens = [150, 64]
    pool, table = _cache(2, 3, 2, 128, lens, 16)
    q = (mag * torch.randn(2, 1, 8, 128, generator=torch.Generator().manual_seed(6))).to(DT[dt]).cuda()
    _check(q, pool, table, lens, dt)
    q[0, 0, 0] = 0.0
    _check(q, pool, table, lens, dt, scale=0.7)


def test_attention_of_wide_ranging_queries():
    """One dimension 2^20 times the others: the small ones still count to fp32 accuracy of the sum."""
    pool, table = _cache(1, 2, 1, 64, [100], 17)
    q = torch.randn(1, 1, 4, 64, generator=torch.Generator().manual_seed(7))
    q[..., 5] *= 2.0 ** 20
    _check((q * 1e-5).cuda(), pool, table, [100], "fp32")


@pytest.mark.parametrize("B,width,lens", [(1, 80, [5000]), (3, 40, [2500, 3, 1700]), (40, 3, list(range(1, 161, 4)))])
def test_attention_long_and_ragged(B, width, lens):
    """Work of one stream split over many warps, and many short streams; the same answer twice."""
    from rngd_pd import kv4
    pool, table = _cache(B, width, 2, 128, lens, 18)
    q = torch.randn(B, 1, 8, 128, generator=torch.Generator().manual_seed(8)).cuda()
    got = _check(q, pool, table, lens, "fp32")
    for _ in range(3):
        again = kv4.attention(q, pool, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
        assert np.array_equal(_np(again), got)
    _check(q, pool, table, lens, "fp32", window=700, sinks=130)


def test_attention_on_another_stream_and_in_a_graph():
    from rngd_pd import kv4
    lens = torch.tensor([150, 90], dtype=torch.int32, device="cuda")
    pool, table = _cache(2, 3, 2, 128, [150, 90], 19)
    q = torch.randn(2, 1, 8, 128, device="cuda")
    want = kv4.attention(q, pool, table, lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = kv4.attention(q, pool, table, lens)
    s.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv4.attention(q, pool, table, lens, out=out)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    lens.copy_(torch.tensor([70, 1], dtype=torch.int32))   # the graph follows lengths on the device
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, kv4.attention(q, pool, table, lens))


def test_attention_keeps_its_workspace_through_the_call(monkeypatch):
    """What another thread allocates on the stream while the call runs is not the call's workspace."""
    from rngd_pd import kv4
    q = torch.zeros(1, 1, 8, 128, dtype=torch.bfloat16, device="cuda")
    table = torch.full((1, 65), -1, dtype=torch.int32, device="cuda")
    lens, pool = torch.zeros(1, dtype=torch.int32, device="cuda"), kv4.alloc_pool(1, 2, 2, 128)[0]
    seen = []

    def entry(*a):                                          # in place of the C entry: nothing is launched
        ws, need = a[18], a[19]
        others = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(3)]
        seen.append((ws, need, [t.data_ptr() for t in others]))
        return 0

    monkeypatch.setattr(kv4, "_attn", entry)
    kv4.attention(q, pool, table, lens)
    (ws, need, others), = seen
    assert need > 0 and all(p + need <= ws or ws + need <= p for p in others)


# ------------------------------------- attention split over warps: tables wide enough for long sequences
def _shared(B, width, NKV, HD, lens, seed, P=90):
    """P full pages, and a table of them in which sequences share pages; entries past a length hold none."""
    from rngd_pd import kv4
    g = torch.Generator().manual_seed(seed)
    pool = _pool_of(1, P, NKV, HD)
    rows = torch.randn(2, 1, P, 64, NKV, HD, generator=g)
    rows[0] += torch.randn(1, 1, 1, NKV, HD, generator=g)
    kv4.store(pool, torch.arange(P, dtype=torch.int32, device="cuda").view(P, 1),
              torch.zeros(P, dtype=torch.int32, device="cuda"), *rows.cuda())
    table = torch.randint(0, P, (B, width), generator=g).to(torch.int32)
    for b, n in enumerate(lens):
        table[b, -(-n // 64):] = -1
    return pool[0], table.cuda()


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("HD", [64, 128])
@pytest.mark.parametrize("G,T", [(1, 1), (4, 1), (7, 1), (4, 4), (4, 5), (3, 11)])
def test_runs_over_rows_and_types(dt, HD, G, T):
    """1 to 33 query rows of a kv head: every layout of q and P, over lengths from none to 4401."""
    lens = [0, 1, 33, 700, 4401, 2050]
    pool, table = _shared(len(lens), 70, 2, HD, lens, 41)
    q = torch.randn(len(lens), T, 2 * G, HD, generator=torch.Generator().manual_seed(HD + G + T)).to(DT[dt]).cuda()
    got = _check(q, pool, table, lens, dt)
    assert np.all(got[0] == 0) and np.all(got[1, :T - 1] == 0)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("HD", [64, 128])
@pytest.mark.parametrize("G,T,window,sinks", [(4, 1, 4100, 70), (4, 1, 2000, 5), (4, 5, 4097, 1), (7, 1, 4200, 0), (4, 4, 2500, 200)])
def test_runs_with_windows_and_sinks(dt, HD, G, T, window, sinks):
    """Units of sinks and of the window, in segments that are cut."""
    lens = [5100, 4100, 0, 130, 4801]
    pool, table = _shared(len(lens), 80, 2, HD, lens, 42)
    q = torch.randn(len(lens), T, 2 * G, HD, generator=torch.Generator().manual_seed(HD + G + T)).to(DT[dt]).cuda()
    _check(q, pool, table, lens, dt, window, sinks)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("HD", [64, 128])
@pytest.mark.parametrize("G,T", [(4, 1), (4, 4), (2, 3)])
def test_runs_of_many_segments(dt, HD, G, T):
    """160 segments, most of them cut in two or not at all: the join takes all rows of one at a time."""
    lens = [(617 * b) % 900 for b in range(38)] + [4480, 3001]
    pool, table = _shared(len(lens), 70, 4, HD, lens, 43)
    q = torch.randn(len(lens), T, 4 * G, HD, generator=torch.Generator().manual_seed(HD + G + T)).to(DT[dt]).cuda()
    got = _check(q, pool, table, lens, dt)
    from rngd_pd import kv4
    again = kv4.attention(q, pool, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert np.array_equal(_np(again), got)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("HD,G,T", [(64, 4, 1), (128, 4, 1), (64, 4, 4), (128, 4, 4), (128, 5, 4)])
def test_runs_over_missing_pages_and_unseen_nans(dt, HD, G, T):
    """No page, ids that are none, a table too narrow, and NaN before the window: none of it has a part."""
    from rngd_pd import kv4
    lens = [4400, 4400, 2100, 5000, 4000]
    pool, table = _shared(len(lens), 70, 2, HD, lens, 44, P=95)
    table[0, 3], table[0, 40], table[1, 0], table[1, 68], table[2, 20:] = -1, 95, -7, 2 ** 31 - 1, -1
    table[4] = -1
    lost = torch.full((1, 1, 64, 2, HD), float("nan"), device="cuda")
    kv4.store(pool.unsqueeze(0), torch.tensor([[94]], dtype=torch.int32, device="cuda"),
              torch.zeros(1, dtype=torch.int32, device="cuda"), lost, lost)
    window, sinks = 4150, 3
    table[table == 94] = 93
    table[0, 1] = table[1, 2] = 94                          # positions 64..191, past the sinks and before the window
    q = torch.randn(len(lens), T, 2 * G, HD, generator=torch.Generator().manual_seed(HD + G)).to(DT[dt]).cuda()
    got = _check(q, pool, table, lens, dt, window, sinks)
    assert np.all(got[4] == 0)


def test_runs_of_more_streams_than_a_launch_takes():
    """Records and prefix sums are used again by the second launch."""
    B = 1030
    lens = [(37 * b) % 150 for b in range(B)]
    lens[3], lens[500], lens[1026], lens[1029] = 4160, 3000, 4100, 2999
    pool, table = _shared(B, 65, 1, 64, lens, 45, P=70)
    q = torch.randn(B, 1, 2, 64, generator=torch.Generator().manual_seed(9)).cuda()
    _check(q, pool, table, lens, "fp32")


# -------------------------------------------------------------------------------------------- pages
def _run_fork(ref0, table, lens, parents, room, L=2, NKV=2, HD=64):
    from rngd_pd import kv4
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    P = len(ref0)
    pool = torch.randint(0, 256, (L, P, NKV, 4, 20 * HD), dtype=torch.uint8, device="cuda")
    before = pool.clone()
    t = i32(table).view(len(table), -1)
    old = (i32(ref0), t, i32(lens))
    keep = [x.clone() for x in old]
    got = kv4.fork(pool, *old, None if parents is None else i32(parents), room=room)
    want = ref.fork(ref0, table, lens, parents if parents is not None else list(range(len(table))), room)
    assert [x.tolist() for x in got[:3]] == [want[0], want[1], want[2]] and got[3].tolist() == [want[3]]
    for s, d, n in want[4]:
        before[:, d, :, :n] = before[:, s, :, :n]
    assert torch.equal(pool, before)
    assert all(torch.equal(a, b) for a, b in zip(old, keep))
    return got


def test_fork_of_beams():
    ref0 = [0] * 20
    table = [[3, 7, 9, -1], [3, 7, 4, -1], [3, 11, -1, -1], [1, -1, -1, -1]]
    for row in table:
        for p in row:
            if p >= 0:
                ref0[p] += 1
    lens = [150, 140, 128, 5]
    for parents in ([0, 0, 0, 0], [1, 0, 3, 3], [2, 2, 1, -1], [-1, -1, -1, -1], [0, 1, 2, 3], None, [3, 3, 2, 0]):
        for room in (0, 1, 64, 70, 1000):
            _run_fork(ref0, table, lens, parents, room)


def test_fork_when_others_hold_the_page():
    """A last page with a holder outside the rows is copied for every row."""
    _run_fork([0, 3, 2, 0, 0], [[1, 2], [1, -1]], [100, 64], [0, 0], 1)
    _run_fork([0, 3, 2, 0, 0], [[1, 2], [1, -1]], [100, 64], None, 0)


def test_fork_without_free_pages():
    _run_fork([1, 1], [[0, 1, -1]], [100], None, 100)
    _run_fork([2, 1, 0], [[0, 1], [0, -1]], [100, 64], [0, 0], 30)
    _run_fork([2, 1], [[0, 1], [0, -1]], [100, 64], [0, 0], 30)


@pytest.mark.parametrize("R,width,seed", [(1, 1, 0), (7, 5, 1), (64, 33, 2), (300, 9, 3), (1024, 2, 4)])
def test_fork_of_random_states(R, width, seed):
    g = np.random.default_rng(seed)
    lens = [int(x) for x in g.integers(0, width * 64 + 1, R)]
    P = R * width + 5000
    ids = [int(x) for x in g.permutation(P)]
    table, ref0 = [], [0] * P
    for n in lens:
        row = [ids.pop() for _ in range(-(-n // 64))]
        table.append(row + [-1] * (width - len(row)))
        for p in row:
            ref0[p] += 1
    for p in g.choice(P, 50):
        ref0[int(p)] += int(g.integers(0, 3))
    parents = [int(x) for x in g.integers(-1, R, R)]
    _run_fork(ref0, table, lens, parents, int(g.integers(0, 3)), L=1, NKV=1)


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 63, 2 ** 31 - 64])
def test_fork_of_lengths_near_the_largest_number(n):
    """A length far beyond the table keeps the table's pages; what is missing beyond them is counted."""
    from rngd_pd import kv4
    pool = kv4.alloc_pool(1, 8, 1, 64)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    ref0, table, lens = i32([1, 1, 1, 1, 0, 0, 0, 0]), i32([[2, 0], [1, 3]]), i32([n, 70])
    for room in (0, 100):
        new_ref, new_table, new_lens, short = kv4.fork(pool, ref0, table, lens, i32([0, 1]), room=room)
        assert new_table.tolist() == [[2, 0], [1, 3]] and new_lens.tolist() == [n, 70]
        assert new_ref.tolist() == ref0.tolist()
        assert short.item() == -(-(n + room) // 64) - 2 + (1 if room else 0)
    new_ref, new_table, _, short = kv4.fork(pool, ref0, table, lens, i32([0, 0]))
    assert new_table.tolist() == [[2, 0], [2, 0]] and new_ref.tolist() == [2, 0, 2, 0, 0, 0, 0, 0]
    assert short.item() == 2 * (-(-n // 64) - 2)


@pytest.mark.parametrize("R,room", [(1024, 2 ** 30), (130, 2 ** 30), (3, 2 ** 30), (1024, 2 ** 26)])
def test_fork_counts_more_missing_pages_than_a_number_holds(R, room):
    """`short` stays at 2^31 - 1 where more pages are missing."""
    from rngd_pd import kv4
    pool = kv4.alloc_pool(1, 2, 1, 64)
    ref0, table, lens = kv4.empty_state(R, 1, 2)
    new_ref, new_table, _, short = kv4.fork(pool, ref0, table, lens, room=room)
    assert short.item() == min(R * (room // 64) - 2, 2 ** 31 - 1)
    assert new_table[:, 0].tolist() == [0, 1] + [-1] * (R - 2) and new_ref.tolist() == [1, 1]


@pytest.mark.parametrize("P,live,seed", [(1, 0, 0), (1, 1, 1), (5, 5, 2), (100, 60, 3), (3000, 10, 4), (5000, 2600, 5)])
def test_compact(P, live, seed):
    from rngd_pd import kv4
    g = np.random.default_rng(seed)
    L, NKV, HD = 2, 1, 64
    held = np.sort(g.permutation(P)[:live])
    ref0 = np.zeros(P, np.int32)
    ref0[held] = g.integers(1, 4, live)
    rows = 4
    table = np.full((rows, live // rows + 2), -1, np.int32)
    table.reshape(-1)[:live] = g.permutation(held)
    pool = torch.randint(0, 256, (L, P, NKV, 4, 20 * HD), dtype=torch.uint8, device="cuda")
    before = pool.clone()
    t0, r0 = torch.from_numpy(table).cuda(), torch.from_numpy(ref0).cuda()
    ref1, table1, n = kv4.compact(pool, r0, t0)
    src, dst = held[held >= live], np.setdiff1d(np.arange(live), held)
    to = np.arange(P)
    to[src] = dst
    want = ref0.copy()
    want[dst], want[src] = ref0[src], 0
    assert n.tolist() == [live] and np.array_equal(ref1.cpu().numpy(), want)
    assert np.array_equal(table1.cpu().numpy(), np.where(table >= 0, to[table.clip(0)], -1))
    before[:, torch.from_numpy(dst).cuda()] = before[:, torch.from_numpy(src).cuda()]
    assert torch.equal(pool, before)
    assert np.array_equal(r0.cpu().numpy(), ref0) and np.array_equal(t0.cpu().numpy(), table)


def test_forked_beams_attend_as_their_own_copies():
    """Store, fork, store on: each beam reads what it would had it its own cache from the start."""
    from rngd_pd import kv4
    B, NKV, HD, P = 3, 2, 128, 16
    g = torch.Generator().manual_seed(20)
    pool = kv4.alloc_pool(1, P, NKV, HD)
    ref0, table, lens = kv4.empty_state(B, 4, P)
    rows = torch.randn(2, 1, B, 100, NKV, HD, generator=g).cuda()
    ref0, table, lens, short = kv4.fork(pool, ref0, table, lens, room=100)
    kv4.store(pool, table, lens, *rows)
    lens = lens + 100
    parents = torch.tensor([2, 2, 0], dtype=torch.int32, device="cuda")
    ref0, table, lens, short = kv4.fork(pool, ref0, table, lens, parents, room=40)
    more = torch.randn(2, 1, B, 40, NKV, HD, generator=g).cuda()
    kv4.store(pool, table, lens, *more)
    lens = lens + 40
    assert short.item() == 0 and int((ref0 > 0).sum()) == 2 + 3 + 3  # two shared, a partly filled one and a new one each
    whole = torch.cat((rows[:, :, parents.long()], more), 3)
    own = kv4.alloc_pool(1, 9, NKV, HD)
    flat = torch.arange(9, dtype=torch.int32, device="cuda").view(3, 3)
    kv4.store(own, flat, torch.zeros(3, dtype=torch.int32, device="cuda"), *whole)
    q = torch.randn(B, 1, 8, HD, generator=g).cuda()
    n = torch.full((3,), 140, dtype=torch.int32, device="cuda")
    assert torch.equal(kv4.attention(q, pool[0], table, lens), kv4.attention(q, own[0], flat, n))
    assert torch.equal(lens, n)
    ref1, table1, live = kv4.compact(pool, ref0, table)
    assert live.item() == 8 and int(table1.max()) == 7
    assert torch.equal(kv4.attention(q, pool[0], table1, lens), kv4.attention(q, own[0], flat, n))


# ----------------------------------------------------------------------------------------- refusals
def test_refusals_on_the_gpu():
    from rngd_pd import kv4
    pool = kv4.alloc_pool(1, 4, 2, 64)
    ref0, table, lens = kv4.empty_state(2, 2, 4)
    q = torch.zeros(2, 1, 8, 64, device="cuda")
    k = torch.zeros(1, 2, 1, 2, 64, device="cuda")
    bad = [
        lambda: kv4.attention(q, pool, table, lens),                        # all layers' pool
        lambda: kv4.attention(q[..., :32], pool[0], table, lens),           # head dimension
        lambda: kv4.attention(q[:, :, :3], pool[0], table, lens),           # heads not a multiple
        lambda: kv4.attention(q.double(), pool[0], table, lens),
        lambda: kv4.attention(q.transpose(2, 3), pool[0], table, lens),     # last dimension strided
        lambda: kv4.attention(q, pool[0], table.long(), lens),
        lambda: kv4.attention(q, pool[0], table, lens[:1]),
        lambda: kv4.attention(q, pool[0], table, lens, window=-1),
        lambda: kv4.attention(q, pool[0], table, lens, out=torch.zeros(2, 1, 8, 64)),
        lambda: kv4.store(pool, table, lens, k[..., :32], k[..., :32]),
        lambda: kv4.store(pool, table, lens, k, k.half()),
        lambda: kv4.store(pool, table, lens, k, k[:, :1]),
        lambda: kv4.store(pool, table, lens.float(), k, k),
        lambda: kv4.load(pool, table, lens, -1),
        lambda: kv4.load(pool, table, lens, 1, dtype=torch.float64),
        lambda: kv4.fork(pool, ref0[:3], table, lens),
        lambda: kv4.fork(pool, ref0, table, lens, lens[:1]),
        lambda: kv4.compact(pool, ref0.long(), table),
        lambda: kv4.alloc_pool(1, 4, 2, 96),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    from rngd_pd import _lib
    with pytest.raises(_lib.RngdError):
        kv4.fork(pool, ref0, table, lens, room=-1)
    with pytest.raises(_lib.RngdError):
        kv4.fork(pool, *kv4.empty_state(1025, 1, 4))


def test_memory_that_would_be_written_twice_is_refused():
    """Pools whose layers lie on one another, and outputs whose rows do."""
    from rngd_pd import kv4
    pool = kv4.alloc_pool(1, 4, 2, 64)
    two = pool.expand(2, 4, 2, 4, 1280)
    near = kv4.alloc_pool(1, 5, 2, 64).view(-1).as_strided((2, 4, 2, 4, 1280), (10240, 10240, 5120, 1280, 1))
    ref0, table, lens = kv4.empty_state(2, 2, 4)
    k = torch.zeros(2, 2, 1, 2, 64, device="cuda")
    for bad in (two, near):
        for f in (lambda: kv4.store(bad, table, lens, k, k), lambda: kv4.fork(bad, ref0, table, lens),
                  lambda: kv4.compact(bad, ref0, table), lambda: kv4.load(bad, table, lens, 1)):
            with pytest.raises(ValueError):
                f()
    part = kv4.alloc_pool(3, 6, 2, 64)[:, 1:5]              # pages of a larger pool: layers lie apart
    kv4.store(part, table, lens, torch.zeros(3, 2, 1, 2, 64, device="cuda"), torch.zeros(3, 2, 1, 2, 64, device="cuda"))
    one = kv4.alloc_pool(1, 4, 2, 64)[0].unsqueeze(0)
    kv4.load(one, table, lens, 1)
    q = torch.zeros(2, 3, 8, 64, device="cuda")
    for shape in ((1, 3, 8, 64), (2, 1, 8, 64), (2, 3, 1, 64)):
        with pytest.raises(ValueError):
            kv4.attention(q, pool[0], table, lens, out=torch.zeros(shape, device="cuda").expand(q.shape))
    kv4.attention(q[:1, :1].expand(2, 3, 8, 64), pool[0], table, lens)   # q may be read twice


def test_rooms_beyond_32_bits_are_refused():
    """Not taken by their lowest 32 bits."""
    from rngd_pd import _lib, kv4
    pool = kv4.alloc_pool(1, 4, 2, 64)
    for room in (2 ** 30 + 1, 2 ** 32, 2 ** 32 + 64, -2 ** 32, -2 ** 32 + 1):
        with pytest.raises(_lib.RngdError):
            kv4.fork(pool, *kv4.empty_state(2, 2, 4), room=room)
