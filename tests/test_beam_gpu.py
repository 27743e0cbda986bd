"""Beam selection on the GPU against a plain numpy form in 64 bits."""
import numpy as np
import pytest
import torch

from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _check(logits, scores, done, W, eos):
    """The choice has to be the plain form's wherever 64 bits tell its candidates apart by more than fp32 may blur."""
    from rngd_pd import beam
    out = beam.select(logits.cuda(), scores.cuda(), done.cuda(), W, eos)
    x = logits.double().numpy()
    best, parent, token, ended, every = ref.select(x, scores.double().numpy(), done.numpy(), W, eos)
    got = [t.cpu().numpy() for t in out]
    V = x.shape[1]
    # score = cum + (x - lse): lse to 16 roundings of 2^-23 of itself, then two roundings of the magnitudes met
    fin = np.isfinite(x) & (np.abs(x) < 1e30)
    big = np.abs(np.where(fin, x, 0)).max() + np.log(V) + np.abs(np.where(np.isfinite(scores.numpy()), scores.numpy(), 0)).max()
    tol = 24 * 2.0 ** -23 * (big + 1)
    at = (got[1] - W * np.arange(len(best))[:, None]) * V + got[2]
    assert got[1].dtype == np.int32 and got[2].dtype == np.int32 and got[3].dtype == np.bool_
    assert (at >= 0).all() and (at < W * V).all()
    assert all(len(set(row)) == W for row in at.tolist())
    picked = np.take_along_axis(every, at, 1)
    inf = np.isinf(best)
    assert np.array_equal(inf, np.isinf(picked)) and np.array_equal(got[0][inf], picked[inf].astype(np.float32))
    assert np.all(np.abs(got[0][~inf] - picked[~inf]) <= tol) and np.all(np.abs(best[~inf] - picked[~inf]) <= 2 * tol)
    srt = -np.sort(-every, axis=1)[:, :W + 1]
    with np.errstate(invalid="ignore"):
        gap = np.abs(np.diff(srt, axis=1))  # nan between two -inf
    clear = np.ones(best.shape, bool)
    close = gap <= 2 * tol
    clear &= ~close[:, :W] if close.shape[1] >= W else ~np.pad(close, ((0, 0), (0, W - close.shape[1])))
    clear[:, 1:] &= ~close[:, :W - 1]
    assert np.array_equal(got[1][clear], parent[clear]) and np.array_equal(got[2][clear], token[clear])
    assert np.array_equal(got[3], done.numpy()[got[1]] | (got[2] == eos))
    return got, (best, parent, token, ended), clear


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("G,W,V", [(1, 1, 1), (1, 1, 7), (2, 4, 4), (3, 4, 1000), (1, 5, 32003), (2, 8, 8192),
                                   (1, 32, 8193), (5, 3, 16385), (2, 16, 40001), (1, 32, 32)])
def test_select_matches_the_plain_form(dt, G, W, V):
    g = torch.Generator().manual_seed(V + W)
    logits = (3 * torch.randn(G * W, V, generator=g)).to(DT[dt])
    scores = -5 + 2 * torch.randn(G * W, generator=g)
    for n_done in {0, W // 2, W}:
        done = (torch.arange(G * W) % W) < n_done
        _, _, clear = _check(logits, scores, done, W, V // 2)
        if n_done == 0 and dt == "fp32" and V >= 1000:
            assert clear.mean() > 0.9


def test_ties_go_to_the_lowest_row_and_token():
    from rngd_pd import beam
    G, W, V = 2, 4, 20000
    logits = torch.zeros(G * W, V)
    logits[:, 700] = 2.0
    logits[:, 19999] = 2.0
    out = beam.select(logits.cuda(), torch.zeros(G * W).cuda(), torch.zeros(G * W, dtype=torch.bool).cuda(), W)
    assert out[1].tolist() == [[0, 0, 1, 1], [4, 4, 5, 5]] and out[2].tolist() == [[700, 19999] * 2] * 2
    logits[:] = -1.0
    out = beam.select(logits.cuda(), torch.zeros(G * W).cuda(), torch.zeros(G * W, dtype=torch.bool).cuda(), W)
    assert out[1].tolist() == [[0] * 4, [4] * 4] and out[2].tolist() == [[0, 1, 2, 3]] * 2


def test_first_step_from_one_live_beam():
    """Beams at -inf have no continuation while others have any."""
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(8, 500, generator=g)
    scores = torch.tensor([0.0, -np.inf, -np.inf, -np.inf] * 2)
    got, want, _ = _check(logits, scores, torch.zeros(8, dtype=torch.bool), 4, -1)
    assert got[1].tolist() == [[0] * 4, [4] * 4]


def test_masked_infinite_and_nan_logits():
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(12, 9000, generator=g)
    scores = torch.randn(12, generator=g)
    logits[0] = -np.inf                  # a row without continuation
    logits[1, 5] = np.nan                # a row that is lost
    logits[2, 7] = np.inf                # another
    logits[3, 100:] = -np.inf
    logits[4:8] = -np.inf                # a whole group without continuation: the lowest places
    logits[9, ::2] = torch.finfo(torch.float32).min
    logits[10] = torch.finfo(torch.float32).min
    got, want, _ = _check(logits, scores, torch.zeros(12, dtype=torch.bool), 4, 3)
    assert np.isinf(got[0][1]).all() and got[2][1].tolist() == [0, 1, 2, 3] and got[1][1].tolist() == [4] * 4
    assert (got[1][0] == 3).all()
    # done beams whose own score is -inf, or without an eos, are lost too
    done = torch.ones(12, dtype=torch.bool)
    got, want, _ = _check(logits, torch.full((12,), -np.inf), done, 4, 3)
    assert got[2].tolist() == [[0, 1, 2, 3]] * 3
    got, want, _ = _check(logits, scores, done, 4, -1)
    assert got[2].tolist() == [[0, 1, 2, 3]] * 3


def test_done_beams_keep_their_score():
    logits = torch.zeros(4, 1000)
    scores = torch.tensor([-3.0, -1.0, -50.0, -2.0])
    done = torch.tensor([True, False, True, True])
    got, want, _ = _check(logits, scores, done, 4, 17)
    assert got[0][0, :2].tolist() == [-2.0, -3.0] and got[1][0, :2].tolist() == [3, 0]
    assert got[2][0, :2].tolist() == [17, 17] and got[3][0, :2].all()


def test_rows_apart_and_odd_addresses():
    from rngd_pd import beam
    g = torch.Generator().manual_seed(5)
    for dt in DT.values():
        big = torch.randn(6, 5003, generator=g).to(dt).cuda()
        view = big[:, 1:4999]
        scores, done = torch.randn(6, generator=g).cuda(), torch.zeros(6, dtype=torch.bool, device="cuda")
        a = beam.select(view, scores, done, 3, 5)
        b = beam.select(view.contiguous(), scores, done, 3, 5)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_vocabulary_too_large_for_the_list():
    """Many chunks of many beams: the candidates are taken one after the other."""
    g = torch.Generator().manual_seed(6)
    logits = 3 * torch.randn(32, 500009, generator=g)
    _, _, clear = _check(logits, -5 + torch.randn(32, generator=g), torch.arange(32) == 3, 32, 77)
    assert clear.mean() > 0.9


@pytest.mark.parametrize("order", ["up", "down", "late", "steps"])
def test_long_rows_whose_best_come_late(order):
    """Many rows, each CTA goes through several chunks: rising logits fill the list of candidates again and again."""
    W, R, V = 16, 320, 100003
    g = torch.Generator().manual_seed(8)
    base = torch.linspace(-20, 20, V)
    if order == "up":
        logits = base.repeat(R, 1) + 0.001 * torch.rand(R, 1, generator=g)
    elif order == "down":
        logits = base.flip(0).repeat(R, 1) + 0.001 * torch.rand(R, 1, generator=g)
    elif order == "late":
        logits = torch.randn(R, V, generator=g)
        logits[:, 60000:] += 30
    else:
        logits = (torch.arange(V) // 3000).float().repeat(R, 1) / 4
    _check(logits, torch.linspace(-3, 0, R), torch.zeros(R, dtype=torch.bool), W, 1)


@pytest.mark.parametrize("keep", [1, 5, 40])
def test_vocabulary_masked_to_a_few_tokens(keep):
    """All but a few logits at -inf, anywhere in the row."""
    W, R, V = 16, 320, 70001
    g = torch.Generator().manual_seed(keep)
    logits = torch.full((R, V), -np.inf)
    at = torch.stack([torch.randperm(V, generator=g)[:keep] for _ in range(R)])
    logits.scatter_(1, at, torch.randn(R, keep, generator=g))
    _check(logits, torch.randn(R, generator=g), torch.arange(R) % 40 == 3, W, 1)
    scores = torch.full((R,), -np.inf)
    scores[::W] = 0.0
    _check(logits, scores, torch.zeros(R, dtype=torch.bool), W, -1)


def test_equal_logits_in_many_places():
    """The bound falls on a value that many places share: rows of few distinct values, and of two."""
    g = torch.Generator().manual_seed(7)
    for V in (2048, 9000, 40003):
        logits = torch.randint(0, 40, (6, V), generator=g).float() / 8
        logits[3:] = torch.randint(0, 2, (3, V), generator=g).float()
        _check(logits, torch.tensor([0.0, -0.3, -0.7, 0.0, -0.1, -0.2]), torch.zeros(6, dtype=torch.bool), 3, 1)


def test_select_refusals():
    from rngd_pd import beam
    x, s, d = torch.zeros(4, 100, device="cuda"), torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.bool, device="cuda")
    for f in (lambda: beam.select(x.cpu(), s, d, 2), lambda: beam.select(x, s, d, 3), lambda: beam.select(x, s, d, 0),
              lambda: beam.select(x.double(), s, d, 2), lambda: beam.select(x[:, :1], s, d, 2),
              lambda: beam.select(x.t(), s, d, 2), lambda: beam.select(x, s.double(), d, 2),
              lambda: beam.select(x, s, d.int(), 2), lambda: beam.select(x, s[:2], d, 2),
              lambda: beam.select(x, s, d, 2, 100), lambda: beam.select(x[:1].expand(4, 100), s, d, 2)):
        with pytest.raises(ValueError):
            f()
    assert beam.select(x[:0], s[:0], d[:0], 2)[0].shape == (0, 2)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("R", [40, 80, 160])
@pytest.mark.parametrize("W", [1, 2, 4])
def test_few_sets_hold_many_of_the_best(dt, R, W):
    """Logits that repeat with a chunk's stride: the W sets that reach the bound hold more logits than are listed at
    once.  Rows of one chunk (or parts of one) with 2, 4 and 8 vectors a thread."""
    vl = 8 if dt == "bf16" else 4
    step, run = 256 * vl, 4 * vl                            # logits of a vector per thread, and of a set
    V = 8 * step - 3 * vl
    logits = torch.zeros(R, V)
    at = torch.arange(V) % step // run                      # the set that a place falls to
    for i in range(W):
        logits[:, at == (37 * i + 5) % 64] = 3.0 + i        # a value of its own for each of W sets
    logits += torch.arange(R).view(R, 1) % 3                # the same order, other values
    logits = logits.to(DT[dt])
    scores = -0.01 * torch.arange(R).float()
    got, _, _ = _check(logits, scores, torch.zeros(R, dtype=torch.bool), W, 1)
    if W == 1:
        assert np.array_equal(got[2][:, 0], logits.float().numpy().argmax(1))  # the first of the equal ones
    noise = logits + (torch.rand(R, V, generator=torch.Generator().manual_seed(R)) * 0.25).to(DT[dt])
    _check(noise, scores, torch.arange(R) % 7 == 3, W, 1)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("V", [50, 9000])
def test_rows_that_are_lost_offer_their_lowest_tokens(dt, V):
    """A row whose scores are all -inf (by a NaN or +inf logit, by its own score) ranks by place, whatever its logits."""
    from rngd_pd import beam
    W = 4
    logits = torch.randn(4 * W, V, generator=torch.Generator().manual_seed(9)).to(DT[dt])
    scores = torch.zeros(4 * W)
    logits[:W, V // 2] = float("nan")                       # group 0: lost by NaN
    logits[W:2 * W, V // 2] = float("inf")                  # 1: by +inf
    scores[2 * W:3 * W] = -np.inf                           # 2: by their own scores
    scores[3 * W:] = torch.tensor([-np.inf, 0.0, np.nan, -np.inf])
    logits[3 * W + 1, 2:] = -np.inf                         # 3: two continuations, then the lowest places of row 0
    done = torch.zeros(4 * W, dtype=torch.bool)
    out = beam.select(logits.cuda(), scores.cuda(), done.cuda(), W)
    assert torch.isinf(out[0][:3]).all() and out[2][:3].tolist() == [[0, 1, 2, 3]] * 3
    assert out[1][:3].tolist() == [[0] * 4, [W] * 4, [2 * W] * 4]
    assert torch.isinf(out[0][3]).tolist() == [False, False, True, True]
    assert sorted(out[2][3, :2].tolist()) == [0, 1] and out[1][3, :2].tolist() == [3 * W + 1] * 2
    assert out[2][3, 2:].tolist() == [0, 1] and out[1][3, 2:].tolist() == [3 * W] * 2


def test_logits_that_round_to_one_score():
    """At -1000 scores lie 2^-14 apart: a row offers its largest logits, and of those equal scores go by the token."""
    from rngd_pd import beam
    logits = torch.zeros(2, 100)
    logits[:, 50], logits[:, 20], logits[:, 80] = 1.000002, 1.0, 1.000004
    args = lambda s: (torch.tensor(s, device="cuda"), torch.zeros(len(s), dtype=torch.bool, device="cuda"))
    one = beam.select(logits[:1].cuda(), *args([-1000.0]), 1)
    assert one[2].tolist() == [[80]]
    two = beam.select(logits.cuda(), *args([-1000.0, -np.inf]), 2)
    assert two[2].tolist() == [[50, 80]] and two[1].tolist() == [[0, 0]] and two[0][0, 0] == two[0][0, 1]


def test_eos_below_32_bits_ends_nothing():
    from rngd_pd import beam
    logits = torch.randn(2, 100, generator=torch.Generator().manual_seed(2)).cuda()
    s, d = torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.bool, device="cuda")
    best = int(logits.float().argmax() % 100)
    for eos in (-1, -5, -2 ** 31 - 1, best - 2 ** 32):
        out = beam.select(logits, s, d, 2, eos)
        assert not out[3].any() and best in out[2][0].tolist()
