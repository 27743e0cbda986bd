"""Beam search over the paged 4-bit cache through the engine, on a small model: every step's logits against the
numpy restatement of the reference's layer reading the same cache values, the search against its plain form,
one beam against greedy decoding, and pages given back."""
import numpy as np
import pytest
import torch

from oracle import ref_np as R
from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu

SMALL = R.Dims(H=512, M=1024, NH=8, NKV=2, HD=128, L=2, V=1000)


def _cfg(d):
    from rngd_pd.engines.model import ModelConfig
    return ModelConfig.from_dims(H=d.H, M=d.M, NH=d.NH, NKV=d.NKV, HD=d.HD, L=d.L, V=d.V, eps=d.eps, theta=d.theta)


@pytest.fixture(scope="module")
def model():
    from rngd_pd.engines.prefill_full import FullPrefillEngine
    from rngd_pd.synth import SyntheticState
    cfg = _cfg(SMALL)
    return cfg, FullPrefillEngine(cfg, SyntheticState(cfg, seed=0), C=256, group=2, S=256), R.SynthModel(SMALL, seed=0)


def _engine(model, **kw):
    from rngd_pd.engines.beam_decode import BeamDecodeEngine
    return BeamDecodeEngine(model[0], model[1].w, **kw)


def _begin(eng, pre, group, tokens):
    kv, _ = pre.prefill_kv_device(tokens)
    eng.begin(group, tokens, kv, pre.logits())


def _oracle_logits(m, tok, pos, K, V, window, sinks):
    """cpu_layer's arithmetic for one stream with the cache as given (K, V [L, n, NKV, HD], the new row included)."""
    d, inv = m.d, R.inv_freq(m.d)
    x = m.embed()[[tok]].astype(np.float32)
    see = ref.visible(pos, window, sinks)
    new = []
    for l in range(d.L):
        n1, wq, wk, wv, wo, n2, wgu, wd = m.layer(l)
        h = R.rms(x, n1, d.eps)
        q = R._rope_rows(h @ wq.T, [pos], inv, d.NH, d.HD)[0]
        new.append((R._rope_rows(h @ wk.T, [pos], inv, d.NKV, d.HD)[0], (h @ wv.T).reshape(d.NKV, d.HD)))
        ao = np.zeros((d.NH, d.HD), np.float32)
        for a in range(d.NH):
            s = K[l, see, a // d.G] @ q[a] / np.sqrt(d.HD)
            p = np.exp(s - s.max())
            ao[a] = (p / p.sum()) @ V[l, see, a // d.G]
        x = ao.reshape(1, -1) @ wo.T + x
        gu = R.rms(x, n2, d.eps) @ wgu.T
        g, u = gu[:, :d.M], gu[:, d.M:]
        x = (g / (1 + np.exp(-g)) * u) @ wd.T + x
    return R.lm_logits(x, m.norm(), m.lm_head(), d.eps)[0], new


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_step_logits_match_the_oracle_on_the_same_cache(model, window, sinks):
    """Logits within the decode tests' bar for small models (1e-3); the new rows within half a step of 4 bits."""
    from rngd_pd import kv4
    cfg, pre, m = model
    eng = _engine(model, beams=3, groups=2, pages=40, width=4, window=window, sinks=sinks)
    for g, n in ((0, 100), (1, 63)):
        _begin(eng, pre, g, [(7 * j + g) % SMALL.V for j in range(n)])
    for _ in range(3):
        torch.cuda.synchronize()
        toks, scores, done = eng.toks.cpu().numpy().copy(), eng.scores.cpu().numpy().copy(), eng.done.cpu().numpy().copy()
        eng.step()
        torch.cuda.synchronize()
        lens = eng.lens.cpu().numpy()
        logits = eng._e._logits.cpu().numpy()
        n = int(lens.max())
        zero = torch.zeros(eng.B, dtype=torch.int32, device="cuda")
        K, V = (t.cpu().numpy().astype(np.float32) for t in kv4.load(eng.pool, eng.table, zero, n))
        for r in range(eng.B):
            want, new = _oracle_logits(m, int(toks[r]), int(lens[r]) - 1, K[:, r], V[:, r], window, sinks)
            assert np.abs(logits[r] - want).max() < 1e-3
            for l in range(SMALL.L):
                for x, y in zip(new[l], (K[l, r, lens[r] - 1], V[l, r, lens[r] - 1])):
                    step = ((x.reshape(SMALL.NKV, -1, 32).max(-1) - x.reshape(SMALL.NKV, -1, 32).min(-1)) / 15).repeat(32, -1)
                    assert np.all(np.abs(x - y) <= 0.6 * step.reshape(x.shape) + 0.02)
        # the selection that followed
        best, parent, token, ended, _ = ref.select(logits.astype(np.float64), scores.astype(np.float64), done, eng.W, eng.eos)
        assert np.array_equal(eng.parents.cpu().numpy(), parent.reshape(-1))
        assert np.array_equal(eng.toks.cpu().numpy(), token.reshape(-1))
        np.testing.assert_allclose(eng.scores.cpu().numpy(), best.reshape(-1), rtol=0, atol=1e-4)
    from rngd_pd import _lib
    assert _lib.device_status() == 0 and int(eng.short.item()) == 0


def test_one_beam_is_greedy_and_many_steps_are_one_by_one(model):
    """A search of one beam picks each step's largest logit; a graph of steps equals steps run alone."""
    cfg, pre, m = model
    prompt = [(11 * j + 3) % SMALL.V for j in range(50)]
    eng = _engine(model, beams=1, groups=2, pages=20, width=3)
    _begin(eng, pre, 1, prompt)
    first = int(pre.logits().argmax())
    picked = [first]
    for _ in range(20):
        eng.step()
        torch.cuda.synchronize()
        picked.append(int(eng._e._logits[1].argmax()))
    (score, seq), = eng.result(1)
    assert seq == picked
    two = _engine(model, beams=1, groups=2, pages=20, width=3)
    two._e.use_graph = False
    _begin(two, pre, 1, prompt)
    two.step(20)
    assert two.result(1) == [(score, seq)]


def test_search_beats_greedy_and_gives_pages_back(model):
    """Scores come sorted and are sums of log-probabilities at least as good as greedy's; ended groups and a new
    search reuse the pages; compaction changes nothing a search sees."""
    cfg, pre, m = model
    prompt = [(5 * j + 1) % SMALL.V for j in range(70)]
    one, four = _engine(model, beams=1, groups=1, pages=16, width=3), _engine(model, beams=4, groups=2, pages=24, width=3)
    for e in (one, four):
        _begin(e, pre, 0, prompt)
        e.step(8)
    res = four.result(0)
    assert len(res) == 4 and [s for s, _ in res] == sorted((s for s, _ in res), reverse=True)
    assert len({tuple(t) for _, t in res}) == 4 and all(len(t) == 9 for _, t in res)
    assert res[0][0] >= one.result(0)[0][0] - 1e-3
    _begin(four, pre, 1, prompt[:40])
    four.step(3)
    live = int((four.ref > 0).sum())
    before = four.result(0), four.result(1)
    assert four.compact() == live and int(four.table.max()) == live - 1
    again = _engine(model, beams=4, groups=2, pages=24, width=3)
    _begin(again, pre, 0, prompt)
    again.step(8)
    _begin(again, pre, 1, prompt[:40])
    again.step(3)
    assert (again.result(0), again.result(1)) == before
    four.step(2)
    again.step(2)
    assert again.result(0) == four.result(0) and again.result(1) == four.result(1)
    four.end(0)
    four.end(1)
    torch.cuda.synchronize()
    assert int(four.ref.abs().sum()) == 0 and int(four.table.max()) == -1
    _begin(four, pre, 0, prompt)
    four.step(8)
    assert four.result(0) == res


def test_eos_ends_beams_and_refusals(model):
    from rngd_pd.engines.beam_decode import BeamDecodeEngine
    cfg, pre, m = model
    prompt = [(3 * j + 2) % SMALL.V for j in range(30)]
    free = _engine(model, beams=3, groups=1, pages=12, width=2)
    _begin(free, pre, 0, prompt)
    free.step(6)
    eos = free.result(0)[0][1][2]
    eng = _engine(model, beams=3, groups=1, pages=12, width=2, eos=eos)
    _begin(eng, pre, 0, prompt)
    eng.step(6)
    res = eng.result(0)
    ended = [t for _, t in res if t[-1] == eos]
    assert ended and all(eos not in t[:-1] for _, t in res)
    with pytest.raises(ValueError):
        eng.step(200)                       # more positions than a sequence's pages hold
    kv, _ = pre.prefill_kv_device(prompt)
    for bad in (lambda: eng.begin(0, [1] * 128, kv, pre.logits()), lambda: eng.begin(0, prompt, kv[:1], pre.logits()),
                lambda: eng.begin(0, prompt, kv, pre.logits()[:5]), lambda: BeamDecodeEngine(cfg, pre.w, beams=5, groups=4),
                lambda: BeamDecodeEngine(cfg, pre.w, beams=4, groups=4, eos=SMALL.V), lambda: free.result(0) and eng.end(1)):
        with pytest.raises((ValueError, IndexError)):
            bad()
    small = _engine(model, beams=3, groups=1, pages=2, width=2)
    _begin(small, pre, 0, prompt)
    small.step(2)
    with pytest.raises(RuntimeError):
        small.result(0)                     # two pages do not hold three beams


def test_compact_waits_for_the_steps_before_it(model):
    """Called with steps still queued and nothing synchronised, the count is that of the state after them."""
    cfg, pre, m = model
    prompt = [(5 * j + 1) % SMALL.V for j in range(70)]
    eng = _engine(model, beams=4, groups=2, pages=40, width=4)
    for n in (40, 20, 1):
        for g in (0, 1):
            _begin(eng, pre, g, prompt)
        eng.step(n)
        live = eng.compact()
        assert live == int((eng.ref > 0).sum()) == int(eng.table.max()) + 1 and live >= 5
        eng.end(1)
        assert eng.compact() == int((eng.ref > 0).sum()) < live


def _same(a, b):
    """Equal sequences; scores as close as another make-up of the batch leaves them."""
    return [t for _, t in a] == [t for _, t in b] and np.allclose([s for s, _ in a], [s for s, _ in b], rtol=0, atol=1e-4)


def test_a_shortage_concerns_its_own_search_alone(model):
    """A search that ran out of pages cannot give a result; others can, and the group can after a new begin."""
    cfg, pre, m = model
    prompt = [(3 * j + 2) % SMALL.V for j in range(30)]
    one = _engine(model, beams=3, groups=1, pages=12, width=2)
    _begin(one, pre, 0, prompt)
    one.step(5)
    want = one.result(0)
    eng = _engine(model, beams=3, groups=2, pages=4, width=2)
    _begin(eng, pre, 0, prompt)
    eng.step(1)                             # three pages held
    _begin(eng, pre, 1, prompt)             # the fourth: its beams cannot part
    eng.step(4)
    assert _same(eng.result(0), want)
    with pytest.raises(RuntimeError):
        eng.result(1)
    eng.step(2)
    with pytest.raises(RuntimeError):
        eng.result(1)                       # for good
    eng.result(0)
    eng.end(0)
    _begin(eng, pre, 1, prompt)
    eng.step(5)
    assert _same(eng.result(1), want)
    # a prompt that the pool cannot hold
    tiny = _engine(model, beams=2, groups=2, pages=2, width=4)
    _begin(tiny, pre, 0, [1] * 30)
    _begin(tiny, pre, 1, [1] * 90)
    assert len(tiny.result(0)) == 2
    with pytest.raises(RuntimeError):
        tiny.result(1)


def test_history_is_as_long_as_the_oldest_search(model):
    """Searches that overlap: steps before the oldest one still alive are forgotten, results are not."""
    cfg, pre, m = model
    prompt = [(5 * j + 1) % SMALL.V for j in range(20)]
    alone = _engine(model, beams=2, groups=1, pages=12, width=3)
    _begin(alone, pre, 0, prompt)
    alone.step(9)
    want = alone.result(0)
    eng = _engine(model, beams=2, groups=2, pages=24, width=3)
    _begin(eng, pre, 0, prompt)
    for i in range(6):                      # the groups in turn: one begins three steps after the other
        eng.step(3)
        _begin(eng, pre, (i + 1) % 2, prompt)
        eng.step(6)
        assert _same(eng.result(i % 2), want)
        assert len(eng.result((i + 1) % 2)[0][1]) == 7
        assert len(eng._steps) <= 9
        eng.end(i % 2)
        assert len(eng._steps) <= 6
        _begin(eng, pre, i % 2, prompt)     # begun anew without an end in between
        eng.step(9 - 6)
        assert _same(eng.result((i + 1) % 2), want)
        eng.end(i % 2)
        _begin(eng, pre, (i + 1) % 2, prompt)
        assert len(eng._steps) == 0
    eng.end(0)
    eng.end(1)
    eng.step(4)
    assert len(eng._steps) == 0


def test_engine_refuses_groups_and_steps_out_of_range(model):
    cfg, pre, m = model
    eng = _engine(model, beams=2, groups=2, pages=8, width=2)
    prompt = [1, 2, 3]
    _begin(eng, pre, 1, prompt)
    for bad in (lambda: eng.result(-1), lambda: eng.result(2), lambda: eng.end(-1), lambda: eng.step(-1)):
        with pytest.raises((ValueError, IndexError)):
            bad()
    eng.step(0)
    assert len(eng.result(1)) == 2 and len(eng.result(1)[0][1]) == 1


def test_a_device_wait_that_ran_out_spoils_every_search_alive(model, monkeypatch):
    """The library's status is read and cleared once; each search that was alive then has no result."""
    from rngd_pd import _lib
    cfg, pre, m = model
    eng = _engine(model, beams=2, groups=2, pages=8, width=2)
    for g in (0, 1):
        _begin(eng, pre, g, [1, 2, 3])
    eng.step(2)
    codes = [7, 0, 0, 0, 0, 0]              # as if a wait had run out in one of the steps
    monkeypatch.setattr(_lib, "device_status", lambda reset=True: codes.pop(0))
    for g in (0, 1, 0):
        with pytest.raises(RuntimeError):
            eng.result(g)
    _begin(eng, pre, 1, [1, 2, 3])
    eng.step(2)
    assert len(eng.result(1)) == 2
    with pytest.raises(RuntimeError):
        eng.result(0)


def test_engine_takes_windows_sinks_and_eos_beyond_32_bits(model):
    """They mean what they say (no window, all sinks, no eos), not what their lowest 32 bits do."""
    cfg, pre, m = model
    prompt = [(3 * j + 2) % SMALL.V for j in range(40)]
    res = []
    for kw in ({}, dict(window=2 ** 32 + 2), dict(window=2, sinks=2 ** 32), dict(window=2 ** 31 + 5, sinks=2 ** 31 + 1)):
        eng = _engine(model, beams=3, groups=1, pages=12, width=2, **kw)
        _begin(eng, pre, 0, prompt)
        eng.step(5)
        res.append(eng.result(0))
    assert all(_same(r, res[0]) for r in res)
    eos = res[0][0][1][2] - 2 ** 32
    eng = _engine(model, beams=3, groups=1, pages=12, width=2, eos=eos)
    _begin(eng, pre, 0, prompt)
    eng.step(5)
    assert eng.result(0) == res[0]
