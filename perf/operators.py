"""Measured cases of the beam-search operators: the paged 4-bit KV cache (store, load, attention with
a sliding window and sinks), its pages (fork, compact) and the selection over beams and vocabulary.

`run` computes each in a plain form of elementary torch operations, or, where `own` is true, through
the package's entry points (rngd_pd.kv4, rngd_pd.beam).

Cache format.  A page holds 64 positions of one layer: uint8 [NKV][4][20 * HD], one 20 * HD byte block
per 16 positions of a kv head.  Along the head dimension every 32 values share a pair of fp16 numbers
(s, c), and a 4-bit code u stands for fp16(s * (16 + u) + c).  A block is
  K codes   [16 keys][t 0..3][j 0..NG-1][4 bytes]: nibble e of the word is dimension 32 j + 8 t + e;
  V codes   [2][g 0..7][8 keys][j 0..NG-1][2 bytes]: nibble e of the half word is dimension 32 j + 4 g + e;
  K scales  [16 keys][NG][s, c];
  V scales  [2][4 key pairs][NG][s of both keys, c of both keys],
with NG = HD / 32, the lowest nibble first.
"""
import math
import os
import sys

import torch

own = False

PAGE = 64
LIMIT = 16384.0  # values are held to this magnitude


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # attention of one short conversation: latency
        {"name": "attend 1x387", "op": "attend", "B": 1, "T": 1, "NH": 32, "NKV": 8, "HD": 128, "lo": 387, "hi": 387,
         "window": 0, "sinks": 0, "dtype": "bfloat16"},
        # the benchmark's decode step: 16 streams of 64 to 384 positions, queries in fp32
        {"name": "attend 16x384 fp32", "op": "attend", "B": 16, "T": 1, "NH": 32, "NKV": 8, "HD": 128, "lo": 64,
         "hi": 384, "window": 0, "sinks": 0, "dtype": "float32"},
        # five drafted tokens to verify per stream, heads of 64, only a window and four sinks visible
        {"name": "attend window 32x15001", "op": "attend", "B": 32, "T": 5, "NH": 16, "NKV": 4, "HD": 64, "lo": 901,
         "hi": 15001, "window": 1000, "sinks": 4, "dtype": "float16"},
        # long documents of unequal length
        {"name": "attend 8x65001", "op": "attend", "B": 8, "T": 1, "NH": 32, "NKV": 8, "HD": 128, "lo": 9001,
         "hi": 65001, "window": 0, "sinks": 0, "dtype": "bfloat16"},
        # the keys and values of one decode step, and a look at them
        {"name": "store 16x1", "op": "store", "L": 1, "B": 16, "T": 1, "lo": 1, "hi": 1, "NKV": 8, "HD": 128,
         "dtype": "bfloat16", "prefill": False},
        # a prompt of all layers out of the prefill engine's cache (512 positions wide)
        {"name": "store prompt 448", "op": "store", "L": 32, "B": 1, "T": 448, "lo": 448, "hi": 448, "NKV": 8,
         "HD": 128, "dtype": "bfloat16", "prefill": True},
        # one search of five beams over a small vocabulary of odd size
        {"name": "select 1x5x32003", "op": "select", "G": 1, "W": 5, "V": 32003, "dtype": "float32", "done": 1},
        # many searches over the large vocabulary
        {"name": "select 64x8x128256", "op": "select", "G": 64, "W": 8, "V": 128256, "dtype": "bfloat16", "done": 1},
        # beams of one engine's 16 lanes after a selection, all layers
        {"name": "fork 4x4", "op": "fork", "G": 4, "W": 4, "L": 32, "NKV": 8, "HD": 128, "lo": 101, "hi": 420,
         "ended": 0, "room": 1, "spare": 40},
        # many beams with long prompts, some searches at their end
        {"name": "fork 32x8", "op": "fork", "G": 32, "W": 8, "L": 8, "NKV": 8, "HD": 64, "lo": 501, "hi": 2000,
         "ended": 5, "room": 5, "spare": 300},
        # a few pages out of place
        {"name": "compact 12 of 300", "op": "compact", "L": 8, "P": 512, "live": 300, "move": 12, "R": 16,
         "NKV": 8, "HD": 64},
        # a pool left in pieces
        {"name": "compact 600 of 1300", "op": "compact", "L": 4, "P": 2048, "live": 1300, "move": 600, "R": 64,
         "NKV": 8, "HD": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "store", "store", "select", "select", "fork", "compact"])
    HD = rng.choice([64, 128, 128])
    if op == "attend":
        NH, NKV = rng.choice([(32, 8), (16, 4), (8, 8), (16, 2), (14, 2), (24, 8)])
        B, T = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 3, 4, 7])
        hi = _log(rng, 8, max(16, min(65000, 200000 * 8 * 128 // (B * NKV * HD))))
        return {"op": op, "B": B, "T": T, "NH": NH, "NKV": NKV, "HD": HD, "lo": rng.randint(1, hi), "hi": hi,
                "window": rng.choice([0, 0, _log(rng, 1, 4000)]), "sinks": rng.choice([0, 4, rng.randint(1, 150)]),
                "dtype": rng.choice(["bfloat16", "float16", "float32"])}
    if op == "store":
        NKV, L = rng.choice([2, 4, 8]), rng.choice([1, 1, 4, 16])
        B = _log(rng, 1, 32)
        T = _log(rng, 1, max(2, 14000 * 8 // (L * B * NKV)))
        return {"op": op, "L": L, "B": B, "T": T, "lo": rng.randint(1, T), "hi": T, "NKV": NKV, "HD": HD,
                "dtype": rng.choice(["bfloat16", "float16", "float32"]), "prefill": rng.random() < 0.5}
    if op == "select":
        W = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        V = _log(rng, 500, 150000)
        G = _log(rng, 1, max(2, min(64, 32000000 // (W * V))))
        return {"op": op, "G": G, "W": W, "V": V, "dtype": rng.choice(["bfloat16", "float16", "float32"]),
                "done": rng.randint(0, W // 2)}
    NKV = rng.choice([2, 4, 8])
    if op == "fork":
        G, W = _log(rng, 1, 24), rng.choice([2, 3, 4, 6, 8])
        hi = _log(rng, 10, max(20, min(4000, 250000 // (G * W))))
        return {"op": op, "G": G, "W": W, "L": rng.choice([1, 3, 4]), "NKV": NKV, "HD": HD, "lo": rng.randint(1, hi),
                "hi": hi, "ended": rng.randint(0, G // 2), "room": rng.choice([0, 1, 1, 3, 70]),
                "spare": rng.choice([3, G * W * 3])}
    P = _log(rng, 40, 2000)
    live = rng.randint(P // 4, P * 3 // 4)
    return {"op": op, "L": rng.choice([1, 2, 4]), "P": P, "live": live,
            "move": rng.randint(0, min(live, P - live) * 2 // 3), "R": _log(rng, 1, 64), "NKV": NKV, "HD": HD}


def _spread(lo, hi, n):
    """n lengths from lo to hi."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _block(HD):
    return 20 * HD


def _pages(n):
    return -(-n // PAGE)


def work(case):
    c, op = case, case["op"]
    if op == "attend":
        esz = 4 if c["dtype"] == "float32" else 2
        seen = pairs = 0
        for n in _spread(c["lo"], c["hi"], c["B"]):
            low = max(0, max(0, n - c["T"]) - c["window"] + 1) if c["window"] else 0
            seen += n - low + min(c["sinks"], low)
            for i in range(max(0, n - c["T"]), n):
                low = max(0, i - c["window"] + 1) if c["window"] else 0
                pairs += i + 1 - low + min(c["sinks"], low)
        io = 2 * c["B"] * c["T"] * c["NH"] * c["HD"] * esz
        return {"bytes": seen * c["NKV"] * c["HD"] * 5 // 4 + io, "flops": 4 * pairs * c["NH"] * c["HD"]}
    if op == "store":
        esz = 4 if c["dtype"] == "float32" else 2
        rows = c["L"] * c["NKV"] * sum(_spread(c["lo"], c["hi"], c["B"]))
        every = c["L"] * c["NKV"] * c["B"] * c["T"]
        return {"bytes": rows * c["HD"] * 2 * (esz + 0.625 * 2) + every * c["HD"] * 4, "flops": rows * c["HD"] * 2 * 8}
    if op == "select":
        esz = 4 if c["dtype"] == "float32" else 2
        n = c["G"] * c["W"] * c["V"]
        return {"bytes": n * esz + c["G"] * c["W"] * 18, "flops": 4 * n}
    if op == "fork":
        copied = held = 0
        for g, n in enumerate(_spread(c["lo"], c["hi"], c["G"])):
            held += c["W"] * _pages(n)
            if g >= c["ended"]:
                copied += (c["W"] - len(set(_children(c["W"])))) * -(-(n % PAGE) // 16)
        return {"bytes": 2 * copied * c["L"] * c["NKV"] * _block(c["HD"]) + 12 * held, "flops": 0}
    page = c["L"] * c["NKV"] * 4 * _block(c["HD"])
    return {"bytes": 2 * c["move"] * page + 8 * c["P"] + 8 * c["live"], "flops": 0}


def _children(W):
    """Which beams of a group the next ones come from: the good ones several times, some never."""
    return [i * i // W for i in range(W)]


# --------------------------------------------------------------------------------- the cache format
def _encode(x):
    """Codes (0..15) and the fp16 pair of every 32 values along the last dimension."""
    g = x.float().clamp(-LIMIT, LIMIT).unflatten(-1, (-1, 32))
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / 15.0).half()
    c = (lo - 16.0 * s.float()).half()
    t = (g - c.float().unsqueeze(-1)) / s.float().unsqueeze(-1)
    u = torch.where(s.unsqueeze(-1) > 0, (t.round() - 16.0).clamp(0, 15), 0.0).to(torch.uint8)
    return u, s, c


def _views(pool):
    """The four parts of every block of `pool` [..., 4, 20 * HD] as views."""
    HD = pool.shape[-1] // 20
    NG = HD // 32
    kc = pool[..., :8 * HD].unflatten(-1, (16, HD // 2))
    vc = pool[..., 8 * HD:16 * HD].unflatten(-1, (2, 8, 8, HD // 16))
    ks = pool[..., 16 * HD:18 * HD].view(torch.float16).unflatten(-1, (16, NG, 2))
    vs = pool[..., 18 * HD:].view(torch.float16).unflatten(-1, (2, 4, NG, 2, 2))
    return kc, vc, ks, vs


def _k_bytes(u):
    """[..., NG, 32] codes -> [..., HD / 2] bytes of a key."""
    w = u.unflatten(-1, (4, 4, 2)).transpose(-4, -3)  # [t][j][byte][nibble]
    return (w[..., 0] | (w[..., 1] << 4)).flatten(-3)


def _v_bytes(u):
    """[..., NG, 32] codes -> [..., 8, HD / 16] bytes of a value, by g."""
    w = u.unflatten(-1, (8, 2, 2)).transpose(-4, -3)  # [g][j][byte][nibble]
    return (w[..., 0] | (w[..., 1] << 4)).flatten(-2)


def _nibbles(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _value(u, s, c):
    """What codes stand for, [..., NG, 32]."""
    return (s.float().unsqueeze(-1) * (u + 16.0) + c.float().unsqueeze(-1)).half()


def _decode(pages):
    """pages [..., 4, 20 * HD] -> K and V [..., 64, HD] as fp16."""
    kc, vc, ks, vs = _views(pages)
    ku = _nibbles(kc).unflatten(-1, (4, -1, 8)).transpose(-3, -2).flatten(-2)  # [NG][32]
    k = _value(ku, ks[..., 0], ks[..., 1]).flatten(-2).flatten(-3, -2)
    vu = _nibbles(vc).unflatten(-1, (-1, 4))  # [2][g][key][j][4]
    vu = vu.permute(*range(vu.dim() - 5), -5, -3, -2, -4, -1).flatten(-2)  # [2][key][j][32]
    sc = vs.permute(*range(vs.dim() - 5), -5, -4, -1, -3, -2).flatten(-4, -3)  # [2][key][j][s, c]
    v = _value(vu, sc[..., 0], sc[..., 1]).flatten(-2).flatten(-4, -2)
    return k, v


def _fill_pages(pool, k, v):
    """Whole pages of `pool` [..., 4, 20 * HD] from K and V [..., 64, HD]."""
    kc, vc, ks, vs = _views(pool)
    u, s, c = _encode(k)
    kc.copy_(_k_bytes(u).unflatten(-2, (4, 16)))
    ks.copy_(torch.stack((s, c), -1).unflatten(-3, (4, 16)))
    u, s, c = _encode(v)
    vc.copy_(_v_bytes(u).unflatten(-3, (4, 2, 8)).transpose(-3, -2))
    w = torch.stack((s, c), -1).unflatten(-3, (4, 2, 4, 2))  # [4][2][t][parity][NG][s, c]
    vs.copy_(w.permute(*range(w.dim() - 4), -4, -2, -1, -3))


# --------------------------------------------------------------------------------------- the inputs
def _dtype(case):
    return getattr(torch, case["dtype"])


def _lengths(case, n, gen):
    v = torch.tensor(_spread(case["lo"], case["hi"], n), dtype=torch.int32, device="cuda")
    return v[torch.randperm(n, generator=gen, device="cuda")]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    perm = lambda n: torch.randperm(n, generator=gen, device="cuda").to(torch.int32)
    st = {"case": dict(c)}
    if c["op"] == "attend":
        B, NKV, HD, mp = c["B"], c["NKV"], c["HD"], _pages(c["hi"])
        P = B * mp
        # keys have a mean of their own in every dimension, as after a projection
        k = randn(P, NKV, PAGE, HD).add_(randn(1, NKV, 1, HD), alpha=1.5)
        pool = torch.empty(P, NKV, 4, _block(HD), dtype=torch.uint8, device="cuda")
        _fill_pages(pool, k, randn(P, NKV, PAGE, HD))
        del k
        st.update(pool=pool, table=perm(P).view(B, mp), lens=_lengths(c, B, gen),
                  q=(2.0 * randn(B, c["T"], c["NH"], HD)).to(_dtype(c)))
    elif c["op"] == "store":
        L, B, T, NKV, HD = c["L"], c["B"], c["T"], c["NKV"], c["HD"]
        if c["prefill"]:  # the prefill engine's layout: layer, K or V, head, position
            kv = randn(B, L, 2, NKV, T + 64, HD).to(_dtype(c))
            k, v = (kv[:, :, i, :, :T].permute(1, 0, 3, 2, 4) for i in (0, 1))
        else:
            k, v = (randn(L, B, T, NKV, HD).to(_dtype(c)) for _ in (0, 1))
        mp = _pages(T + 200)
        start = torch.randint(0, 200, (B,), generator=gen, device="cuda").to(torch.int32)
        st.update(k=k, v=v, start=start, count=_lengths(c, B, gen), table=perm(B * mp).view(B, mp),
                  pool=torch.zeros(L, B * mp, NKV, 4, _block(HD), dtype=torch.uint8, device="cuda"))
    elif c["op"] == "select":
        R = c["G"] * c["W"]
        done = torch.zeros(c["G"], c["W"], dtype=torch.bool, device="cuda")
        done[:, :c["done"]] = True
        done = done.gather(1, torch.rand(c["G"], c["W"], generator=gen, device="cuda").argsort(1)).reshape(R)
        st.update(logits=(3.0 * randn(R, c["V"])).to(_dtype(c)), scores=-12.0 + 2.0 * randn(R), done=done,
                  eos=c["V"] // 3)
    elif c["op"] == "fork":
        G, W = c["G"], c["W"]
        R, mp = G * W, _pages(c["hi"] + c["room"]) + 1
        lens = torch.tensor(_spread(c["lo"], c["hi"], G), dtype=torch.int32, device="cuda")
        n, shared = (lens + PAGE - 1) // PAGE, lens * 3 // 4 // PAGE
        col = torch.arange(mp, device="cuda")
        held = (col < n.view(G, 1, 1)).expand(G, W, mp)
        lead = torch.arange(W, device="cuda").view(1, W, 1) == 0
        first = held & (lead | (col >= shared.view(G, 1, 1)))  # the beams of a search share its first pages
        P = sum(_pages(n) + (W - 1) * (_pages(n) - n * 3 // 4 // PAGE) for n in _spread(c["lo"], c["hi"], G)) + c["spare"]
        ids = perm(P)
        at = (first.reshape(-1).cumsum(0) - 1).view(G, W, mp)
        at = torch.where(first, at, at[:, :1])
        table = torch.where(held, ids[at.clamp(0)], -1).view(R, mp)
        ref = torch.zeros(P, dtype=torch.int32, device="cuda")
        ref.scatter_add_(0, table.clamp(0).reshape(-1).long(), (table >= 0).reshape(-1).int())
        child = torch.tensor(_children(W), device="cuda").expand(G, W)
        names, order = (torch.rand(G, W, generator=gen, device="cuda").argsort(1) for _ in (0, 1))
        par = names.gather(1, child.gather(1, order)) + W * torch.arange(G, device="cuda").view(G, 1)
        par[:c["ended"]] = -1
        st.update(table=table.contiguous(), ref=ref, lens=lens.repeat_interleave(W).contiguous(),
                  parents=par.to(torch.int32).reshape(R).contiguous(), pool=_random_pool(c, P, gen))
    else:
        P, live, move, R = c["P"], c["live"], c["move"], c["R"]
        low = torch.randperm(live, generator=gen, device="cuda")[:live - move]
        high = live + torch.randperm(P - live, generator=gen, device="cuda")[:move]
        ids = torch.cat((low, high))[torch.randperm(live, generator=gen, device="cuda")].to(torch.int32)
        mp = -(-live // R)
        table = torch.full((R * mp,), -1, dtype=torch.int32, device="cuda")
        table[:live] = ids
        ref = torch.zeros(P, dtype=torch.int32, device="cuda")
        ref[ids.long()] = 1 + (torch.rand(live, generator=gen, device="cuda") < 0.2).to(torch.int32)
        st.update(table=table.view(R, mp), ref=ref, pool=_random_pool(c, P, gen))
    return st


def _random_pool(c, P, gen):
    n = c["L"] * P * c["NKV"] * 4 * _block(c["HD"])
    words = torch.randint(-2 ** 62, 2 ** 62, (n // 8,), generator=gen, device="cuda", dtype=torch.int64)
    return words.view(torch.uint8).view(c["L"], P, c["NKV"], 4, _block(c["HD"]))


# -------------------------------------------------------------------------------------- the passes
def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _package():
    at = os.path.join(os.getcwd(), "rngd-pd_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from rngd_pd import beam, kv4
    return kv4, beam


def _own_attend(s):
    kv4, _ = _package()
    c = s["case"]
    return kv4.attention(s["q"], s["pool"], s["table"], s["lens"], window=c["window"], sinks=c["sinks"])


def _own_store(s):
    kv4, _ = _package()
    kv4.store(s["pool"], s["table"], s["start"], s["k"], s["v"], count=s["count"])
    return kv4.load(s["pool"], s["table"], s["start"], s["case"]["T"], count=s["count"])


def _own_select(s):
    _, beam = _package()
    return beam.select(s["logits"], s["scores"], s["done"], s["case"]["W"], s["eos"])


def _own_fork(s):
    kv4, _ = _package()
    ref, table, lens, short = kv4.fork(s["pool"], s["ref"], s["table"], s["lens"], s["parents"],
                                       room=s["case"]["room"])
    return ref, table, lens, short, s["pool"].view(torch.int32)


def _own_compact(s):
    kv4, _ = _package()
    ref, table, live = kv4.compact(s["pool"], s["ref"], s["table"])
    return ref, table, live, s["pool"].view(torch.int32)


_OWN = {"attend": _own_attend, "store": _own_store, "select": _own_select, "fork": _own_fork,
        "compact": _own_compact}


def _plain_attend(s):
    """softmax(q K^T / sqrt(HD)) V over the visible positions, all of a table's pages at once."""
    c, q, lens = s["case"], s["q"], s["lens"].view(-1, 1, 1)
    B, T, NH, HD = q.shape
    NKV, G, W = c["NKV"], c["NH"] // c["NKV"], c["window"]
    K, V = (x.transpose(1, 2).flatten(2, 3).float() for x in _decode(s["pool"][s["table"].long()]))
    S = K.shape[2]
    j = torch.arange(S, device=q.device).view(1, 1, S)
    i = lens - T + torch.arange(T, device=q.device).view(1, T, 1)
    seen = j <= i
    if W:
        seen = seen & ((j > i - W) | (j < c["sinks"]))
    x = q.float().view(B, T, NKV, G, HD).permute(0, 2, 3, 1, 4).flatten(2, 3)
    a = (x @ K.transpose(2, 3)) * (1.0 / math.sqrt(HD))
    a = a.view(B, NKV, G, T, S).masked_fill(~seen.view(B, 1, 1, T, S), -math.inf)
    m = a.amax(-1, keepdim=True)
    p = (a - m.masked_fill(m == -math.inf, 0.0)).exp_()
    del a
    l = p.sum(-1, keepdim=True)
    V = V.masked_fill((j >= lens).view(B, 1, S, 1), 0.0)
    o = (p.view(B, NKV, G * T, S) @ V).view(B, NKV, G, T, HD)
    o = torch.where(l > 0, o / l, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, NH, HD).to(q.dtype)


def _plain_store(s):
    """Quantises the counted rows, scatters them over their pages, and gathers them again."""
    pool, table, k, v = s["pool"], s["table"], s["k"], s["v"]
    L, B, T, NKV, HD = k.shape
    t = torch.arange(T, device=k.device)
    there = t < s["count"].view(B, 1)
    pos = s["start"].view(B, 1) + t
    page = table.gather(1, (pos // PAGE).long()).long()
    b, t = there.nonzero(as_tuple=True)
    l, h = torch.arange(L, device=k.device).view(L, 1, 1), torch.arange(NKV, device=k.device)
    pg, blk, key = (x[b, t].long().view(-1, 1) for x in (page, pos % PAGE // 16, pos % 16))
    kc, vc, ks, vs = _views(pool)
    u, sk, ck = _encode(k[:, b, t])
    kc[l, pg, h, blk, key] = _k_bytes(u)
    ks[l, pg, h, blk, key] = torch.stack((sk, ck), -1)
    u, sv, cv = _encode(v[:, b, t])
    vc[l, pg, h, blk, key // 8, :, key % 8] = _v_bytes(u)
    vs[l, pg, h, blk, key // 8, key % 8 // 2, :, :, key % 2] = torch.stack((sv, cv), -1)
    rows = table.shape[1] * PAGE
    at = torch.where(there, pos, 0).long()
    at = at.view(1, B, T, 1, 1).expand(L, B, T, NKV, HD)
    K, V = (x.permute(0, 1, 2, 4, 3, 5).reshape(L, B, rows, NKV, HD) for x in _decode(pool[:, table.long()]))
    keep = there.view(1, B, T, 1, 1)
    return K.gather(2, at).masked_fill(~keep, 0.0), V.gather(2, at).masked_fill(~keep, 0.0)


def _plain_select(s):
    """The W best of a group's W * V continuations, ties to the lowest place."""
    c, done = s["case"], s["done"].view(-1, 1)
    G, W, V = c["G"], c["W"], c["V"]
    x = s["logits"].float()
    m = x.amax(1, keepdim=True)
    lse = m + (x - m).exp_().sum(1, keepdim=True).log_()
    sc = s["scores"].view(-1, 1) + (x - lse)
    is_eos = torch.arange(V, device=x.device) == s["eos"]
    sc = torch.where(done, torch.where(is_eos, s["scores"].view(-1, 1), -math.inf), sc)
    sc = sc.masked_fill(sc.isnan(), -math.inf).view(G, W * V) + 0.0
    bits = sc.view(torch.int32).long()
    key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF) - 1) << 32
    key += 0xFFFFFFFF - torch.arange(W * V, device=x.device)
    at = 0xFFFFFFFF - (key.topk(W, 1).values & 0xFFFFFFFF)
    parent = at // V + W * torch.arange(G, device=x.device).view(G, 1)
    token = at % V
    return (sc.gather(1, at), parent.to(torch.int32), token.to(torch.int32),
            s["done"][parent] | (token == s["eos"]))


def _count(ref, table, sign):
    there = table >= 0
    return ref.scatter_add(0, table.clamp(0).reshape(-1).long(), sign * there.reshape(-1).to(torch.int32))


def _plain_fork(s):
    """Row r goes on as row parents[r] (none: ended); shared last pages are copied, `room` positions made."""
    pool, ref, table, par, room = s["pool"], s["ref"], s["table"], s["parents"].long(), s["case"]["room"]
    (P,), (R, mp) = ref.shape, table.shape
    dev = ref.device
    on = par >= 0
    lens = torch.where(on, s["lens"][par.clamp(0)], 0)
    n = (lens + PAGE - 1) // PAGE
    col = torch.arange(mp, device=dev)
    new = torch.where(col < n.view(R, 1), table[par.clamp(0)], -1)
    ref = _count(_count(ref, table, -1), new, 1)
    # the last page, where it is partly filled: the first of its rows keeps it unless others hold it too
    part = on & (lens % PAGE != 0)
    tail = torch.where(part, new.gather(1, (n - 1).clamp(0).view(R, 1).long()).view(R), -1)
    same = (tail.view(R, 1) == tail.view(1, R)) & part
    lower = (same & (torch.arange(R, device=dev) < torch.arange(R, device=dev).view(R, 1))).any(1)
    copy = part & (lower | (ref[tail.clamp(0).long()] > same.sum(1)))
    n2 = torch.where(on, (lens + room + PAGE - 1) // PAGE, 0)
    last = n2.clamp(max=mp)
    want = copy.int() + (last - n)
    base = want.cumsum(0) - want
    free = torch.where(ref == 0, 0, P) + torch.arange(P, device=dev)
    free = free.sort().values
    free = torch.where(free < P, free, -1).to(torch.int32)
    pick = lambda at: torch.where(at < P, free[at.clamp(max=P - 1)], -1)
    given = torch.where(copy, pick(base), -1)
    ref = ref.scatter_add(0, tail.clamp(0).long(), -copy.int())
    more = (col >= n.view(R, 1)) & (col < last.view(R, 1))
    new = torch.where(more, pick((base + copy).view(R, 1) + col - n.view(R, 1)), new)
    new = torch.where(copy.view(R, 1) & (col == n.view(R, 1) - 1), given.view(R, 1), new)
    ref = _count(_count(ref, given, 1), torch.where(more, new, -1), 1)
    short = (n2 - last).sum() + (copy & (given < 0)).sum() + (more & (new < 0)).sum()
    src, dst = tail[given >= 0].long(), given[given >= 0].long()
    blocks = ((lens % PAGE + 15) // 16)[given >= 0].view(-1, 1, 1, 1)
    filled = torch.arange(4, device=dev).view(4, 1) < blocks
    pool[:, dst] = torch.where(filled, pool[:, src], pool[:, dst])
    return ref, new, lens, short.to(torch.int32).view(1), pool.view(torch.int32)


def _plain_compact(s):
    """The live pages above their own number move into the free places below it, lowest to lowest."""
    pool, ref, table = s["pool"], s["ref"], s["table"]
    P = ref.shape[0]
    at = torch.arange(P, device=ref.device)
    live = ref > 0
    n = live.sum()
    src, dst = (live & (at >= n)).nonzero().view(-1), (~live & (at < n)).nonzero().view(-1)
    to = at.to(torch.int32)
    to[src] = dst.to(torch.int32)
    new = ref.clone()
    new[dst], new[src] = ref[src], 0
    pool[:, dst] = pool[:, src]
    table = torch.where(table >= 0, to[table.clamp(0).long()], -1)
    return new, table, n.to(torch.int32).view(1), pool.view(torch.int32)


_PLAIN = {"attend": _plain_attend, "store": _plain_store, "select": _plain_select, "fork": _plain_fork,
          "compact": _plain_compact}


# ------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # pages are moved: nothing is computed but whole numbers
    s = prepare(case, seed)
    if case["op"] == "attend":
        return torch.stack([_exact_stream(s, b) for b in range(case["B"])])
    if case["op"] == "store":
        there = torch.arange(case["T"], device="cuda") < s["count"].view(-1, 1)
        return tuple(_exact_kept(s[x], there) for x in ("k", "v"))
    return torch.stack([_exact_best(s, g) for g in range(case["G"])]), None, None, None


def _stands_for(words, at, s, c):
    u = ((words >> (4 * at)) & 15).double()
    return (s.double() * (16.0 + u) + c.double()).half().double()


def _exact_page(page, HD):
    """K and V [NKV, 64 n, HD] of pages [n, NKV, 4, 20 HD], each dimension looked up in its word."""
    NG = HD // 32
    n, NKV = page.shape[:2]
    d = torch.arange(HD, device=page.device)
    j, r = d // 32, d % 32
    kw = page[..., :8 * HD].contiguous().view(torch.int32).view(n, NKV, 4, 16, HD // 8)[..., (r // 8) * NG + j]
    sc = page[..., 16 * HD:18 * HD].contiguous().view(torch.float16).view(n, NKV, 4, 16, NG, 2)[..., j, :]
    K = _stands_for(kw.long() & 0xFFFFFFFF, r % 8, sc[..., 0], sc[..., 1])
    vh = page[..., 8 * HD:16 * HD].contiguous().view(torch.int16).view(n, NKV, 4, 2, 8, 8, NG)
    vh = vh.transpose(4, 5)[..., r // 4, j]
    vs = page[..., 18 * HD:].contiguous().view(torch.float16).view(n, NKV, 4, 2, 4, NG, 2, 2).movedim(-1, 5)
    vs = vs.reshape(n, NKV, 4, 2, 8, NG, 2)[..., j, :]
    V = _stands_for(vh.long() & 0xFFFF, r % 4, vs[..., 0], vs[..., 1])
    return (x.reshape(n, NKV, PAGE, HD).transpose(0, 1).reshape(NKV, n * PAGE, HD) for x in (K, V))


def _exact_stream(s, b):
    c, q = s["case"], s["q"][b].double()
    T, NH, HD = q.shape
    n, W = int(s["lens"][b]), c["window"]
    K, V = _exact_page(s["pool"][s["table"][b, :_pages(n)].long()], HD)
    at = n - T + torch.arange(T, device=q.device).view(T, 1)
    past = at - torch.arange(K.shape[1], device=q.device)  # how far back each position lies
    hidden = past < 0
    if W:
        hidden = hidden | ((past >= W) & (torch.arange(K.shape[1], device=q.device) >= c["sinks"]))
    a = torch.einsum("tkgd,ksd->kgts", q.view(T, c["NKV"], -1, HD), K) / math.sqrt(HD)
    w = torch.softmax(a.masked_fill(hidden, -math.inf), -1).masked_fill(hidden, 0.0)
    return torch.einsum("kgts,ksd->tkgd", w, V).reshape(T, NH, HD)


def _exact_kept(x, there):
    g = x.double().clamp(-LIMIT, LIMIT).unflatten(-1, (-1, 32))
    lo, hi = g.min(-1).values, g.max(-1).values
    step = ((hi - lo) / 15).half().double()
    c = (lo - 16 * step).half().double()
    step, c = step.unsqueeze(-1), c.unsqueeze(-1)
    u = (((g - c) / step).round() - 16).clamp(0, 15)
    y = torch.where(step > 0, step * (16 + u) + c, c).half().double().flatten(-2)
    return y * there.view(1, *there.shape, 1, 1)


def _exact_best(s, g):
    c = s["case"]
    W = c["W"]
    r = slice(g * W, (g + 1) * W)
    before = s["scores"][r].double().view(W, 1)
    sc = torch.log_softmax(s["logits"][r].double(), 1) + before
    carry = torch.full_like(sc, -math.inf)
    carry[:, s["eos"]:s["eos"] + 1] = before
    return torch.where(s["done"][r].view(W, 1), carry, sc).reshape(-1).topk(W).values
