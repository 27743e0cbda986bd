"""Plain numpy forms, in 64 bits, of the paged 4-bit cache and of the beam selection (test infrastructure)."""
import numpy as np

PAGE = 64


def encode(x):
    """x [..., HD] -> codes [..., HD], s, c [..., HD / 32] (float64 holding fp16 numbers), and how far each quotient is
    from a tie.  s and c are formed in fp32 and rounded to fp16, as the format has it; the rest is in 64 bits."""
    x = np.clip(x, -16384.0, 16384.0)  # keeps NaN
    g = x.reshape(*x.shape[:-1], -1, 32)
    lo, hi = g.min(-1), g.max(-1)
    with np.errstate(all="ignore"):
        lo4, hi4 = lo.astype(np.float32), hi.astype(np.float32)
        s4 = ((hi4 - lo4) * (np.float32(1) / np.float32(15))).astype(np.float16)
        c4 = (lo4 - np.float32(16) * s4.astype(np.float32)).astype(np.float16)
        s, c = s4.astype(np.float64), c4.astype(np.float64)
        t = (g - c[..., None]) / s[..., None] - 16
        u = np.where(s[..., None] > 0, np.clip(np.rint(t), 0, 15), 0)
        tie = np.where(s[..., None] > 0, np.abs(t - np.floor(t) - 0.5), 1.0)  # distance from a tie, in steps
    return u.reshape(x.shape), s, c, tie.reshape(x.shape)


def values(u, s, c):
    g = u.reshape(*u.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        return (s[..., None] * (16 + g) + c[..., None]).astype(np.float16).astype(np.float64).reshape(u.shape)


def decode_pool(pool):
    """pool [..., NKV, 4, 20 HD] uint8 -> K, V [..., NKV, 64, HD] float64, one dimension at a time."""
    HD = pool.shape[-1] // 20
    NG = HD // 32
    lead = pool.shape[:-2]
    K, V = np.empty(lead + (4, 16, HD)), np.empty(lead + (4, 16, HD))
    half = lambda off: np.ascontiguousarray(pool[..., off:off + 2]).view(np.float16)[..., 0].astype(np.float64)
    with np.errstate(all="ignore"):
        for key in range(16):
            for d in range(HD):
                j, r = d // 32, d % 32
                byte = key * HD // 2 + ((r // 8) * NG + j) * 4 + (r % 8) // 2
                u = (pool[..., byte] >> (4 * (r % 2))) & 15
                at = 16 * HD + (key * NG + j) * 4
                K[..., key, d] = (half(at) * (16.0 + u) + half(at + 2)).astype(np.float16)
                byte = 8 * HD + (((key // 8) * 8 + r // 4) * 8 + key % 8) * NG * 2 + j * 2 + (r % 4) // 2
                u = (pool[..., byte] >> (4 * (r % 2))) & 15
                at = 18 * HD + (((key // 8) * 4 + key % 8 // 2) * NG + j) * 8 + (key % 2) * 2
                V[..., key, d] = (half(at) * (16.0 + u) + half(at + 4)).astype(np.float16)
    return K.reshape(lead + (64, HD)), V.reshape(lead + (64, HD))


def visible(i, window, sinks):
    j = np.arange(i + 1) if i >= 0 else np.arange(0)
    return j if window == 0 else j[(j > i - window) | (j < sinks)]


def attend(q, K, V, table, lens, window, sinks, scale):
    """q [B, T, NH, HD]; K, V [P, NKV, 64, HD] -> out, and a bound on what fp32 arithmetic may be off by."""
    B, T, NH, HD = q.shape
    P, NKV = K.shape[:2]
    G = NH // NKV
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        for t in range(T):
            j = visible(int(lens[b]) - T + t, window, sinks)
            pg = np.array([table[b, x // PAGE] if x // PAGE < table.shape[1] else -1 for x in j], dtype=int)
            j, pg = j[(pg >= 0) & (pg < P)], pg[(pg >= 0) & (pg < P)]
            if len(j) == 0:
                continue
            for h in range(NH):
                k, v = K[pg, h // G, j % PAGE], V[pg, h // G, j % PAGE]
                s = (k @ q[b, t, h]) * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, t, h] = p @ v
                # the scores' rounding: HD + 8 roundings of 2^-23 of the sum of magnitudes, and as much again for
                # the maximum; the exponentials and sums: 64 roundings of 2^-23 of the largest value
                ds = (HD + 8) * 2.0 ** -23 * (np.abs(k) @ np.abs(q[b, t, h])).max() * scale
                bound[b, t, h] = (4 * ds + 64 * 2.0 ** -23) * np.abs(v).max()
    return out, bound


def fork(ref, table, lens, parents, room):
    """Lists of whole numbers -> ref, table, lens, short, copies [(src, dst, blocks)]."""
    P, R, W = len(ref), len(table), len(table[0])
    ref = list(ref)
    pages = lambda n: -(-n // PAGE)
    new, nl = [], []
    for r in range(R):
        p = parents[r]
        nl.append(lens[p] if p >= 0 else 0)
        new.append([table[p][c] if p >= 0 and c < pages(lens[p]) else -1 for c in range(W)])
    for row in table:
        for x in row:
            if x >= 0:
                ref[x] -= 1
    for row in new:
        for x in row:
            if x >= 0:
                ref[x] += 1
    tail = [new[r][pages(nl[r]) - 1] if parents[r] >= 0 and nl[r] % PAGE else -1 for r in range(R)]
    copy = [tail[r] >= 0 and (tail[r] in tail[:r] or ref[tail[r]] > tail.count(tail[r])) for r in range(R)]
    free = [p for p in range(P) if ref[p] == 0]
    short, copies = 0, []

    def give():
        nonlocal short
        if free:
            p = free.pop(0)
            ref[p] += 1
            return p
        short += 1
        return -1

    for r in range(R):
        if copy[r]:
            p = give()
            ref[tail[r]] -= 1
            new[r][pages(nl[r]) - 1] = p
            if p >= 0:
                copies.append((tail[r], p, -(-(nl[r] % PAGE) // 16)))
        if parents[r] >= 0:
            for c in range(pages(nl[r]), pages(nl[r] + room)):
                if c < W:
                    new[r][c] = give()
                else:
                    short += 1
    return ref, new, nl, short, copies


def select(logits, scores, done, W, eos):
    """float64 [R, V] -> per group the sorted candidates' scores and the choice."""
    R, V = logits.shape
    with np.errstate(all="ignore"):
        m = logits.max(1, keepdims=True)
        lse = m + np.log(np.exp(logits - m).sum(1, keepdims=True))
        sc = scores[:, None] + (logits - lse)
    carry = np.full((R, V), -np.inf)
    if 0 <= eos < V:
        carry[:, eos] = scores
    sc = np.where(done[:, None], carry, sc)
    sc = np.where(np.isnan(sc), -np.inf, sc).reshape(R // W, W * V)
    at = np.argsort(-sc, axis=1, kind="stable")[:, :W]
    best = np.take_along_axis(sc, at, 1)
    parent = at // V + W * np.arange(R // W)[:, None]
    token = at % V
    return best, parent, token, done[parent] | (token == eos), sc
