"""Measured cases of the 8-bit linear layers: rows and weights quantised to e4m3 with a scale for each 128
values or each 128 x 128 block, the RMS norm that adds the residual and writes such rows, the matrix product
of such operands, and the gate and up projections with SwiGLU, whose result is quantised again.

`run` computes each in a plain form of elementary torch operations, or, where `own` is true, through the
package's entry points (rngd_pd.fp8).

Format.  A row of K values has ceil(K / 128) scales in fp32, one for each 128 values from the left; a weight
[N, K] has ceil(N / 128) x ceil(K / 128) of them.  With amax the largest magnitude of a group,
scale = max(amax, 2^-100) / 448, and a value x is held as e4m3(x * (448 / max(amax, 2^-100))).
"""
import math
import os
import sys

import torch

own = False

GROUP = 128
MOST = 448.0        # the largest number in e4m3
LEAST = 2.0 ** -100  # groups whose magnitudes are all below it are scaled by it
EPS = 1e-5


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the norm of one decode step of 16 streams, the residual held in fp32
        {"name": "norm 16x4096 fp32", "op": "norm", "T": 16, "K": 4096, "dtype": "float32", "add": True},
        # a prompt's rows, of a width that ends inside a group, without a residual
        {"name": "norm 1001x4104 fp16", "op": "norm", "T": 1001, "K": 4104, "dtype": "float16", "add": False},
        # many prompts at once
        {"name": "norm 8192x4096", "op": "norm", "T": 8192, "K": 4096, "dtype": "bfloat16", "add": True},
        # the attention's output of a decode step, before its projection
        {"name": "rows 16x4096 fp32", "op": "rows", "T": 16, "K": 4096, "dtype": "float32"},
        # the same of many prompts
        {"name": "rows 8191x4096", "op": "rows", "T": 8191, "K": 4096, "dtype": "bfloat16"},
        # one projection of a checkpoint as it is loaded
        {"name": "weight 14336x4096", "op": "weight", "N": 14336, "K": 4096, "dtype": "bfloat16"},
        # the attention's output projection for a single token, onto the residual: latency
        {"name": "matmul 1x4096x4096", "op": "matmul", "M": 1, "N": 4096, "K": 4096, "dtype": "bfloat16", "add": True},
        # the logits of a decode step
        {"name": "matmul 16x128256x4096 fp32", "op": "matmul", "M": 16, "N": 128256, "K": 4096, "dtype": "float32",
         "add": False},
        # one prompt's queries, keys and values
        {"name": "matmul 333x6144x4096 fp16", "op": "matmul", "M": 333, "N": 6144, "K": 4096, "dtype": "float16",
         "add": False},
        # the down projection of many prompts, onto the residual
        {"name": "matmul 8192x4096x14336", "op": "matmul", "M": 8192, "N": 4096, "K": 14336, "dtype": "bfloat16",
         "add": True},
        # gate and up of a decode step
        {"name": "swiglu 16x14336x4096", "op": "swiglu", "M": 16, "N": 14336, "K": 4096},
        # gate and up of several prompts
        {"name": "swiglu 4096x14336x4096", "op": "swiglu", "M": 4096, "N": 14336, "K": 4096},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: whole groups, a multiple of 16 or any number."""
    n = _log(rng, lo, hi)
    m = rng.choice([128, 128, 16, 1])
    return max(m, n // m * m)


def draw(rng):
    op = rng.choice(["norm", "norm", "rows", "weight", "matmul", "matmul", "matmul", "matmul", "swiglu", "swiglu"])
    kind = rng.choice(["bfloat16", "float16", "float32"])
    if op in ("norm", "rows"):
        K = _width(rng, 64, 16384)
        c = {"op": op, "T": _log(rng, 1, max(2, 16000000 // K)), "K": K, "dtype": kind}
        if op == "norm":
            c["add"] = rng.random() < 0.6
        return c
    if op == "weight":
        K = _width(rng, 64, 16384)
        return {"op": op, "N": _log(rng, 100, max(200, 50000000 // K)), "K": K, "dtype": kind}
    # operands of a product start on 16 bytes row by row, whatever their width
    K, N = _width(rng, 64, 16384), _width(rng, 64, 30000)
    if N * K > 2 ** 27:
        N = 2 ** 27 // K
    if op == "matmul":
        M = _log(rng, 1, max(2, min(8192, 400000000000 // (N * K), 50000000 // N)))
        return {"op": op, "M": M, "N": N, "K": K, "dtype": kind, "add": rng.random() < 0.5}
    M = _log(rng, 1, max(2, min(8192, 200000000000 // (N * K), 50000000 // N)))
    return {"op": op, "M": M, "N": N, "K": K}


def _groups(n):
    return -(-n // GROUP)


def _size(case):
    return 4 if case["dtype"] == "float32" else 2


def work(case):
    c, op = case, case["op"]
    if op == "norm":
        n = c["T"] * c["K"]
        moved = n * _size(c) * (3 if c["add"] else 1) + n + 4 * c["T"] * _groups(c["K"]) + c["K"] * _size(c)
        return {"bytes": moved, "flops": 8 * n}
    if op == "rows":
        n = c["T"] * c["K"]
        return {"bytes": n * (_size(c) + 1) + 4 * c["T"] * _groups(c["K"]), "flops": 3 * n}
    if op == "weight":
        n = c["N"] * c["K"]
        return {"bytes": n * (_size(c) + 1) + 4 * _groups(c["N"]) * _groups(c["K"]), "flops": 3 * n}
    M, N, K = c["M"], c["N"], c["K"]
    rows = M * K + 4 * M * _groups(K)
    kept = N * K + 4 * _groups(N) * _groups(K)
    if op == "matmul":
        return {"bytes": rows + kept + M * N * _size(c) * (2 if c["add"] else 1), "flops": 2 * M * N * K}
    return {"bytes": rows + 2 * kept + M * N + 4 * M * _groups(N), "flops": 4 * M * N * K}


# --------------------------------------------------------------------------------------- the inputs
def _dtype(case):
    return getattr(torch, case["dtype"])


def _padded(x, by):
    """Columns of zeros up to a multiple of `by`."""
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % by))


def _quantise_rows(x):
    """e4m3 [T, K] and fp32 [T, G] of x [T, K] in fp32."""
    K = x.shape[1]
    g = _padded(x, GROUP).unflatten(1, (-1, GROUP))
    amax = g.abs().amax(-1).clamp(min=LEAST)
    q = (g * (MOST / amax).unsqueeze(-1)).clamp(-MOST, MOST).to(torch.float8_e4m3fn)
    return q.flatten(1)[:, :K], amax / MOST


def _quantise_blocks(w):
    """e4m3 [N, K] and fp32 [NB, G] of w [N, K]."""
    N, K = w.shape
    g = torch.nn.functional.pad(w.float(), (0, -K % GROUP, 0, -N % GROUP))
    g = g.unflatten(1, (-1, GROUP)).unflatten(0, (-1, GROUP))
    amax = g.abs().amax((1, 3)).clamp(min=LEAST)
    q = (g * (MOST / amax).view(amax.shape[0], 1, -1, 1)).clamp(-MOST, MOST).to(torch.float8_e4m3fn)
    return q.flatten(2).flatten(0, 1)[:N, :K], amax / MOST


def _aligned(q):
    """The same values in rows that start on 16 bytes."""
    N, K = q.shape
    held = torch.zeros(N, K + -K % 16, dtype=torch.uint8, device=q.device)
    held[:, :K] = q.view(torch.uint8)
    return held.view(torch.float8_e4m3fn)[:, :K]


def _activations(T, K, gen):
    """Rows as a transformer has them: each of its own size, a few channels much larger than the rest."""
    x = torch.randn(T, K, generator=gen, device="cuda")
    x *= torch.rand(T, 1, generator=gen, device="cuda") + 0.5
    loud = torch.randint(0, K, (max(1, K // 500),), generator=gen, device="cuda")
    x[:, loud] *= 12.0
    return x


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    st = {"case": dict(c)}
    if c["op"] in ("norm", "rows"):
        st["x"] = _activations(c["T"], c["K"], gen).to(_dtype(c))
        if c["op"] == "norm":
            st["weight"] = (1.0 + 0.2 * randn(c["K"])).to(_dtype(c))
            st["residual"] = _activations(c["T"], c["K"], gen).to(_dtype(c)) if c["add"] else None
        return st
    if c["op"] == "weight":
        st["w"] = (0.02 * randn(c["N"], c["K"])).to(_dtype(c))
        return st
    q, s = _quantise_rows(_activations(c["M"], c["K"], gen))
    st.update(a=_aligned(q), a_scale=s)
    for name in ("b",) if c["op"] == "matmul" else ("gate", "up"):
        q, s = _quantise_blocks((0.02 * randn(c["N"], c["K"])).to(torch.bfloat16))
        st.update({name: _aligned(q), name + "_scale": s})
    if c["op"] == "matmul":
        st["add"] = _activations(c["M"], c["N"], gen).to(_dtype(c)) if c["add"] else None
    return st


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
    from rngd_pd import fp8
    return fp8


def _own_norm(s):
    q, scale, total = _package().rms_norm(s["x"], s["weight"], EPS, residual=s["residual"])
    return (q, scale) if total is None else (q, scale, total)


def _own_rows(s):
    return _package().quantize(s["x"])


def _own_weight(s):
    return _package().quantize_weight(s["w"])


def _own_matmul(s):
    return _package().matmul(s["a"], s["a_scale"], s["b"], s["b_scale"], dtype=_dtype(s["case"]), add=s["add"])


def _own_swiglu(s):
    return _package().matmul_swiglu(s["a"], s["a_scale"], s["gate"], s["gate_scale"], s["up"], s["up_scale"])


_OWN = {"norm": _own_norm, "rows": _own_rows, "weight": _own_weight, "matmul": _own_matmul, "swiglu": _own_swiglu}


def _plain_norm(s):
    """The residual's sum is rounded to its type, and what is normalised is that sum."""
    x = s["x"].float()
    total = None
    if s["residual"] is not None:
        total = (x + s["residual"].float()).to(s["x"].dtype)
        x = total.float()
    y = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * s["weight"].float()
    q, scale = _quantise_rows(y)
    return (q, scale) if total is None else (q, scale, total)


def _plain_rows(s):
    return _quantise_rows(s["x"].float())


def _plain_weight(s):
    return _quantise_blocks(s["w"])


def _rows_of(q, s):
    return q.float() * s.repeat_interleave(GROUP, 1)[:, :q.shape[1]]


def _weight_of(q, s):
    N, K = q.shape
    return q.float() * s.repeat_interleave(GROUP, 0)[:N].repeat_interleave(GROUP, 1)[:, :K]


def _plain_matmul(s):
    y = _rows_of(s["a"], s["a_scale"]) @ _weight_of(s["b"], s["b_scale"]).t()
    if s["add"] is not None:
        y = y + s["add"].float()
    return y.to(_dtype(s["case"]))


def _plain_swiglu(s):
    a = _rows_of(s["a"], s["a_scale"])
    g = a @ _weight_of(s["gate"], s["gate_scale"]).t()
    u = a @ _weight_of(s["up"], s["up_scale"]).t()
    return _quantise_rows(g / (1.0 + torch.exp(-g)) * u)


_PLAIN = {"norm": _plain_norm, "rows": _plain_rows, "weight": _plain_weight, "matmul": _plain_matmul,
          "swiglu": _plain_swiglu}


# ------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """What is held in 8 bits is given as it is before its rounding, in units of its scale."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x, total = s["x"].double(), None
        if s["residual"] is not None:
            total = x + s["residual"].double()
            x = total.to(s["x"].dtype).double()  # the sum as it is stored
        rms = (torch.linalg.vector_norm(x, dim=1) ** 2 / x.shape[1] + EPS).sqrt()
        held = _exact_held(x / rms.view(-1, 1) * s["weight"].double())
        return held if total is None else (*held, total)
    if op == "rows":
        return _exact_held(s["x"].double())
    if op == "weight":
        return _exact_blocks(s["w"].double())
    if op == "matmul":
        y = _exact_product(s["a"], s["a_scale"], s["b"], s["b_scale"])
        return y if s["add"] is None else y + s["add"].double()
    g = _exact_product(s["a"], s["a_scale"], s["gate"], s["gate_scale"])
    u = _exact_product(s["a"], s["a_scale"], s["up"], s["up_scale"])
    return _exact_held(g * torch.sigmoid(g) * u)


def _exact_held(y):
    K = y.shape[1]
    most = torch.stack([p.abs().max(1).values for p in y.split(GROUP, 1)], 1).clamp(min=LEAST)
    at = torch.arange(K, device=y.device) // GROUP
    return y * MOST / most[:, at], most / MOST


def _exact_blocks(w):
    most = torch.stack([torch.stack([b.abs().max() for b in p.split(GROUP, 1)]) for p in w.split(GROUP, 0)])
    most = most.clamp(min=LEAST)
    n, k = (torch.arange(d, device=w.device) // GROUP for d in w.shape)
    return w * MOST / most[n][:, k], most / MOST


def _exact_product(a, a_scale, b, b_scale):
    """The sum over the groups of (scale of the row * scale of the block) * (the group's products)."""
    k = torch.arange(a.shape[1], device=a.device) // GROUP
    n = torch.arange(b.shape[0], device=a.device) // GROUP
    x = a.double() * a_scale.double()[:, k]
    w = b.double() * b_scale.double()[n][:, k]
    return torch.einsum("mk,nk->mn", x, w)
