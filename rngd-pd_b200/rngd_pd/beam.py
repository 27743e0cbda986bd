"""Beam search's selection over beams and vocabulary.

The reference decodes greedily (greedy_tokens, src/rngd_pd/engines/decode_batch.py:162-171); this is the same
step for a search that keeps the W best continuations of each prompt.  The parents it returns are what
rngd_pd.kv4.fork takes to reorder the sequences.
"""
import torch

from rngd_pd import _lib

MAX_BEAMS = 32
_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_select = _lib.lib.rngd_beam_select


def _vector(name, t, dt, n, dev):
    if t.dtype is not dt or t.shape != (n,) or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dt} [{n}] tensor on {dev}, got {tuple(t.shape)} {t.dtype}")


def select(logits, scores, done, beams, eos=-1):
    """Of each group's beams x V continuations the `beams` best by scores + log_softmax(logits).

    logits: [R, V] bfloat16, float16 or float32 (rows may lie apart), rows g * beams .. of group g;
    scores: float32 [R], the beams' own; done: bool [R].  A beam that is done goes on with `eos` alone, at its own
    score (eos < 0: none ends, and a beam that is done is lost).  NaN counts as -inf.  Equal scores: the lowest row,
    then the lowest token; but a row takes part with its `beams` largest logits alone (equal ones: the lowest
    tokens), so where logits that differ round to one score, its smaller ones may stay behind.
    Returns, best first, [R / beams, beams]: scores float32, parents int32 (rows), tokens int32, done bool."""
    if logits.dim() != 2 or logits.dtype not in _DT or not logits.is_cuda:
        raise ValueError(f"logits must be a CUDA matrix of bfloat16, float16 or float32, got {tuple(logits.shape)} "
                         f"{logits.dtype} on {logits.device}")
    R, V = logits.shape
    dev = logits.device
    if not 1 <= beams <= MAX_BEAMS or R % beams:
        raise ValueError(f"beams={beams}: 1..{MAX_BEAMS}, and {R} rows must be whole groups")
    if V < beams or V * beams >= 2 ** 31 or (V > 1 and logits.stride(1) != 1) or (R > 1 and logits.stride(0) < V):
        raise ValueError(f"logits {tuple(logits.shape)} strides {logits.stride()}: rows must be contiguous, at least "
                         f"{beams} wide and not overlap")
    _vector("scores", scores, torch.float32, R, dev)
    _vector("done", done, torch.bool, R, dev)
    if eos >= V:
        raise ValueError(f"eos={eos} outside the vocabulary of {V}")
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return select(logits, scores, done, beams, eos)
    shape = (R // beams, beams)
    out = torch.empty(shape, dtype=torch.float32, device=dev)
    parents = torch.empty(shape, dtype=torch.int32, device=dev)
    tokens = torch.empty_like(parents)
    ended = torch.empty(shape, dtype=torch.bool, device=dev)
    need = _lib.workspace_bytes("rngd_beam_workspace", _DT[logits.dtype], R, V, beams)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _lib.check(_select(logits.data_ptr(), _DT[logits.dtype], logits.stride(0), R, V, beams, scores.data_ptr(),
                       done.data_ptr(), max(eos, -1), out.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                       ended.data_ptr(), ws.data_ptr(), need, _lib.raw_stream(dev.index)))
    return out, parents, tokens, ended
