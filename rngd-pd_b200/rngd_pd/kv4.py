"""Paged KV cache held in 4 bits: store, load, attention, and the pages of its sequences.

The reference keeps its cache in bf16 lanes of a fixed width (src/rngd_pd/engines/decode_batch.py:300-420).
Here positions live in pages of 64, at 5 bits a value (4-bit codes, and two fp16 numbers per 32 values along
the head dimension), so sequences of unequal length share one pool and the beams of a search share the pages
they have in common.

  pool   uint8 [L, P, NKV, 4, 20 * HD] (alloc_pool); the attention takes one layer's, pool[l]
  table  int32 [R, width]: page ids of each sequence, position p in entry p // 64; -1 = no page
  lens   int32 [R]: positions held
  ref    int32 [P]: holders of each page, 0 = free

Everything lives on the pool's GPU; calls are queued on the current stream and wait for nothing, so they can
be captured into a CUDA graph.  As with torch's own operators, a tensor made on another stream has to be
ordered before the call by the caller (and kept alive with record_stream).  Nothing falls back to the CPU.
"""
import torch

from rngd_pd import _lib

PAGE = 64     # positions of a page
HEAD_DIMS = (64, 128)

_DT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_INT_MAX = 2 ** 31 - 1
_check = _lib.check
_store, _load, _attn = _lib.lib.rngd_kv4_store, _lib.lib.rngd_kv4_load, _lib.lib.rngd_kv4_attn
_fork, _compact = _lib.lib.rngd_kv4_fork, _lib.lib.rngd_kv4_compact


def page_bytes(n_kv, head_dim):
    """Bytes of one layer's page."""
    return n_kv * 4 * 20 * head_dim


def alloc_pool(layers, pages, n_kv, head_dim, device="cuda"):
    """A pool of free pages: uint8 [layers, pages, n_kv, 4, 20 * head_dim]."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim={head_dim}: the kernels take {HEAD_DIMS}")
    return torch.zeros((layers, pages, n_kv, 4, 20 * head_dim), dtype=torch.uint8, device=device)


def empty_state(rows, width, pages, device="cuda"):
    """(ref, table, lens) of `rows` sequences that hold nothing, tables `width` pages wide."""
    i32 = dict(dtype=torch.int32, device=device)
    return (torch.zeros(pages, **i32), torch.full((rows, width), -1, **i32), torch.zeros(rows, **i32))


def _elsewhere(dev):
    """Whether another GPU than the tensors' is current (the calls below then start over with theirs)."""
    return dev.index != torch.cuda.current_device()


def _pool_dims(pool, layers):
    """(L, P, NKV, HD, bytes between layers) of a pool, or of one layer's where `layers` is false."""
    shape = pool.shape
    if len(shape) != (5 if layers else 4) or pool.dtype is not torch.uint8 or not pool.is_cuda:
        raise ValueError(f"pool must be a {5 if layers else 4}-dimensional uint8 CUDA tensor, got {tuple(shape)} "
                         f"{pool.dtype} on {pool.device}")
    P, NKV, four, blk = shape[-4:]
    HD = blk // 20
    if four != 4 or blk % 20 or HD not in HEAD_DIMS:
        raise ValueError(f"pool {tuple(shape)}: the last dimensions must be [pages, kv heads, 4, 20 * head_dim]")
    if not pool.is_contiguous() and pool.stride()[-4:] != (NKV * 4 * blk, 4 * blk, blk, 1):
        raise ValueError("pool: a layer's pages must be contiguous")
    if layers and shape[0] > 1 and pool.stride(0) < P * NKV * 4 * blk:
        raise ValueError(f"pool: layers {pool.stride(0)} bytes apart lie on one another")
    return (shape[0], P, NKV, HD, pool.stride(0)) if layers else (1, P, NKV, HD, 0)


def _i32(name, t, shape, dev):
    if t.dtype is not torch.int32 or t.shape != shape or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 {tuple(shape)} tensor on {dev}, got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}")
    return t.data_ptr()


def _rows(name, t, dims):
    """A tensor of rows whose last dimension is contiguous -> (pointer, strides)."""
    st = t.stride()
    if len(st) != dims or (st[-1] != 1 and t.shape[-1] > 1):
        raise ValueError(f"{name} must have {dims} dimensions, the last one contiguous, got {tuple(t.shape)} "
                         f"strides {st}")
    return t.data_ptr(), _lib.i64_array(st)


def store(pool, table, start, k, v, count=None):
    """Quantise rows into pages: row t of sequence b goes to position start[b] + t, for t < count[b] (None: all).

    k, v: [L, B, T, NKV, HD] (any strides, the last dimension contiguous), or [B, T, NKV, HD] with one layer's
    pool; bfloat16, float16 or float32.  Magnitudes are held to 16384, a group of 32 with a NaN reads back as
    NaN.  Positions without a page are dropped.  No two rows of a call may fall on one position."""
    L, P, NKV, HD, layer = _pool_dims(pool, k.dim() == 5)
    if k.dim() == 4:
        k, v = k.unsqueeze(0), v.unsqueeze(0)
    dev = pool.device
    shape = k.shape
    if len(shape) != 5 or v.shape != shape or shape[0] != L or shape[3] != NKV or shape[4] != HD:
        raise ValueError(f"k and v must be [{L}, streams, tokens, {NKV}, {HD}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype not in _DT or v.dtype is not k.dtype or k.device != dev or v.device != dev:
        raise ValueError(f"k and v must be bfloat16, float16 or float32 on {dev}, got {k.dtype} and {v.dtype}")
    B, T = shape[1], shape[2]
    kp, ks = _rows("k", k, 5)
    vp, vs = _rows("v", v, 5)
    width = table.shape[-1]
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return store(pool if pool.dim() == 5 else pool.unsqueeze(0), table, start, k, v, count)
    _check(_store(pool.data_ptr(), layer, P, NKV, HD, L, _i32("table", table, (B, width), dev), width,
                  _i32("start", start, (B,), dev), None if count is None else _i32("count", count, (B,), dev), B, T,
                  kp, ks, vp, vs, _DT[k.dtype], _lib.raw_stream(dev.index)))


def load(pool, table, start, tokens, count=None, dtype=torch.float16):
    """The values that positions start[b] .. start[b] + tokens - 1 stand for: (k, v) [L, B, tokens, NKV, HD]
    (without L for one layer's pool).  Zeros for t >= count[b] and where there is no page.  float16 and
    float32 are exact, bfloat16 is rounded once."""
    layers = pool.dim() == 5
    L, P, NKV, HD, layer = _pool_dims(pool, layers)
    dev = pool.device
    if dtype not in _DT:
        raise ValueError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    B, width = table.shape
    if tokens < 0:
        raise ValueError(f"tokens={tokens}")
    shape = (L, B, tokens, NKV, HD) if layers else (B, tokens, NKV, HD)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return load(pool, table, start, tokens, count, dtype)
    k = torch.empty(shape, dtype=dtype, device=dev)
    v = torch.empty_like(k)
    _check(_load(pool.data_ptr(), layer, P, NKV, HD, L, _i32("table", table, (B, width), dev), width,
                 _i32("start", start, (B,), dev), None if count is None else _i32("count", count, (B,), dev), B,
                 tokens, k.data_ptr(), v.data_ptr(), _DT[dtype], _lib.raw_stream(dev.index)))
    return k, v


def attention(q, pool, table, lens, window=0, sinks=0, scale=None, out=None):
    """Attention of the last T tokens of each sequence over its pages of one layer.

    q: [B, T, NH, HD] bfloat16, float16 or float32 (any strides, the last dimension contiguous), NH a multiple of
    the pool's kv heads; pool: one layer's.  Token t of sequence b stands at i = lens[b] - T + t (its own key and
    value are stored already) and sees positions j <= i with j > i - window (0: no window) or j < sinks; what it
    does not see, and what lies where there is no page, has no part in the result, NaN included.  A token that sees
    nothing gives zeros; one that sees a NaN gives NaN, at least in the dimensions concerned.  scale: 1 / sqrt(HD) by default.  Returns [B, T, NH, HD] of q's type, in `out` where given."""
    _, P, NKV, HD, _ = _pool_dims(pool, False)
    dev, dt = pool.device, q.dtype
    qp, qs = _rows("q", q, 4)
    B, T, NH, D = q.shape
    if D != HD or NH % NKV or NH == 0:
        raise ValueError(f"q {tuple(q.shape)} does not fit a pool of {NKV} kv heads of {HD}")
    if dt not in _DT or q.device != dev:
        raise ValueError(f"q must be bfloat16, float16 or float32 on {dev}, got {dt} on {q.device}")
    if window < 0 or sinks < 0:
        raise ValueError(f"window={window} and sinks={sinks} must not be negative")
    width = table.shape[-1]
    window, sinks = min(window, _INT_MAX), min(sinks, _INT_MAX)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return attention(q, pool, table, lens, window, sinks, scale, out)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype is not dt or out.device != dev:
        raise ValueError(f"out must be {tuple(q.shape)} {dt} on {dev}, got {tuple(out.shape)} {out.dtype}")
    elif any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise ValueError(f"out {tuple(out.shape)} strides {out.stride()}: rows lie on one another")
    op, os = _rows("out", out, 4)
    need = _lib.workspace_bytes("rngd_kv4_attn_workspace", _DT[dt], B, T, NH, NKV, HD, width, window,
                                 sinks)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None  # held until the launches are queued
    _check(_attn(qp, qs, op, os, _DT[dt], pool.data_ptr(), P, NKV, HD, _i32("table", table, (B, width), dev), width,
                 _i32("lens", lens, (B,), dev), B, T, NH, window, sinks,
                 HD ** -0.5 if scale is None else scale, None if ws is None else ws.data_ptr(), need,
                 _lib.raw_stream(dev.index)))
    return out


def fork(pool, ref, table, lens, parents=None, room=0):
    """The state after row r went on as row parents[r] (None: every row as itself; negative: the row ends and lets
    go of its pages), with pages for `room` more positions in every row: (ref, table, lens, short).

    Full pages are shared.  A partly filled last page belongs to one row alone afterwards: the lowest row keeps it
    if only such rows hold it, the others get copies of its filled blocks, in all layers.  Free pages are given
    lowest first, in the order of rows; short (int32 [1]) counts those that could not be given (-1 in the table), up
    to 2^31 - 1.
    The old state's tensors are left as they are.  The pool changes only in pages that were free or that this call
    lets go of: pages that the new state holds too keep their content, the others may be handed out at once."""
    L, P, NKV, HD, layer = _pool_dims(pool, True)
    dev = pool.device
    R, width = table.shape
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return fork(pool, ref, table, lens, parents, room)
    rp, tp, lp = _i32("ref", ref, (P,), dev), _i32("table", table, (R, width), dev), _i32("lens", lens, (R,), dev)
    room = max(-1, min(room, _INT_MAX))  # the library refuses both ends; more would be cut to 32 bits on the way
    new_ref, new_table, new_lens = torch.empty_like(ref), torch.empty_like(table), torch.empty_like(lens)
    short = torch.empty(1, dtype=torch.int32, device=dev)
    need = _lib.workspace_bytes("rngd_kv4_fork_workspace", R, width)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _check(_fork(pool.data_ptr(), layer, L, P, NKV, HD, rp, tp, width, lp, R,
                 None if parents is None else _i32("parents", parents, (R,), dev), room, new_ref.data_ptr(),
                 new_table.data_ptr(), new_lens.data_ptr(), short.data_ptr(), ws.data_ptr(), need,
                 _lib.raw_stream(dev.index)))
    return new_ref, new_table, new_lens, short


def compact(pool, ref, table):
    """The state with the n held pages in places 0 .. n-1 of the pool: (ref, table, live), live (int32 [1]) being n.

    The k-th held page from place n on moves into the k-th free place below n, in all layers; the rest stay.  Page
    ids change: `table` has to hold the rows of every sequence that goes on using the pool.  The old state's
    tensors are left as they are, but its free places below n now hold pages."""
    L, P, NKV, HD, layer = _pool_dims(pool, True)
    dev = pool.device
    R, width = table.shape
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return compact(pool, ref, table)
    rp, tp = _i32("ref", ref, (P,), dev), _i32("table", table, (R, width), dev)
    new_ref, new_table = torch.empty_like(ref), torch.empty_like(table)
    live = torch.empty(1, dtype=torch.int32, device=dev)
    need = _lib.workspace_bytes("rngd_kv4_compact_workspace", P)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _check(_compact(pool.data_ptr(), layer, L, P, NKV, HD, rp, tp, width, R, new_ref.data_ptr(),
                    new_table.data_ptr(), live.data_ptr(), ws.data_ptr(), need, _lib.raw_stream(dev.index)))
    return new_ref, new_table, live
