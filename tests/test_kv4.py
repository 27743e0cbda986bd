"""Argument checks of the paged cache and the beam selection that need no GPU, and the plain forms they are tested with."""
import ctypes

import numpy as np
import pytest
import torch

from rngd_pd import _lib, beam, kv4
from tests import kv4_ref as ref


def test_tensors_off_the_gpu_are_refused():
    pool = torch.zeros(2, 4, 2, 4, 20 * 64, dtype=torch.uint8)
    t, z = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    k = torch.zeros(2, 2, 1, 2, 64)
    for f in (lambda: kv4.store(pool, t, z, k, k), lambda: kv4.load(pool, t, z, 1),
              lambda: kv4.attention(torch.zeros(2, 1, 4, 64), pool[0], t, z),
              lambda: kv4.fork(pool, torch.zeros(4, dtype=torch.int32), t, z),
              lambda: kv4.compact(pool, torch.zeros(4, dtype=torch.int32), t),
              lambda: beam.select(torch.zeros(2, 10), torch.zeros(2), torch.zeros(2, dtype=torch.bool), 2)):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(ValueError):
        kv4.alloc_pool(1, 1, 1, 80, device="cpu")
    assert kv4.alloc_pool(2, 3, 4, 64, device="cpu").shape == (2, 3, 4, 4, 1280) and kv4.page_bytes(8, 128) == 81920
    r, t, n = kv4.empty_state(3, 2, 5, device="cpu")
    assert r.tolist() == [0] * 5 and t.tolist() == [[-1, -1]] * 3 and n.tolist() == [0] * 3


def test_c_entries_refuse_bad_arguments():
    """Refused on the host, with a message, before anything is launched."""
    lib, p = _lib.lib, ctypes.c_void_p(4096)
    i3, i4 = (ctypes.c_int64 * 3)(1, 1, 1), (ctypes.c_int64 * 4)(1, 1, 1, 1)
    bad = [
        (lib.rngd_kv4_store(None, 0, 1, 1, 64, 1, p, 1, p, None, 1, 1, p, i4, p, i4, 0, None), b"aligned"),
        (lib.rngd_kv4_store(p, 0, 1, 1, 96, 1, p, 1, p, None, 1, 1, p, i4, p, i4, 0, None), b"96"),
        (lib.rngd_kv4_store(p, 0, 1, 1, 64, 1, p, 1, p, None, 1, 1, p, i4, p, i4, 7, None), b"data type"),
        (lib.rngd_kv4_store(p, 0, 1, 1, 64, 1, p, 1, None, None, 1, 1, p, i4, p, i4, 0, None), b"null"),
        (lib.rngd_kv4_load(p, 8, 1, 1, 64, 1, p, 1, p, None, 1, 1, p, p, 0, None), b"aligned"),
        (lib.rngd_kv4_attn(p, i3, p, i3, 0, p, 1, 3, 64, p, 1, p, 1, 1, 4, 0, 0, 1.0, p, 1 << 30, None), b"multiple"),
        (lib.rngd_kv4_attn(p, i3, p, i3, 0, p, 1, 2, 64, p, 1, p, 1, 1, 4, -1, 0, 1.0, p, 1 << 30, None), b"window"),
        (lib.rngd_kv4_fork(p, 0, 1, 1, 1, 64, p, p, 1, p, 2000, None, 0, p, p, p, p, p, 1 << 30, None), b"rows"),
        (lib.rngd_kv4_fork(p, 0, 1, 1, 1, 64, p, p, 1, p, 1, None, 0, p, p, p, p, p, 1 << 30, None), b"in place"),
        (lib.rngd_kv4_compact(p, 0, 1, 0, 1, 64, p, p, 1, 1, p, p, p, p, 1 << 30, None), b"P=0"),
        (lib.rngd_beam_select(p, 0, 10, 4, 10, 33, p, p, 0, p, p, p, p, p, 1 << 30, None), b"33 beams"),
        (lib.rngd_beam_select(p, 9, 10, 4, 10, 2, p, p, 0, p, p, p, p, p, 1 << 30, None), b"data type"),
    ]
    for st, _ in bad:
        assert st == _lib.RNGD_ERR_ARG
    # the message of the last refusal is there, and each call's own is
    assert b"data type" in _lib.last_error().encode()
    lib.rngd_kv4_fork(p, 0, 1, 1, 1, 64, p, p, 1, p, 2000, None, 0, p, p, p, p, p, 1 << 30, None)
    assert "2000 rows" in _lib.last_error()


def test_struct_matches_the_header():
    assert ctypes.sizeof(_lib.Kv4) == 64


def test_plain_forms_on_small_cases():
    """What the GPU tests compare with, on cases that can be checked by eye."""
    x = np.linspace(0, 15, 32)
    u, s, c, _ = ref.encode(x)
    assert s[0] == 1.0 and c[0] == -16.0 and np.array_equal(ref.values(u, s, c), np.rint(x))
    assert ref.visible(5, 0, 0).tolist() == [0, 1, 2, 3, 4, 5] and ref.visible(5, 2, 1).tolist() == [0, 4, 5]
    assert ref.visible(-1, 0, 0).tolist() == []
    # two rows go on as row 0, whose last page holds 10 positions: the second gets a copy on the lowest free page
    got = ref.fork([1, 0, 1, 0], [[2, -1], [0, -1]], [10, 64], [0, 0], 0)
    assert got == ([1, 0, 1, 0], [[2, -1], [0, -1]], [10, 10], 0, [(2, 0, 1)])
    best, parent, token, done, _ = ref.select(np.log(np.array([[.5, .3, .2], [.1, .1, .8]])), np.array([0.0, -1.0]),
                                              np.array([False, False]), 2, 2)
    assert parent.tolist() == [[0, 0]] and token.tolist() == [[0, 1]] and not done.any()


def test_tables_wider_than_positions_are_refused():
    """Positions are 32-bit numbers: 2^25 pages of 64 are one too many."""
    lib, p, i3 = _lib.lib, ctypes.c_void_p(4096), (ctypes.c_int64 * 3)(1, 1, 1)
    need = ctypes.c_size_t(0)
    for ld in (2 ** 25, 2 ** 31 - 1):
        for window in (0, 100):
            assert lib.rngd_kv4_attn_workspace(0, 1, 1, 4, 2, 64, ld, window, 0, ctypes.byref(need)) == _lib.RNGD_ERR_ARG
            assert f"table of {ld} pages" in _lib.last_error()
        assert lib.rngd_kv4_attn(p, i3, p, i3, 0, p, 1, 2, 64, p, ld, p, 1, 1, 4, 0, 0, 1.0, p, 1 << 40, None) == _lib.RNGD_ERR_ARG
        assert f"table of {ld} pages" in _lib.last_error()


def test_missing_workspaces_and_those_off_their_alignment_are_refused():
    lib, p, odd, r = _lib.lib, ctypes.c_void_p(4096), ctypes.c_void_p(4097), ctypes.c_void_p(8192)
    for name, st in (("kv4_fork", lib.rngd_kv4_fork(p, 0, 1, 1, 1, 64, p, p, 1, p, 1, None, 0, r, r, r, r, odd, 1 << 20, None)),
                     ("kv4_compact", lib.rngd_kv4_compact(p, 0, 1, 1, 1, 64, p, p, 1, 1, r, r, r, odd, 1 << 20, None))):
        assert st == _lib.RNGD_ERR_ARG, name
    # none at all, with no rows to fork: the count of copies is written all the same
    assert lib.rngd_kv4_fork(p, 0, 1, 1, 1, 64, p, None, 0, None, 0, None, 0, r, None, None, r, None, 16, None) == _lib.RNGD_ERR_ARG
    for f in (lambda: lib.rngd_kv4_fork(p, 0, 1, 1, 1, 64, p, p, 1, p, 1, None, 0, r, r, r, r, odd, 1 << 20, None),
              lambda: lib.rngd_kv4_compact(p, 0, 1, 1, 1, 64, p, p, 1, 1, r, r, r, odd, 1 << 20, None)):
        f()
        assert "aligned" in _lib.last_error()
