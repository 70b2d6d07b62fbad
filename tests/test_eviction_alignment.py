"""Pointers off their elements' alignment are refused on the host, before a
kernel reads through them.  CPU only: every call fails validation."""

from __future__ import annotations

import ctypes

import pytest

from specdecode_b200 import _lib

PTR = 4096  # never dereferenced


@pytest.fixture(scope="module")
def library():
    return _lib.load_library()


def pool():
    return _lib.PagePool(PTR, PTR, PTR, PTR, 8, 16, 2, 2, 64, 4096, 2048, 1024, 64, 32, 16)


def select(h, mass=PTR, tables=PTR, lens=PTR, kept=PTR, status=PTR):
    return h.sdc_select_tokens(ctypes.byref(pool()), mass, 1, tables, 8, lens, 100, 10, 2, 1, kept, status, 0)


def compact(h, mass=PTR, tables=PTR, lens=PTR, kept=PTR, status=PTR):
    return h.sdc_compact_tokens(ctypes.byref(pool()), mass, 1, tables, 8, lens, kept, 10, status, 0)


def clear(h, mass=PTR, slots=PTR, status=PTR):
    return h.sdc_clear_mass(ctypes.byref(pool()), mass, slots, 1, status, 0)


def observe(h, mass=PTR, query=PTR, tables=PTR, lens=PTR, workspace=PTR, status=PTR):
    return h.sdc_observe_attention(ctypes.byref(pool()), 0, mass, query, _lib.DTYPE_BF16, 1, 4, 2, tables, 8, lens, 5000,
                                   workspace, 1 << 24, status, 0)


def rotate(h, positions=PTR, slots=PTR, out=PTR, status=PTR):
    batch = _lib.RotateBatch(PTR, PTR, PTR, _lib.DTYPE_BF16, 2, 3, 4, *[1536, 512, 64] * 3, positions, 3, PTR, 100, 64, 0,
                             None, None, _lib.DTYPE_BF16, 1e-6)
    return h.sdc_norm_rotate_append(ctypes.byref(pool()), 0, ctypes.byref(batch), slots, out, status, 0)


@pytest.mark.parametrize("call, argument, off", [
    *[(call, name, off) for call in (select, compact) for name in ("mass", "tables", "lens", "kept", "status")
      for off in (1, 2)],
    *[(clear, name, 2) for name in ("mass", "status")], (clear, "slots", 4),
    *[(observe, name, 2) for name in ("mass", "tables", "lens", "status")], (observe, "query", 8),
    (observe, "workspace", 8),
    (rotate, "positions", 4), (rotate, "slots", 4), (rotate, "status", 2), (rotate, "out", 8),
])
def test_misaligned_pointers_are_refused(library, call, argument, off):
    assert call(library.handle, **{argument: PTR + off}) == _lib.STATUS_MISALIGNED
