"""Rotated append and eviction on the host: the library refuses bad arguments
before any device work, the rotary table has the angles of far positions, and
the oracle's pieces agree with each other.  CPU only."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from oracle.eviction import attention_mass_fp64, norm_rotate_fp64, select_kept
from specdecode_b200 import _lib
from specdecode_b200.eviction import _budget
from specdecode_b200.rotary import RotaryTable

PTR = 4096  # a pointer that is never dereferenced: every call fails validation first


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


def pool(head_dim=64, layers=2, heads=2):
    page = 16 * head_dim
    return _lib.PagePool(PTR, PTR, PTR, PTR, 8, 16, layers, heads, head_dim, layers * heads * page, heads * page, page,
                         layers * heads * 16, heads * 16, 16)


def rotate_batch(**changes):
    fields = dict(query=PTR, key=PTR, value=PTR, dtype=_lib.DTYPE_BF16, batch=2, tokens=3, query_heads=4,
                  query_batch_stride=1536, query_token_stride=512, query_head_stride=64, key_batch_stride=1536,
                  key_token_stride=512, key_head_stride=64, value_batch_stride=1536, value_token_stride=512,
                  value_head_stride=64, positions=PTR, position_stride=3, table=PTR, table_positions=100,
                  rotary_dim=64, interleaved=0, query_weight=None, key_weight=None, weight_dtype=_lib.DTYPE_BF16,
                  eps=1e-6)
    fields.update(changes)
    batch = _lib.RotateBatch()
    for name, value in fields.items():
        setattr(batch, name, value)
    return batch


@pytest.mark.parametrize("changes, expected", [
    (dict(query=None), _lib.STATUS_NULL_ARGUMENT),
    (dict(value=None), _lib.STATUS_NULL_ARGUMENT),
    (dict(positions=None), _lib.STATUS_NULL_ARGUMENT),
    (dict(table=None), _lib.STATUS_NULL_ARGUMENT),
    (dict(dtype=_lib.DTYPE_F64), _lib.STATUS_UNSUPPORTED),
    (dict(batch=-1), _lib.STATUS_INVALID_SIZE),
    (dict(query_heads=0), _lib.STATUS_INVALID_SIZE),
    (dict(table_positions=0), _lib.STATUS_INVALID_SIZE),
    (dict(position_stride=2), _lib.STATUS_INVALID_SIZE),
    (dict(key_token_stride=-512), _lib.STATUS_INVALID_SIZE),
    (dict(key=PTR + 8), _lib.STATUS_MISALIGNED),
    (dict(table=PTR + 4), _lib.STATUS_MISALIGNED),
    (dict(query_head_stride=60), _lib.STATUS_MISALIGNED),
    (dict(rotary_dim=63), _lib.STATUS_INVALID_ARGUMENT),
    (dict(rotary_dim=66), _lib.STATUS_INVALID_ARGUMENT),
    (dict(rotary_dim=0), _lib.STATUS_INVALID_ARGUMENT),
    (dict(query_weight=PTR, weight_dtype=_lib.DTYPE_F64), _lib.STATUS_UNSUPPORTED),
    (dict(key_weight=PTR + 2), _lib.STATUS_MISALIGNED),
    (dict(key_weight=PTR, eps=0.0), _lib.STATUS_INVALID_ARGUMENT),
    (dict(key_weight=PTR, eps=float("nan")), _lib.STATUS_INVALID_ARGUMENT),
    (dict(batch=1 << 20, tokens=1 << 20, position_stride=1 << 20), _lib.STATUS_OVERFLOW),
])
def test_rotated_append_validates_on_the_host(lib, changes, expected):
    call = lib.handle.sdc_norm_rotate_append
    assert call(ctypes.byref(pool()), 0, ctypes.byref(rotate_batch(**changes)), PTR, PTR, PTR, 0) == expected


def test_rotated_append_validates_its_other_arguments(lib):
    call, p, b = lib.handle.sdc_norm_rotate_append, pool(), rotate_batch()
    assert call(None, 0, ctypes.byref(b), PTR, PTR, PTR, 0) == _lib.STATUS_NULL_ARGUMENT
    assert call(ctypes.byref(p), 0, None, PTR, PTR, PTR, 0) == _lib.STATUS_NULL_ARGUMENT
    assert call(ctypes.byref(p), 0, ctypes.byref(b), None, PTR, PTR, 0) == _lib.STATUS_NULL_ARGUMENT
    assert call(ctypes.byref(p), 0, ctypes.byref(b), PTR, None, PTR, 0) == _lib.STATUS_NULL_ARGUMENT
    assert call(ctypes.byref(p), 0, ctypes.byref(b), PTR, PTR, None, 0) == _lib.STATUS_NULL_ARGUMENT
    assert call(ctypes.byref(p), 2, ctypes.byref(b), PTR, PTR, PTR, 0) == _lib.STATUS_INVALID_SIZE
    assert call(ctypes.byref(p), 0, ctypes.byref(b), PTR, PTR + 8, PTR, 0) == _lib.STATUS_MISALIGNED
    # nothing to do
    empty = rotate_batch(batch=0)
    assert call(ctypes.byref(p), 0, ctypes.byref(empty), PTR, PTR, PTR, 0) == _lib.STATUS_OK


def test_observe_validates_on_the_host(lib):
    h = lib.handle

    def call(p=None, layer=0, mass=PTR, query=PTR, dtype=_lib.DTYPE_BF16, batch=1, heads=4, window=2, tables=PTR,
             stride=8, lens=PTR, max_len=5000, workspace=PTR, size=1 << 24, status=PTR):
        p = p or pool()
        return h.sdc_observe_attention(ctypes.byref(p), layer, mass, query, dtype, batch, heads, window, tables, stride,
                                       lens, max_len, workspace, size, status, 0)

    for name in ("mass", "query", "tables", "lens", "workspace", "status"):
        assert call(**{name: None}) == _lib.STATUS_NULL_ARGUMENT, name
    assert call(layer=2) == _lib.STATUS_INVALID_SIZE
    assert call(batch=0) == _lib.STATUS_INVALID_SIZE
    assert call(window=0) == _lib.STATUS_INVALID_SIZE
    assert call(window=5001) == _lib.STATUS_INVALID_SIZE
    assert call(heads=5) == _lib.STATUS_INVALID_ARGUMENT
    assert call(heads=4, window=33) == _lib.STATUS_UNSUPPORTED  # 2 x 33 rows
    assert call(heads=130, window=1) == _lib.STATUS_UNSUPPORTED
    assert call(dtype=_lib.DTYPE_F64) == _lib.STATUS_UNSUPPORTED
    assert call(p=pool(head_dim=48)) == _lib.STATUS_UNSUPPORTED
    assert call(query=PTR + 1) == _lib.STATUS_MISALIGNED
    assert call(mass=PTR + 2) == _lib.STATUS_MISALIGNED
    assert call(max_len=1 << 31) == _lib.STATUS_OVERFLOW
    assert call(batch=1 << 30) == _lib.STATUS_OVERFLOW
    assert call(workspace=PTR + 4) == _lib.STATUS_MISALIGNED
    least, most = ctypes.c_size_t(), ctypes.c_size_t()
    size = h.sdc_observe_workspace_size
    assert size(3, 4, 2, 64, 2, 5000, ctypes.byref(least), ctypes.byref(most)) == _lib.STATUS_OK
    assert 0 < least.value and most.value == 6 * least.value  # one (sequence, KV head), all of them
    assert call(batch=3, size=least.value - 1) == _lib.STATUS_INVALID_SIZE
    # a context whose scores one block keeps needs none
    small, most_small = ctypes.c_size_t(7), ctypes.c_size_t(7)
    assert size(3, 4, 2, 64, 2, 100, ctypes.byref(small), ctypes.byref(most_small)) == _lib.STATUS_OK
    assert (small.value, most_small.value) == (0, 0)
    assert size(3, 4, 2, 64, 2, 5000, None, ctypes.byref(most)) == _lib.STATUS_NULL_ARGUMENT
    assert size(0, 4, 2, 64, 2, 5000, ctypes.byref(least), ctypes.byref(most)) == _lib.STATUS_INVALID_SIZE
    assert size(1, 5, 2, 64, 2, 5000, ctypes.byref(least), ctypes.byref(most)) == _lib.STATUS_INVALID_ARGUMENT
    assert size(1, 130, 2, 64, 1, 5000, ctypes.byref(least), ctypes.byref(most)) == _lib.STATUS_UNSUPPORTED


def test_select_and_compact_validate_on_the_host(lib):
    h = lib.handle

    def select(mass=PTR, batch=1, tables=PTR, stride=8, lens=PTR, max_len=100, budget=10, recent=2, sinks=1, kept=PTR,
               status=PTR):
        p = pool()
        return h.sdc_select_tokens(ctypes.byref(p), mass, batch, tables, stride, lens, max_len, budget, recent, sinks,
                                   kept, status, 0)

    for name in ("mass", "tables", "lens", "kept", "status"):
        assert select(**{name: None}) == _lib.STATUS_NULL_ARGUMENT, name
    assert select(batch=0) == _lib.STATUS_INVALID_SIZE
    assert select(budget=0) == _lib.STATUS_INVALID_SIZE
    assert select(recent=-1) == _lib.STATUS_INVALID_ARGUMENT
    assert select(recent=6, sinks=5) == _lib.STATUS_INVALID_ARGUMENT
    assert select(max_len=1 << 31) == _lib.STATUS_OVERFLOW
    assert select(batch=1 << 30) == _lib.STATUS_OVERFLOW

    def compact(mass=PTR, batch=1, tables=PTR, stride=8, lens=PTR, kept=PTR, budget=10, status=PTR):
        p = pool()
        return h.sdc_compact_tokens(ctypes.byref(p), mass, batch, tables, stride, lens, kept, budget, status, 0)

    for name in ("tables", "lens", "kept", "status"):
        assert compact(**{name: None}) == _lib.STATUS_NULL_ARGUMENT, name
    assert compact(batch=0) == _lib.STATUS_INVALID_SIZE
    assert compact(budget=0) == _lib.STATUS_INVALID_SIZE
    assert compact(budget=1 << 31) == _lib.STATUS_OVERFLOW

    def clear(mass=PTR, slots=PTR, count=1, status=PTR):
        p = pool()
        return h.sdc_clear_mass(ctypes.byref(p), mass, slots, count, status, 0)

    assert clear(mass=None) == _lib.STATUS_NULL_ARGUMENT
    assert clear(status=None) == _lib.STATUS_NULL_ARGUMENT
    assert clear(slots=None) == _lib.STATUS_NULL_ARGUMENT
    assert clear(count=-1) == _lib.STATUS_INVALID_SIZE
    assert clear(count=1 << 40) == _lib.STATUS_OVERFLOW
    assert clear(slots=None, count=0) == _lib.STATUS_OK


def test_budget_arguments():
    assert _budget(8, 3, 5) == (8, 3, 5)
    for bad in ((0, 0, 0), (8, 5, 4), (8, -1, 0), (8.0, 0, 0), (True, 0, 0), (8, 0, -2)):
        with pytest.raises(ValueError):
            _budget(*bad)


@pytest.mark.parametrize("rotary_dim, base, scaling", [(64, 10000.0, 1.0), (128, 500000.0, 1.0), (20, 10000.0, 1.25)])
def test_rotary_table_has_the_angles_of_far_positions(rotary_dim, base, scaling):
    positions = 131072
    table = RotaryTable(rotary_dim, positions, base=base, scaling=scaling, device="cpu")
    assert tuple(table.values.shape) == (positions, rotary_dim // 2, 2)
    rows = np.array([0, 1, 7, 4095, 65537, 131071])
    freq = np.longdouble(base) ** (-np.arange(0, rotary_dim, 2).astype(np.longdouble) / rotary_dim)
    angles = rows[:, None].astype(np.longdouble) * freq
    got = table.values[rows].numpy().astype(np.float64)
    # the float64 angle is off by at most 131072 * 3 * 2^-53, the entry rounds
    # once to float32 and once for the scaling product
    tolerance = 131072 * 3 * 2.0 ** -53 + 2 * 2.0 ** -24 * scaling
    assert np.abs(got[..., 0] - np.cos(angles) * scaling).max() <= tolerance
    assert np.abs(got[..., 1] - np.sin(angles) * scaling).max() <= tolerance


def test_rotary_table_refusals():
    for bad in (dict(rotary_dim=0, max_positions=4), dict(rotary_dim=7, max_positions=4),
                dict(rotary_dim=8, max_positions=0), dict(rotary_dim=8, max_positions=4, inv_freq=[1.0] * 3)):
        with pytest.raises(ValueError):
            RotaryTable(**bad, device="cpu")


def test_oracle_rotation_keeps_norms_and_relative_positions():
    rng = np.random.default_rng(1)
    freq = 10000.0 ** (-np.arange(8) / 8)
    x, y = rng.standard_normal((2, 1, 1, 16))
    for interleaved in (False, True):
        a, _ = norm_rotate_fp64(x, [50], freq, interleaved=interleaved)
        assert abs(np.linalg.norm(a) - np.linalg.norm(x)) < 1e-12
        dots = [float((norm_rotate_fp64(x, [p + 9], freq, interleaved=interleaved)[0] *
                       norm_rotate_fp64(y, [p], freq, interleaved=interleaved)[0]).sum()) for p in (0, 13, 400)]
        assert max(dots) - min(dots) < 1e-11


def test_oracle_mass_and_selection():
    rng = np.random.default_rng(2)
    mass = attention_mass_fp64(rng.standard_normal((4, 3, 8)), rng.standard_normal((11, 2, 8)))
    assert np.allclose(mass.sum(axis=1), 2 * 3)  # one unit per query row
    assert np.array_equal(select_kept(np.array([5, 1, 1, 9, 1, 2, 0], np.float32), 4, 1, 1), [0, 3, 5, 6])
    assert np.array_equal(select_kept(np.array([0, 1, 1, 1, np.nan, 0], np.float32), 3, 0, 0), [1, 2, 4])
    assert np.array_equal(select_kept(np.array([0, 1], np.float32), 4, 1, 1), [0, 1, -1, -1])
