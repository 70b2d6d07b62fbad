"""norm_rotate_append against float64: queries, keys and values of every type,
pairing, rotary width and head size; its refusals and faults.

Tolerances.  u = 2^-24.  With y the exact normalised head and |y_i| + |y_j| the
magnitudes a rotated element is formed from (``span``), the float32 path errs by
at most: the sum of squares, sixteen terms in a lane then up to five shuffle
steps, 21 u, halved by the root; the mean and eps, u each, halved; rsqrtf, 2
ulp = 4 u; the two products with it, 2 u; the table entry, u (plus the float64
angle's own error, below u / 8); the rotation, two products and a sum, 3 u:
11 + 1 + 4 + 2 + 1 + 1 + 3 = 23, taken as 24 u span.  A query then rounds once
to its type, finfo.eps / 2 relative.  A key's scale is max / 127 of such
elements, off by the largest error / 127 plus two roundings, and a code is the
nearest integer: the value it stands for is within half a scale of the element,
plus the element's error, plus 127 times the scale's."""

from __future__ import annotations

import numpy as np
import pytest

from gpu_helpers import make_cache
from oracle.eviction import norm_rotate_fp64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def projections(device, B, n, Hq, H, D, dtype, seed, spread=0.5):
    import torch

    g = torch.Generator(device=device).manual_seed(seed)
    packed = torch.randn((B, n, Hq + 2 * H, D), generator=g, device=device)
    packed *= torch.exp(torch.randn(D, generator=g, device=device) * spread)
    packed = packed.to(dtype)
    return packed[:, :, :Hq], packed[:, :, Hq:Hq + H], packed[:, :, Hq + H:]


def stored(cache, slots, layer):
    """float64 values and float32 scales of the slots: keys, values [n, H, D]."""
    bs = cache.config.block_size
    block, off = slots // bs, slots % bs
    out = []
    for codes, scales in ((cache.key_codes, cache.key_scale_pages), (cache.value_codes, cache.value_scale_pages)):
        s = scales[block, layer, :, off]
        out += [(codes[block, layer, :, off].double() * s.double()[..., None]).cpu().numpy(),
                s.double().cpu().numpy()]
    return out


def f64(t):
    return t.detach().double().cpu().numpy()


def check(device, B, n, Hq, H, D, dtype, rotary_dim, interleaved, norm, weight_dtype, block_size, seed=0, far=60000):
    import torch

    from specdecode_b200.rotary import RotaryTable, norm_rotate_append

    cache = make_cache(device, 2, H, D, block_size, B * (-(-n // block_size) + 1), max_sequences=B)
    for s in range(B):
        cache.create_sequence(s)
    pending = cache.reserve(list(range(B)), n)
    q, k, v = projections(device, B, n, Hq, H, D, dtype, seed)
    rng = np.random.default_rng(seed)
    positions = torch.from_numpy(rng.integers(0, far, size=(B, n))).to(device)
    base = 500000.0
    freq = base ** (-np.arange(0, rotary_dim, 2) / rotary_dim)
    table = RotaryTable(rotary_dim, far, base=base, interleaved=interleaved, device=device)
    wq = wk = None
    if norm:
        wq, wk = (torch.rand(D, device=device).add_(0.5).to(weight_dtype) for _ in range(2))
    out = norm_rotate_append(cache, pending, 1, q, k, v, positions, table, query_weight=wq, key_weight=wk, eps=1e-6)
    assert cache.status_bits() == 0
    pos = positions.cpu().numpy()
    want, span = norm_rotate_fp64(f64(q), pos, freq, f64(wq) if norm else None, 1e-6, interleaved)
    want, span = want.transpose(0, 2, 1, 3), span.transpose(0, 2, 1, 3)
    assert out.shape == (B, Hq, n, D) and out.dtype == dtype and out.is_contiguous()
    half_step = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half a step of its subnormals
    err = np.abs(f64(out) - want)
    bound = 24 * U * span * (1 + half_step) + half_step * np.abs(want) + tiny
    assert (err <= bound).all(), float((err - bound).max())

    slots = pending.slots
    keys, kscale, values, vscale = stored(cache, slots, 1)
    for got, scale, source, weight, turn in ((keys, kscale, k, wk, True), (values, vscale, v, None, False)):
        exact, sp = f64(source), np.abs(f64(source))
        if turn:
            exact, sp = norm_rotate_fp64(exact, pos, freq, f64(weight) if norm else None, 1e-6, interleaved)
        exact, sp = exact.reshape(B * n, H, D), sp.reshape(B * n, H, D)
        e = 24 * U * sp if turn else np.zeros_like(sp)
        s_exact = np.abs(exact).max(-1) / 127
        s_err = e.max(-1) / 127 + 2 * U * s_exact
        assert (np.abs(scale - s_exact) <= s_err).all()
        bound = 0.5 * (s_exact + s_err)[..., None] + e + 127 * s_err[..., None]
        assert (np.abs(got - exact) <= bound).all()
    # the other layer, and the slots beyond the reservation, stay zero
    assert int(cache.key_codes[:, 0].abs().max()) == 0
    used = torch.zeros(cache.config.capacity_tokens, dtype=torch.bool, device=device)
    used[slots] = True
    rest = cache.key_codes[:, 1].permute(0, 2, 1, 3).reshape(-1, H, D)[~used]
    assert rest.numel() == 0 or int(rest.abs().max()) == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("D, rotary_dim, interleaved", [
    (64, 64, False), (128, 128, False), (128, 128, True), (16, 16, False), (256, 256, True), (512, 512, False),
    (80, 80, False), (96, 96, True), (80, 32, False), (128, 50, False), (64, 2, True), (112, 112, False)])
def test_every_type_pairing_and_width(device, dtype, D, rotary_dim, interleaved):
    import torch

    check(device, 2, 5, 6, 2, D, getattr(torch, dtype), rotary_dim, interleaved, True, getattr(torch, dtype), 4)


@pytest.mark.parametrize("B, n, Hq, H, block_size", [(1, 1, 1, 1, 1), (1, 1, 32, 8, 16), (3, 37, 7, 7, 5), (64, 6, 32, 8, 16),
                                                     (2, 700, 5, 1, 32)])
@pytest.mark.parametrize("norm", [False, True])
def test_batches_and_heads(device, B, n, Hq, H, block_size, norm):
    import torch

    check(device, B, n, Hq, H, 64, torch.bfloat16, 64, False, norm, torch.float32, block_size)


def test_one_weight_only_and_mixed_weight_types(device):
    import torch

    from specdecode_b200.rotary import RotaryTable, norm_rotate_append

    cache = make_cache(device, 1, 2, 32, 8, 4)
    cache.create_sequence(0)
    table = RotaryTable(32, 64, device=device)
    q, k, v = projections(device, 1, 3, 4, 2, 32, torch.bfloat16, 5)
    positions = torch.arange(3, device=device)
    w = torch.rand(32, device=device) + 0.5
    pending = cache.reserve([0], 3)
    plain = norm_rotate_append(cache, pending, 0, q, k, v, positions, table)
    only_key = norm_rotate_append(cache, pending, 0, q, k, v, positions, table, key_weight=w)
    assert torch.equal(plain, only_key)
    both = norm_rotate_append(cache, pending, 0, q, k, v, positions, table, query_weight=w, key_weight=w)
    mixed = norm_rotate_append(cache, pending, 0, q, k, v, positions, table, query_weight=w,
                               key_weight=w.to(torch.bfloat16))
    assert torch.equal(both, mixed) and not torch.equal(both, plain)


def test_norms_of_large_and_small_elements(device):
    """Squares beyond float32 and below its smallest number."""
    import torch

    from specdecode_b200.rotary import RotaryTable, norm_rotate_append

    D = 64
    for dtype in (torch.bfloat16, torch.float32):
        for exponent in (120, 70, -70, -120):
            cache = make_cache(device, 1, 2, D, 8, 4)
            cache.create_sequence(0)
            pending = cache.reserve([0], 4)
            q, k, v = projections(device, 1, 4, 4, 2, D, torch.float32, 21)
            q, k, v = ((t * 2.0 ** exponent).to(dtype) for t in (q, k, v))
            q[0, 1] *= 2.0 ** -exponent  # ordinary rows beside them
            w = torch.ones(D, device=device)
            freq = 10000.0 ** (-np.arange(0, D, 2) / D)
            pos = np.arange(4)[None]
            table = RotaryTable(D, 8, device=device)
            out = norm_rotate_append(cache, pending, 0, q, k, v, torch.arange(4, device=device), table,
                                     query_weight=w, key_weight=w, eps=1e-6)
            assert cache.status_bits() == 0
            want, span = norm_rotate_fp64(f64(q), pos, freq, f64(w), 1e-6)
            half_step = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
            err = np.abs(f64(out) - want.transpose(0, 2, 1, 3))
            # the second, scaled sum has one rounding more per element
            bound = 28 * U * span.transpose(0, 2, 1, 3) * (1 + half_step) + \
                half_step * np.abs(want.transpose(0, 2, 1, 3)) + 2.0 ** -126
            assert (err <= bound).all(), exponent


def test_position_zero_appends_what_write_layer_appends(device):
    """No rotation, no norm: the same codes and scales, bit for bit, as the
    plain append, from packed views and from separate tensors."""
    import torch

    from specdecode_b200.rotary import RotaryTable, norm_rotate_append

    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        a, b = (make_cache(device, 1, 4, 128, 16, 8) for _ in range(2))
        q, k, v = projections(device, 1, 70, 8, 4, 128, dtype, 3)
        k[0, 3] = 0  # a zero vector: scale 0
        k[0, 4] *= 2.0 ** -100 if dtype != torch.float16 else 1.0
        for c in (a, b):
            c.create_sequence(0)
        pa, pb = a.reserve([0], 70), b.reserve([0], 70)
        table = RotaryTable(128, 4, device=device)
        out = norm_rotate_append(a, pa, 0, q, k, v, torch.zeros(70, dtype=torch.int64, device=device), table)
        b.write_layer(pb, 0, k[0], v[0])
        assert torch.equal(out, q.transpose(1, 2))
        for x, y in ((a.key_codes, b.key_codes), (a.value_codes, b.value_codes),
                     (a.key_scale_pages, b.key_scale_pages), (a.value_scale_pages, b.value_scale_pages)):
            assert torch.equal(x, y)
        # a transposed, misaligned copy of the inputs gives the same
        buffer = torch.empty(k.numel() + 3, dtype=dtype, device=device)[3:].view(k.shape)
        buffer.copy_(k)
        again = norm_rotate_append(a, pa, 0, q.transpose(1, 2).contiguous().transpose(1, 2), buffer, v,
                                   torch.zeros(70, dtype=torch.int32, device=device), table)
        assert torch.equal(again, out) and torch.equal(a.key_codes, b.key_codes)
        assert a.status_bits() == 0


def test_device_paged_cache_slots(device):
    import torch

    from specdecode_b200.device_pages import DevicePagedCache
    from specdecode_b200.kv_cache import KVCacheConfig
    from specdecode_b200.rotary import RotaryTable, norm_rotate_append

    config = KVCacheConfig(1, 2, 64, block_size=8, num_blocks=16)
    a = DevicePagedCache(config, max_rows=2, device=device)
    b = make_cache(device, 1, 2, 64, 8, 16)
    q, k, v = projections(device, 2, 9, 4, 2, 64, torch.float16, 8)
    table = RotaryTable(64, 100, device=device)
    positions = torch.randint(0, 100, (2, 9), device=device)
    for s in range(2):
        b.create_sequence(s)
    x = norm_rotate_append(a, a.reserve([0, 1], [9, 9]), 0, q, k, v, positions, table)
    y = norm_rotate_append(b, b.reserve([0, 1], 9), 0, q, k, v, positions, table)
    a.check_status()
    assert torch.equal(x, y) and torch.equal(a.key_codes, b.key_codes) and torch.equal(a.value_codes, b.value_codes)


def test_faults_leave_slots_unwritten(device):
    import torch

    from specdecode_b200 import _lib
    from specdecode_b200.rotary import RotaryTable, norm_rotate_append

    cache = make_cache(device, 1, 2, 64, 8, 2)
    cache.create_sequence(0)
    pending = cache.reserve([0], 6)
    q, k, v = projections(device, 1, 6, 2, 2, 64, torch.float32, 9)
    k[0, 1, 0, 5] = float("nan")
    v[0, 2, 1, 7] = float("inf")
    k[0, 5, 1] = 0
    k[0, 5, 1, 3] = 2.0 ** -149  # max / 127 underflows
    table = RotaryTable(64, 50, device=device)
    positions = torch.tensor([0, 1, 2, 50, -1, 3], device=device)
    out = norm_rotate_append(cache, pending, 0, q, k, v, positions, table)
    assert cache.status_bits() == (_lib.FAULT_POSITION_RANGE | _lib.FAULT_NONFINITE_VALUE | _lib.FAULT_INVALID_SCALE)
    assert torch.equal(out[0, :, 3:5], torch.zeros_like(out[0, :, 3:5]))
    assert (out[0, :, [0, 1, 2, 5]].abs().amax(-1) > 0).all()
    keys, ks, values, vs = stored(cache, pending.slots, 0)
    written = ks > 0
    assert written.tolist() == [[True, True], [False, True], [True, True], [False, False], [False, False], [True, False]]
    assert (vs > 0).tolist() == [[True, True], [True, True], [True, False], [False, False], [False, False], [True, True]]
    # slots outside the pool: queries still come back, nothing is written
    before = cache.key_codes.clone()
    slots = torch.tensor([-1, 16, 1 << 40, -5, 17, 99], device=device)
    q2, k2, v2 = projections(device, 1, 6, 2, 2, 64, torch.float32, 10)
    out = norm_rotate_append(cache, slots, 0, q2, k2, v2, torch.arange(6, device=device), table)
    assert cache.status_bits() == _lib.FAULT_SLOT_RANGE
    assert torch.equal(cache.key_codes, before) and bool((out.abs().amax(-1) > 0).all())


def test_a_stream_a_graph_and_a_given_output(device):
    import torch

    from specdecode_b200.rotary import RotaryTable, norm_rotate_append

    cache = make_cache(device, 1, 2, 128, 16, 4)
    cache.create_sequence(0)
    pending = cache.reserve([0], 5)
    q, k, v = projections(device, 1, 5, 8, 2, 128, torch.bfloat16, 11)
    positions = torch.arange(5, device=device)
    table = RotaryTable(128, 64, device=device)
    want = norm_rotate_append(cache, pending, 0, q, k, v, positions, table)
    codes = cache.key_codes.clone()
    out = torch.empty_like(want)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    cache.key_codes.zero_()
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        norm_rotate_append(cache, pending, 0, q, k, v, positions, table, out=out)
    torch.cuda.current_stream(device).wait_stream(side)
    assert torch.equal(out, want) and torch.equal(cache.key_codes, codes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm_rotate_append(cache, pending, 0, q, k, v, positions, table, out=out)
    cache.key_codes.zero_()
    q.mul_(-1.0)
    graph.replay()
    assert torch.equal(out, -want) and torch.equal(cache.key_codes, codes)


def test_refusals(device):
    import torch

    from specdecode_b200.rotary import RotaryTable, norm_rotate_append

    cache = make_cache(device, 1, 2, 64, 8, 4)
    cache.create_sequence(0)
    pending = cache.reserve([0], 3)
    q, k, v = projections(device, 1, 3, 4, 2, 64, torch.bfloat16, 1)
    positions = torch.arange(3, device=device)
    table = RotaryTable(64, 64, device=device)
    w = torch.ones(64, device=device)

    def call(q=q, k=k, v=v, positions=positions, table=table, pending=pending, layer=0, **kw):
        return norm_rotate_append(cache, pending, layer, q, k, v, positions, table, **kw)

    call()
    for error, kw in [
            (ValueError, dict(q=q[0])), (ValueError, dict(q=q[:, :, :3])), (TypeError, dict(q=q.double())),
            (TypeError, dict(k=k.float())), (ValueError, dict(v=v[:, :2])), (ValueError, dict(k=k.cpu())),
            (ValueError, dict(layer=1)), (ValueError, dict(positions=positions[:2])),
            (TypeError, dict(positions=positions.float())), (ValueError, dict(positions=positions.cpu())),
            (TypeError, dict(table=table.values)), (ValueError, dict(table=RotaryTable(128, 4, device=device))),
            (ValueError, dict(table=RotaryTable(64, 4, device="cpu"))), (TypeError, dict(pending=[0, 1, 2])),
            (ValueError, dict(pending=pending.slots[:2])), (ValueError, dict(pending=pending.slots.cpu())),
            (ValueError, dict(query_weight=w[:32])), (TypeError, dict(key_weight=w.double())),
            (ValueError, dict(key_weight=w.cpu())), (ValueError, dict(key_weight=w, eps=0.0)),
            (ValueError, dict(out=torch.empty((1, 4, 3, 64), device=device)))]:
        with pytest.raises(error):
            call(**kw)
    # no tokens: an empty result, no launch
    empty = call(q=q[:, :0], k=k[:, :0], v=v[:, :0], positions=positions[:0], pending=pending.slots[:0])
    assert empty.shape == (1, 4, 0, 64)
    assert cache.status_bits() == 0
