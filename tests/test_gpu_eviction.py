"""Attention mass, selection, compaction and eviction against float64 and
against the definitions: exact where whole numbers or moved bits come out.

Tolerance of the mass.  u = 2^-24.  A score is a sum of D products, exact in
float32 (an f16 query element times a code), each addition of the tensor cores
off by at most 2 u of the partial sums: 2 D u A with A the largest sum over d of
|q_d k_d| / sqrt(D); the three scaling products add 3 u A.  float32 queries lose
2^-22 of their row's largest element: 2^-22 B with B that element times the
largest sum |k_d| / sqrt(D).  The running maximum and the row sum's own scores
err alike, so a weight is off by exp of twice that, and by its sums: at most n =
T / 32 + 300 additions and products of u each (a thread adds the tokens of its
tiles, one in 128 of a block's, two at a time; then eight lanes, eight warps,
sixteen blocks), with 2 ulp = 4 u for each of four exponentials.  The rows' sum
adds 70 u, the addition to the stored mass one u of the result."""

from __future__ import annotations

import math

import numpy as np
import pytest

from gpu_helpers import make_cache
from oracle.attention import attention_fp64
from oracle.eviction import attention_mass_fp64, norm_rotate_fp64, select_kept

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def filled(device, lengths, layers, heads, head_dim, block_size, seed=0, spare=3, track=True, scale=(0.005, 0.05)):
    """A cache of sequences 0, 1, ... with random codes and scales in their
    slots, blocks in shuffled order, zeros elsewhere."""
    import torch

    blocks = sum(-(-n // block_size) for n in lengths) + spare
    rng = np.random.default_rng(seed)
    longest = max(max(-(-n // block_size) for n in lengths) + 2, 1)
    cache = make_cache(device, layers, heads, head_dim, block_size, blocks, block_order=rng.permutation(blocks),
                       max_sequences=len(lengths), max_blocks_per_sequence=longest)
    g = torch.Generator(device=device).manual_seed(seed)
    if track:
        cache.track_attention()
    for s, n in enumerate(lengths):
        cache.create_sequence(s)
        if n:
            slots = cache.reserve([s], n).slots
            b, o = slots // block_size, slots % block_size
            shape = (n, layers, heads, head_dim)
            for codes, scales in ((cache.key_codes, cache.key_scale_pages),
                                  (cache.value_codes, cache.value_scale_pages)):
                codes[b, :, :, o] = torch.randint(-127, 128, shape, generator=g, device=device).to(torch.int8)
                scales[b, :, :, o] = torch.rand(shape[:3], generator=g, device=device) * (scale[1] - scale[0]) + scale[0]
    return cache


def tokens(cache, sequence, pages):
    """Pages [block, layer, head, offset, ...] of a sequence as [T, layer, head, ...]."""
    import torch

    slots = torch.from_numpy(cache.page_table.slots_of(sequence, 0, cache.sequence_length(sequence))).to(pages.device)
    bs = cache.config.block_size
    return pages[slots // bs, :, :, slots % bs]


def keys_fp64(cache, sequence, layer):
    k = tokens(cache, sequence, cache.key_codes)[:, layer].double()
    return (k * tokens(cache, sequence, cache.key_scale_pages)[:, layer].double()[..., None]).cpu().numpy()


def mass_of(cache, sequence, layer):
    return tokens(cache, sequence, cache.attention_mass)[:, layer].double().cpu().numpy().T  # [H, T]


def free_mass(cache):
    """The largest mass of a slot no token occupies."""
    import torch

    occupied = torch.from_numpy(cache.page_table.occupied).to(cache.device)
    m = cache.attention_mass.abs().amax(dim=(1, 2))
    return float(m[~occupied].max()) if bool((~occupied).any()) else 0.0


def bounds(q, keys, T, split):
    D = q.shape[-1]
    group = q.shape[0] // keys.shape[1]
    A = B = 0.0
    for h in range(q.shape[0]):
        k = np.abs(keys[:, h // group])
        A = max(A, float((np.abs(q[h]) @ k.T).max()) / math.sqrt(D))
        B = max(B, float(np.abs(q[h]).max() * k.sum(axis=1).max()) / math.sqrt(D))
    score = (2 * D + 3) * U * A + (2.0 ** -22 * B if split else 0.0)
    return math.expm1(2 * score) + (T / 32 + 300 + 16 + 70) * U


def check_observe(device, lengths, Hq, H, D, window, dtype, block_size, seed=0, passes=1, layer=1, qscale=1.0):
    import torch

    from specdecode_b200.eviction import observe_attention

    cache = filled(device, lengths, 2, H, D, block_size, seed)
    g = torch.Generator(device=device).manual_seed(seed + 1)
    want = [np.zeros((H, n)) for n in lengths]
    rel = 0.0
    for _ in range(passes):
        q = (torch.randn((len(lengths), Hq, window, D), generator=g, device=device) * 2 * qscale).to(dtype)
        pages = observe_attention(cache, q, list(range(len(lengths))), layer)
        assert pages is cache.attention_mass
        for s in range(len(lengths)):
            qs, ks = q[s].double().cpu().numpy(), keys_fp64(cache, s, layer)
            want[s] += attention_mass_fp64(qs, ks)
            rel = max(rel, bounds(qs, ks, lengths[s], dtype == torch.float32))
    assert cache.status_bits() == 0
    for s in range(len(lengths)):
        got = mass_of(cache, s, layer)
        # weights below 2^-126 may flush to zero, row by row
        bound = rel * want[s] + passes * U * want[s] + passes * Hq * window * 2.0 ** -126
        assert (np.abs(got - want[s]) <= bound).all(), (s, float((np.abs(got - want[s]) - bound).max()))
        assert not mass_of(cache, s, 1 - layer).any()
    assert free_mass(cache) == 0.0


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
def test_observe_every_type_and_head_size(device, dtype, D):
    import torch

    check_observe(device, [5, 131, 64, 700], 8, 2, D, 5, getattr(torch, dtype), 16, passes=2)


@pytest.mark.parametrize("lengths, Hq, H, window, block_size", [
    ([1], 1, 1, 1, 1),              # one token, one row
    ([7, 9, 8], 4, 2, 7, 3),        # a window as long as its context, blocks inside a tile
    ([16, 17, 15, 1], 6, 3, 1, 7),  # tile borders
    ([300, 60], 2, 2, 60, 32),      # many window rows: 60
    ([129], 64, 1, 1, 64),          # 64 heads on one KV head
    ([513, 40], 9, 1, 3, 16),       # 27 rows
    ([200], 10, 1, 2, 5),           # 20 rows
    ([100] * 40, 8, 4, 2, 16),      # more sequences than blocks per SM
])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_observe_shapes(device, lengths, Hq, H, window, block_size, dtype):
    import torch

    check_observe(device, lengths, Hq, H, 64, window, getattr(torch, dtype), block_size)


@pytest.mark.parametrize("lengths, Hq, H, D, window, dtype", [
    ([30011], 16, 1, 64, 4, "bfloat16"),     # 64 rows: most tiles do not stay in shared memory
    ([20001, 37, 9000], 8, 2, 128, 5, "float16"),
    ([16400], 32, 1, 256, 2, "float32"),
    ([70001], 4, 1, 16, 1, "bfloat16"),
])
def test_observe_long_contexts(device, lengths, Hq, H, D, window, dtype):
    import torch

    check_observe(device, lengths, Hq, H, D, window, getattr(torch, dtype), 16)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("qscale", [2.0 ** 40, 2.0 ** -60, 0.0])
def test_observe_extreme_queries(device, dtype, qscale):
    """Queries whose scores saturate (one token takes the row), or vanish
    (every visible token gets the same)."""
    import torch

    if qscale > 1:  # one token takes all: exactly its rows' count
        from specdecode_b200.eviction import observe_attention

        cache = filled(device, [333], 2, 2, 64, 16)
        q = (torch.randn((1, 4, 1, 64), device=device) * qscale).to(getattr(torch, dtype))
        observe_attention(cache, q, [0], 1)
        keys = keys_fp64(cache, 0, 1)
        want = np.zeros((2, 333))
        for h in range(4):
            want[h // 2, int(np.argmax(keys[:, h // 2] @ q[0, h, 0].double().cpu().numpy()))] += 1
        assert np.array_equal(mass_of(cache, 0, 1), want)
        assert cache.status_bits() == 0
    else:
        check_observe(device, [333, 4], 4, 2, 64, 3, getattr(torch, dtype), 16, qscale=qscale)


def test_observe_leaves_out_rows_that_are_not_finite(device):
    import torch

    from specdecode_b200 import _lib
    from specdecode_b200.eviction import observe_attention

    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        cache = filled(device, [70, 90], 2, 2, 64, 16)
        q = torch.randn((2, 4, 3, 64), device=device).to(dtype)
        clean = q.clone()
        q[0, 0, 1, 5] = float("nan")
        q[1, 3, 2, 0] = float("-inf")
        observe_attention(cache, q, [0, 1], 1)
        assert cache.status_bits() == _lib.FAULT_NONFINITE_VALUE
        for s, (h, i) in ((0, (0, 1)), (1, (3, 2))):
            keys = keys_fp64(cache, s, 1)
            qs = clean[s].double().cpu().numpy()
            want = attention_mass_fp64(qs, keys)
            # less the poisoned row, alone
            T = keys.shape[0]
            visible = T - 3 + i + 1
            sc = qs[h, i] @ keys[:visible, h // 2].T / 8.0
            p = np.exp(sc - sc.max())
            want[h // 2, :visible] -= p / p.sum()
            got = mass_of(cache, s, 1)
            assert np.isfinite(got).all()
            # (the subtraction above is exact to 2^-50)
            assert (np.abs(got - want) <= bounds(qs, keys, T, True) * np.abs(want) + 1e-12 + U * want).all()


def test_observe_faults_change_nothing_or_leave_tokens_out(device):
    import torch

    from specdecode_b200 import _lib
    from specdecode_b200.eviction import observe_rows

    cache = filled(device, [50, 60], 1, 2, 64, 16)
    q = torch.randn((2, 4, 2, 64), device=device)
    tables, lens, longest = cache.attention_inputs([0, 1])
    assert longest == 60
    # a bound below the second context; a context shorter than the window
    observe_rows(cache, q, tables, lens, 55, 0)
    assert cache.status_bits() == _lib.FAULT_CONTEXT_RANGE
    assert mass_of(cache, 0, 0).any() and not mass_of(cache, 1, 0).any()
    cache.attention_mass.zero_()
    observe_rows(cache, q, tables, torch.tensor([1, -3], dtype=torch.int32, device=device), 60, 0)
    assert cache.status_bits() == _lib.FAULT_CONTEXT_RANGE
    assert not bool(cache.attention_mass.any())
    observe_rows(cache, q, tables, torch.tensor([50, 1 << 20], dtype=torch.int32, device=device), 1 << 21, 0)
    assert cache.status_bits() == _lib.FAULT_CONTEXT_RANGE
    assert mass_of(cache, 0, 0).any() and not mass_of(cache, 1, 0).any()
    # blocks outside the pool: their tokens are left out of the softmax
    cache.attention_mass.zero_()
    broken = tables.clone()
    broken[0, 1] = -1
    broken[0, 2] = cache.config.num_blocks
    observe_rows(cache, q, broken, lens, 60, 0)
    assert cache.status_bits() == _lib.FAULT_BLOCK_RANGE
    keys = keys_fp64(cache, 0, 0)
    left = np.r_[0:16, 48:50]
    got, qs = mass_of(cache, 0, 0), q[0].double().cpu().numpy()
    assert not got[:, 16:48].any()
    # the window's two rows see 48 and 49 tokens: here 16 + 1 and 16 + 2
    want = attention_mass_fp64(qs, keys[left])
    assert (np.abs(got[:, left] - want) <= bounds(qs, keys, 50, True) * want + U * want).all()


@pytest.mark.parametrize("rows", range(1, 25))
def test_observe_every_number_of_rows_of_short_contexts(device, rows):
    import torch

    for D, dtype in ((64, torch.float32), (128, torch.bfloat16)):
        check_observe(device, [rows, 161, 320], 2, 2, D, rows, dtype, 16)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("Hq, window, D", [(4, 2, 64), (8, 3, 128), (16, 3, 64), (16, 4, 128)])
def test_observe_in_one_launch_and_in_two(device, dtype, Hq, window, D):
    """The bound on the contexts decides whether one block keeps a context's
    scores; both forms hold, with a poisoned row and a block outside the pool."""
    import torch

    from specdecode_b200 import _lib
    from specdecode_b200.eviction import observe_rows

    lengths = [333, window, 160]
    cache = filled(device, lengths, 1, 2, D, 16)
    split = dtype == "float32"
    q = torch.randn((3, Hq, window, D), device=device).to(getattr(torch, dtype))
    clean = q.double().cpu().numpy()
    q[2, Hq - 1, 0, 7] = float("nan")
    tables, lens, _ = cache.attention_inputs([0, 1, 2])
    tables = tables.clone()
    tables[2, 3] = cache.config.num_blocks  # tokens 48 .. 63
    left = np.r_[0:48, 64:160]
    for bound in (333, 40000):
        cache.attention_mass.zero_()
        observe_rows(cache, q, tables, lens, bound, 0)
        assert cache.status_bits() == _lib.FAULT_NONFINITE_VALUE | _lib.FAULT_BLOCK_RANGE
        for s in range(3):
            keys, qs, got = keys_fp64(cache, s, 0), clean[s], mass_of(cache, s, 0)
            rel = bounds(qs, keys, lengths[s], split)
            assert np.isfinite(got).all()
            if s == 2:
                assert not got[:, 48:64].any()
                got, keys = got[:, left], keys[left]
            want = attention_mass_fp64(qs, keys)
            if s == 2:  # less the poisoned row
                visible = len(left) - window + 1
                sc = qs[Hq - 1, 0] @ keys[:visible, 1].T / math.sqrt(D)
                p = np.exp(sc - sc.max())
                want[1, :visible] -= p / p.sum()
            assert (np.abs(got - want) <= rel * np.abs(want) + 1e-12 + U * np.abs(want)).all()


@pytest.mark.parametrize("lengths, Hq, H, D, window, dtype", [
    ([1500] * 80, 8, 8, 64, 2, "float32"),       # 640 pairs with 47 KB of scores each: two launches
    ([1100, 700] * 40, 8, 8, 64, 1, "bfloat16"),  # with 35 KB: one launch
    ([1024], 12, 2, 128, 4, "float16"),          # few pairs: chunks of four tiles
    ([800] * 50, 12, 4, 128, 3, "float32"),
    ([512] * 60, 24, 4, 128, 4, "float32"),      # 24 rows, two blocks an SM, one launch
    ([513, 512, 33], 24, 2, 64, 2, "float16"),
    ([2200, 1], 4, 4, 128, 1, "float32"),
    ([2200, 3], 24, 2, 64, 2, "bfloat16"),
    ([40000], 4, 1, 64, 1, "float16"),           # chunks of three tiles a warp
])
def test_observe_between_one_launch_and_two(device, lengths, Hq, H, D, window, dtype):
    import torch

    lengths = [max(n, window) for n in lengths]
    check_observe(device, lengths, Hq, H, D, window, getattr(torch, dtype), 16)


def test_observe_is_deterministic_on_a_stream_and_in_a_graph(device):
    import torch

    from specdecode_b200.eviction import observe_attention

    cache = filled(device, [3001, 20, 700], 2, 4, 128, 16)
    q = torch.randn((3, 16, 5, 128), device=device).to(torch.bfloat16)
    first = observe_attention(cache, q, [0, 1, 2], 0).clone()
    for _ in range(3):
        cache.attention_mass.zero_()
        assert torch.equal(observe_attention(cache, q, [0, 1, 2], 0), first)
    cache.attention_mass.zero_()
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        observe_attention(cache, q, [0, 1, 2], 0)
    torch.cuda.current_stream(device).wait_stream(side)
    assert torch.equal(cache.attention_mass, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        observe_attention(cache, q, [0, 1, 2], 0)
    assert torch.equal(cache.attention_mass, first)  # capture runs nothing
    cache.attention_mass.zero_()
    graph.replay()
    assert torch.equal(cache.attention_mass, first)
    # listed in another order, through gathered tables
    cache.attention_mass.zero_()
    observe_attention(cache, q[[2, 0, 1]], [2, 0, 1], 0)
    assert torch.equal(cache.attention_mass, first)


def test_observation_selection_and_compaction_replayed(device):
    """Captured once and replayed: each replay selects by the mass as it then
    is, and compacts."""
    import torch

    from specdecode_b200.eviction import compact_tokens, observe_attention, select_tokens

    cache = filled(device, [300, 257], 2, 2, 64, 16)
    q = torch.randn((2, 4, 3, 64), device=device).to(torch.bfloat16)
    states = [t.clone() for t in (cache.key_codes, cache.key_scale_pages, cache.value_codes, cache.value_scale_pages)]

    def restore():
        for t, s in zip((cache.key_codes, cache.key_scale_pages, cache.value_codes, cache.value_scale_pages), states):
            t.copy_(s)
        cache.attention_mass.zero_()

    def step():
        for layer in range(2):
            observe_attention(cache, q, [0, 1], layer)
        kept = select_tokens(cache, [0, 1], 64, recent=8, sinks=2)
        compact_tokens(cache, [0, 1], kept)
        return kept

    def result(kept):
        return [t.clone() for t in (kept, cache.key_codes, cache.key_scale_pages, cache.value_codes,
                                    cache.value_scale_pages, cache.attention_mass)]

    restore()
    first = result(step())
    restore()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for _ in range(2):
        restore()
        kept.zero_()
        graph.replay()
        for got, want in zip(result(kept), first):
            assert torch.equal(got, want)
    q.mul_(-1.0)  # other queries, the same graph
    restore()
    graph.replay()
    second = result(kept)
    restore()
    for got, want in zip(second, result(step())):
        assert torch.equal(got, want)
    assert not torch.equal(second[0], first[0])
    assert cache.status_bits() == 0


def test_observe_from_two_threads(device):
    """Contexts of different lengths, so blocks of different shared memory, from
    two threads on their own streams and caches."""
    import threading

    import torch

    from specdecode_b200.eviction import observe_attention

    states = []
    for seed, lengths in enumerate(([512] * 20, [400] * 20)):
        cache = filled(device, lengths, 1, 2, 128, 16, seed)
        q = torch.randn((20, 16, 3, 128), device=device).to(torch.bfloat16)
        want = observe_attention(cache, q, list(range(20)), 0).clone()
        cache.attention_mass.zero_()
        states.append((cache, q, want))
    torch.cuda.synchronize(device)
    failures = []

    def work(cache, q, want):
        try:
            with torch.cuda.device(device), torch.cuda.stream(torch.cuda.Stream(device)):
                for _ in range(200):
                    cache.attention_mass.zero_()
                    observe_attention(cache, q, list(range(20)), 0)
                torch.cuda.current_stream(device).synchronize()
            assert torch.equal(cache.attention_mass, want)
        except BaseException as error:  # noqa: BLE001
            failures.append(error)

    threads = [threading.Thread(target=work, args=s) for s in states]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


def test_observe_in_rounds(device, monkeypatch):
    """A workspace for one (sequence, KV head), and for a few of them, gives
    what one for all of them gives."""
    import torch

    from specdecode_b200 import eviction

    cache = filled(device, [900, 31, 2500], 2, 2, 64, 16)
    q = torch.randn((3, 8, 3, 64), device=device).to(torch.float16)
    want = eviction.observe_attention(cache, q, [0, 1, 2], 1).clone()
    for size in (1, 600000, 1000000):
        monkeypatch.setattr(eviction, "WORKSPACE_BYTES", size)
        cache.attention_mass.zero_()
        assert torch.equal(eviction.observe_attention(cache, q, [0, 1, 2], 1), want)
    assert cache.status_bits() == 0


def set_mass(cache, sequence, values):
    """values [T, layers, heads]."""
    import torch

    slots = torch.from_numpy(cache.page_table.slots_of(sequence, 0, cache.sequence_length(sequence))).to(cache.device)
    bs = cache.config.block_size
    cache.attention_mass[slots // bs, :, :, slots % bs] = torch.from_numpy(values.astype(np.float32)).to(cache.device)


def drawn_mass(rng, kind, shape):
    if kind == "heavy":
        return np.exp(rng.standard_normal(shape) * 3)
    if kind == "ties":
        return rng.integers(0, 4, shape) / 4.0
    if kind == "equal":
        return np.full(shape, 0.25)
    m = rng.standard_normal(shape)  # negative, zeros of both signs, infinities, NaN
    m[rng.random(shape) < 0.1] = 0.0
    m[rng.random(shape) < 0.1] = -0.0
    m[rng.random(shape) < 0.05] = np.inf
    m[rng.random(shape) < 0.05] = -np.inf
    m[rng.random(shape) < 0.05] = np.nan
    return m


@pytest.mark.parametrize("kind", ["heavy", "ties", "equal", "odd"])
@pytest.mark.parametrize("lengths, budget, recent, sinks, block_size", [
    ([1, 2, 3], 1, 0, 0, 1),
    ([40, 41, 39, 500], 40, 8, 4, 16),
    ([1000, 17], 999, 3, 1, 7),
    ([2500, 800], 64, 32, 32, 16),    # nothing chosen by mass
    ([3000], 1, 1, 0, 32),
    ([5001, 4097], 1500, 0, 0, 16),
])
def test_select(device, kind, lengths, budget, recent, sinks, block_size):
    from specdecode_b200.eviction import select_tokens

    L, H = 3, 2
    cache = filled(device, lengths, L, H, 16, block_size)
    rng = np.random.default_rng(5)
    masses = [drawn_mass(rng, kind, (n, L, H)).astype(np.float32) for n in lengths]
    for s, m in enumerate(masses):
        set_mass(cache, s, m)
    kept = select_tokens(cache, list(range(len(lengths))), budget, recent=recent, sinks=sinks).cpu().numpy()
    assert cache.status_bits() == 0
    for s, m in enumerate(masses):
        for layer in range(L):
            for h in range(H):
                assert np.array_equal(kept[s, layer, h], select_kept(m[:, layer, h], budget, recent, sinks)), (s, layer, h)


@pytest.mark.parametrize("length, budget", [(70001, 5000), (131072, 100000), (400003, 7)])
def test_select_long_rows(device, length, budget):
    """Rows split over a cluster, and (the longest) larger than its shared memory."""
    from specdecode_b200.eviction import select_tokens

    cache = filled(device, [length], 1, 2, 16, 64)
    rng = np.random.default_rng(6)
    for kind in ("heavy", "ties"):
        m = drawn_mass(rng, kind, (length, 1, 2)).astype(np.float32)
        set_mass(cache, 0, m)
        kept = select_tokens(cache, [0], budget, recent=3, sinks=2).cpu().numpy()
        for h in range(2):
            assert np.array_equal(kept[0, 0, h], select_kept(m[:, 0, h], budget, 3, 2))
    assert cache.status_bits() == 0


@pytest.mark.parametrize("length", [40000, 70001])
def test_select_many_long_rows(device, length):
    """Rows enough for the SMs: a block (or two) holds each, part of it in
    shared memory."""
    from specdecode_b200.eviction import select_tokens

    L, H = 40, 2
    cache = filled(device, [length], L, H, 16, 64)
    rng = np.random.default_rng(8)
    m = drawn_mass(rng, "heavy", (length, L, H)).astype(np.float32)
    m[:, ::2] = drawn_mass(rng, "ties", (length, L // 2, H))
    set_mass(cache, 0, m)
    kept = select_tokens(cache, [0], 3000, recent=5, sinks=3).cpu().numpy()
    assert cache.status_bits() == 0
    for layer in range(L):
        for h in range(H):
            assert np.array_equal(kept[0, layer, h], select_kept(m[:, layer, h], 3000, 5, 3)), (layer, h)


def test_select_faults(device):
    import torch

    from specdecode_b200 import _lib

    cache = filled(device, [40, 50], 1, 1, 16, 16)
    set_mass(cache, 0, np.arange(40.0)[:, None, None])
    set_mass(cache, 1, np.arange(50.0)[:, None, None])
    tables, lens, _ = cache.attention_inputs([0, 1])
    kept = torch.full((2, 1, 1, 20), 7, dtype=torch.int32, device=device)

    def call(tables, lens, longest):
        st = cache.library.handle.sdc_select_tokens(
            cache.pool_desc, cache.attention_mass.data_ptr(), 2, tables.data_ptr(), tables.stride(0), lens.data_ptr(),
            longest, 20, 4, 0, kept.data_ptr(), cache._status.data_ptr(), torch.cuda.current_stream(device).cuda_stream)
        assert st == 0

    call(tables, lens, 45)  # the second context is longer than the bound
    assert cache.status_bits() == _lib.FAULT_CONTEXT_RANGE
    assert kept[0, 0, 0].tolist() == list(range(20, 40)) and kept[1, 0, 0].tolist() == [-1] * 20
    broken = tables.clone()
    broken[0, 1] = -1  # tokens 16 .. 31 count as mass 0: the first of them only where nothing is left
    call(broken, lens, 50)
    assert cache.status_bits() == _lib.FAULT_BLOCK_RANGE
    want = select_kept(np.where((np.arange(40) >= 16) & (np.arange(40) < 32), 0.0, np.arange(40.0)).astype(np.float32),
                       20, 4, 0)
    assert kept[0, 0, 0].tolist() == want.tolist()


def random_kept(rng, lengths, L, H, budget):
    kept = np.full((len(lengths), L, H, budget), -1, dtype=np.int32)
    for s, n in enumerate(lengths):
        for layer in range(L):
            for h in range(H):
                row = np.sort(rng.choice(n, budget, replace=False)) if n > budget else np.arange(n)
                kept[s, layer, h, :len(row)] = row
    return kept


def snapshot(cache):
    return {name: getattr(cache, name).clone() for name in
            ("key_codes", "value_codes", "key_scale_pages", "value_scale_pages", "attention_mass")}


def expect_compacted(cache, before, lengths, kept, skip=()):
    """``before`` with every kept row moved, by indexing."""
    import torch

    budget = kept.shape[-1]
    bs = cache.config.block_size
    want = {name: pages.clone() for name, pages in before.items()}
    for s, n in enumerate(lengths):
        if n <= budget:
            continue
        slots = torch.from_numpy(cache.page_table.slots_of(s, 0, n)).to(cache.device)
        for layer in range(kept.shape[1]):
            for h in range(kept.shape[2]):
                if (s, layer, h) in skip:
                    continue
                src = slots[torch.from_numpy(kept[s, layer, h].astype(np.int64)).to(cache.device)]
                dst = slots[:budget]
                for name, pages in before.items():
                    want[name][dst // bs, layer, h, dst % bs] = pages[src // bs, layer, h, src % bs]
    return want


@pytest.mark.parametrize("D", [16, 48, 64, 128, 512])
@pytest.mark.parametrize("lengths, budget, block_size", [
    ([2, 5, 3], 1, 1), ([100, 64, 63, 300], 63, 16), ([1000], 999, 7), ([3000, 10], 1200, 32), ([50], 50, 16)])
def test_compact(device, D, lengths, budget, block_size):
    import torch

    from specdecode_b200.eviction import compact_tokens

    L, H = 2, 3
    cache = filled(device, lengths, L, H, D, block_size)
    cache.attention_mass.uniform_()
    rng = np.random.default_rng(7)
    kept = random_kept(rng, lengths, L, H, budget)
    kept[0, 0, 0] = np.arange(budget) if lengths[0] > budget else kept[0, 0, 0]  # nothing moves
    before = snapshot(cache)
    compact_tokens(cache, list(range(len(lengths))), torch.from_numpy(kept).to(device))
    assert cache.status_bits() == 0
    for name, want in expect_compacted(cache, before, lengths, kept).items():
        assert torch.equal(getattr(cache, name), want), name
    assert [cache.sequence_length(s) for s in range(len(lengths))] == lengths


def test_compact_without_mass_pages(device):
    import torch

    from specdecode_b200.eviction import compact_tokens

    cache = filled(device, [90], 1, 2, 64, 16, track=False)
    kept = random_kept(np.random.default_rng(1), [90], 1, 2, 30)
    keys = tokens(cache, 0, cache.key_codes)
    compact_tokens(cache, [0], torch.from_numpy(kept).to(device))
    got = tokens(cache, 0, cache.key_codes)[:30]
    for h in range(2):
        assert torch.equal(got[:, 0, h], keys[torch.from_numpy(kept[0, 0, h].astype(np.int64)).to(device), 0, h])


def test_compact_refuses_rows_out_of_order(device):
    """A row that is not ascending inside the sequence moves nothing; the
    other rows do."""
    import torch

    from specdecode_b200 import _lib
    from specdecode_b200.eviction import compact_tokens

    lengths, budget, L, H = [200, 150], 40, 2, 4
    cache = filled(device, lengths, L, H, 64, 16)
    cache.attention_mass.uniform_()
    kept = random_kept(np.random.default_rng(3), lengths, L, H, budget)
    kept[0, 0, 0, 39] = 200                    # past the context
    kept[0, 1, 1, 20] = kept[0, 1, 1, 19]      # twice the same
    kept[1, 0, 2] = kept[1, 0, 2][::-1]        # descending
    kept[1, 1, 3, 0] = -1
    skip = {(0, 0, 0), (0, 1, 1), (1, 0, 2), (1, 1, 3)}
    before = snapshot(cache)
    compact_tokens(cache, [0, 1], torch.from_numpy(kept).to(device))
    assert cache.status_bits() == _lib.FAULT_KEPT_ORDER
    for name, want in expect_compacted(cache, before, lengths, kept, skip).items():
        assert torch.equal(getattr(cache, name), want), name


def test_released_slots_have_no_mass(device):
    import torch

    from specdecode_b200.eviction import observe_attention

    cache = filled(device, [100, 40], 2, 2, 64, 16)
    q = torch.randn((2, 4, 1, 64), device=device)
    for layer in range(2):
        observe_attention(cache, q, [0, 1], layer)
    assert free_mass(cache) == 0.0 and mass_of(cache, 0, 1)[:, 37:].all()
    cache.truncate_batch([0, 1], [37, 39])
    assert free_mass(cache) == 0.0 and mass_of(cache, 0, 1).all()
    cache.remove_sequence(1)
    assert free_mass(cache) == 0.0
    cache.remove_sequence(0)
    assert not bool(cache.attention_mass.any())
    assert cache.status_bits() == 0


def test_a_long_decode_in_a_small_pool(device):
    """The operators as they are used: tokens appended at their true positions
    through norm_rotate_append, attention over them, their weights observed,
    the sequences trimmed whenever they pass a limit -- against float64 kept
    per head on the host."""
    import torch

    from specdecode_b200.cuda_kv_cache import paged_verify_attention
    from specdecode_b200.eviction import evict, observe_attention
    from specdecode_b200.rotary import RotaryTable, norm_rotate_append

    L, Hq, H, D, B, bs = 2, 8, 2, 64, 2, 16
    limit, budget, recent, sinks, step = 96, 48, 12, 2, 10
    cache = make_cache(device, L, H, D, bs, 2 * B * 8, max_sequences=B)
    cache.track_attention()
    table = RotaryTable(D, 4096, base=10000.0, device=device)
    freq = 10000.0 ** (-np.arange(0, D, 2) / D)
    g = torch.Generator(device=device).manual_seed(0)
    w = torch.rand(D, generator=g, device=device) + 0.5
    ids = [0, 1]
    for s in ids:
        cache.create_sequence(s)
    # per (sequence, layer, head): the true positions its cached tokens stand for
    stands = {(s, layer, h): [] for s in ids for layer in range(L) for h in range(H)}
    history = {}
    position, evictions = 0, 0
    while position < 260:
        n = step if position else 30
        pending = cache.reserve(ids, n)
        positions = torch.arange(position, position + n, device=device)
        for layer in range(L):
            packed = torch.randn((B, n, Hq + 2 * H, D), generator=g, device=device).to(torch.bfloat16)
            q, k, v = packed[:, :, :Hq], packed[:, :, Hq:Hq + H], packed[:, :, Hq + H:]
            query = norm_rotate_append(cache, pending, layer, q, k, v, positions, table, query_weight=w, key_weight=w)
            rotated, _ = norm_rotate_fp64(k.double().cpu().numpy(), np.arange(position, position + n)[None].repeat(B, 0),
                                          freq, w.double().cpu().numpy())
            for s in ids:
                for h in range(H):
                    stands[s, layer, h] += range(position, position + n)
                    for i in range(n):
                        history[s, layer, h, position + i] = rotated[s, i, h]
            for i in range(0, n, 16):  # windows of at most 16 rows per query head
                part = query[:, :, i:i + 16]
                if i + 16 < n:
                    continue  # earlier windows only matter to the mass; the last one is checked
                out = paged_verify_attention(cache, part, ids, layer)
                before = cache.attention_mass.clone()
                observe_attention(cache, part, ids, layer)
                grown = (cache.attention_mass - before).double().sum().item()
                rows = B * Hq * part.shape[2]
                assert abs(grown - rows) <= 1e-3 * rows  # one unit a row
                for s in ids:
                    kq, vq = (tokens(cache, s, p)[:, layer].cpu().numpy() for p in (cache.key_codes, cache.value_codes))
                    ks, vs = (tokens(cache, s, p)[:, layer].cpu().numpy() for p in (cache.key_scale_pages,
                                                                                    cache.value_scale_pages))
                    exact = attention_fp64(part[s].double().cpu().numpy(), kq, vq, ks, vs)
                    # the attention's own bound (bf16 output and 15-bit operands)
                    assert np.abs(out[s].double().cpu().numpy() - exact).max() <= 2e-2
                    for h in range(H):
                        # every cached key is its true token's, to half a code step
                        for t, p in enumerate(stands[s, layer, h]):
                            assert np.abs(kq[t, h] * np.float64(ks[t, h]) - history[s, layer, h, p]).max() <= \
                                0.5001 * ks[t, h] + 1e-5
        position += n
        if cache.sequence_length(0) > limit:
            mass = {s: tokens(cache, s, cache.attention_mass).cpu().numpy() for s in ids}
            kept = evict(cache, ids, budget, recent=recent, sinks=sinks).cpu().numpy()
            evictions += 1
            for (s, layer, h), at in stands.items():
                row = select_kept(mass[s][:, layer, h], budget, recent, sinks)
                assert np.array_equal(kept[s, layer, h], row)
                stands[s, layer, h] = [at[t] for t in row]
                assert np.array_equal(tokens(cache, s, cache.attention_mass).cpu().numpy()[:, layer, h],
                                      mass[s][row, layer, h])
            assert [cache.sequence_length(s) for s in ids] == [budget] * B
            cache.validate_invariants()
            assert free_mass(cache) == 0.0
            assert cache.changes_since(0, limit) == 0  # nothing a reader saw is still in place
    assert evictions >= 3 and cache.status_bits() == 0
    assert {stands[0, 0, 0][0], stands[1, 1, 1][1]} == {0, 1}  # the sinks


def test_evict_leaves_short_sequences(device):
    import torch

    from specdecode_b200.eviction import evict

    cache = filled(device, [30, 100, 31], 1, 1, 32, 16)
    cache.attention_mass.uniform_()
    before = [tokens(cache, s, cache.key_codes) for s in range(3)]
    kept = evict(cache, [0, 1, 2], 31, recent=5)
    assert [cache.sequence_length(s) for s in range(3)] == [30, 31, 31]
    assert torch.equal(tokens(cache, 0, cache.key_codes), before[0])
    assert torch.equal(tokens(cache, 2, cache.key_codes), before[2])
    assert torch.equal(tokens(cache, 1, cache.key_codes)[:, 0, 0], before[1][kept[1, 0, 0].long(), 0, 0])
    assert kept[0, 0, 0].tolist() == list(range(30)) + [-1]
    cache.validate_invariants()


def test_session_observes_every_layer(device):
    """The transformers hook with observe_attention: every layer's mass grows
    by one unit per query row, also in prefill windows and captured steps."""
    import torch
    from transformers import LlamaConfig, LlamaForCausalLM

    from specdecode_b200.hf_attention import PagedAttentionSession

    torch.manual_seed(0)
    config = LlamaConfig(hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
                         num_key_value_heads=1, head_dim=64, vocab_size=100, max_position_embeddings=256)
    model = LlamaForCausalLM(config).to(device=device, dtype=torch.bfloat16).eval()
    cache = make_cache(device, 2, 1, 64, 16, 32, max_sequences=2)
    cache.track_attention()
    session = PagedAttentionSession(cache)
    session.observe_attention = True
    model.set_attn_implementation(PagedAttentionSession.NAME)
    for s in range(2):
        cache.create_sequence(s)
    ids = torch.randint(0, 100, (2, 45), device=device)
    with torch.no_grad():
        for start, stop in ((0, 40), (40, 45)):
            with session.step([0, 1], stop - start):
                model(ids[:, start:stop], position_ids=torch.arange(start, stop, device=device).expand(2, -1),
                      use_cache=False)
        # single-token steps through the session's fixed addresses: eager, captured, replayed
        session.check_each_step = False
        session.reserve_fixed_workspace(session.attention.workspace_bytes(2, 4, 1, 64))
        token = torch.zeros((2, 1), dtype=torch.long, device=device)
        position = torch.zeros((2, 1), dtype=torch.long, device=device)
        slots = torch.zeros(2, dtype=torch.int64, device=device)
        graph = None
        for step in range(4):
            with session.fixed_step([0, 1], 1, slots, 64):
                position.fill_(45 + step)
                if step == 0:
                    model(token, position_ids=position, use_cache=False)
                    continue
                if graph is None:
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        model(token, position_ids=position, use_cache=False)
                graph.replay()
    cache.check_status()
    total = cache.attention_mass.double().sum(dim=(0, 2, 3)).cpu().numpy()
    # 2 sequences x (45 + 4) positions x 4 query heads, each row summing to one within its roundings
    assert np.abs(total - 392).max() <= 392 * 1e-4
    assert free_mass(cache) == 0.0


def test_refusals(device):
    import torch

    from specdecode_b200.device_pages import DevicePagedCache
    from specdecode_b200.eviction import compact_tokens, evict, observe_attention, select_tokens

    cache = filled(device, [20, 30], 1, 2, 64, 16)
    bare = filled(device, [20], 1, 2, 64, 16, track=False)
    q = torch.randn((2, 4, 1, 64), device=device)
    kept = torch.zeros((2, 1, 2, 5), dtype=torch.int32, device=device)
    for error, call in [
            (ValueError, lambda: observe_attention(bare, q[:1], [0], 0)),
            (ValueError, lambda: select_tokens(bare, [0], 4)),
            (TypeError, lambda: select_tokens(DevicePagedCache(cache.config, max_rows=1, device=device), [0], 4)),
            (ValueError, lambda: observe_attention(cache, q, [0, 0], 0)),
            (ValueError, lambda: observe_attention(cache, q, [], 0)),
            (KeyError, lambda: observe_attention(cache, q, [0, 5], 0)),
            (ValueError, lambda: observe_attention(cache, q[:1], [0, 1], 0)),
            (ValueError, lambda: observe_attention(cache, q[..., :32], [0, 1], 0)),
            (ValueError, lambda: observe_attention(cache, q.cpu(), [0, 1], 0)),
            (TypeError, lambda: observe_attention(cache, q.double(), [0, 1], 0)),
            (ValueError, lambda: observe_attention(cache, q, [0, 1], 1)),
            (ValueError, lambda: observe_attention(cache, q.expand(2, 4, 21, 64), [0, 1], 0)),
            (ValueError, lambda: select_tokens(cache, [0, 1], 0)),
            (ValueError, lambda: select_tokens(cache, [0, 1], 8, recent=6, sinks=3)),
            (ValueError, lambda: evict(cache, [1, 1], 8)),
            (TypeError, lambda: compact_tokens(cache, [0, 1], kept.long())),
            (ValueError, lambda: compact_tokens(cache, [0, 1], kept[:1])),
            (ValueError, lambda: compact_tokens(cache, [0, 1], kept.cpu())),
            (ValueError, lambda: compact_tokens(cache, [0, 0], kept)),
    ]:
        with pytest.raises(error):
            call()
    with pytest.raises(Exception, match="unsupported"):
        observe_attention(cache, torch.randn((2, 130, 1, 64), device=device), [0, 1], 0)
    assert cache.status_bits() == 0 and not bool(cache.attention_mass.any())
