"""The attention observation's launch forms: every number of rows and tiles that
one block takes, each kernel meeting its sizes in a fresh process, and both
forms against float64 within a bound taken from the split of the call.

Tolerance.  u = 2^-24.  A score errs by at most E = (2 D + 3) u A (+ 2^-22 B for
float32 queries), with A and B the sums below: D products, exact, each addition
off by at most 2 u of the partial sums, and three scaling products; a float32
query keeps 22 bits of its row's largest element.  A weight is exp2(s - M) / S.
The difference rounds once, an error of 2 u A in the exponent; exp2 errs by 2
ulp = 4 u.  A term of S passes, with t the tiles of a warp, at most t rises of the
warp's running maximum, the joining of its lanes, four of the block's warps and,
in two launches, the merging of the chunks (chunks / parts one after the
other in each of the `parts` threads of a row, then the parts): R rescalings, each
a difference, an exp2, a product and a sum, 6 u and 2 u A in the exponent;
and 3 t + 3 additions of its own.  The numerator has an exp2, a difference, the
reciprocal and the product, 6 u together; the rows' sum NT + 3 additions, NT the
eights of rows.  E enters the numerator and S.  Together
    exp(2 E + (2 R + 4) u A + (6 R + 3 t + NT + 16) u) - 1
of the weight; the mass is zero before, so its addition is exact.  Weights below
2^-126 may flush to zero."""

from __future__ import annotations

import math
import subprocess
import sys
from pathlib import Path

import pytest

if __name__ == "__main__":  # run by the test below
    sys.path[:0] = [str(Path(__file__).resolve().parent), str(Path(__file__).resolve().parents[1]),
                    str(Path(__file__).resolve().parents[1] / "llm-inference-accelerator_b200")]

from gpu_helpers import make_cache

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SMS, WARPS = 148, 4


def eights(rows):
    n = -(-rows // 8)
    return n if n <= 4 else 8


def rescalings(pairs, max_len, rows):
    """(t, R) of a call over `pairs` (sequence, KV head) pairs, of whichever
    of the two forms has more."""
    tiles = -(-max_len // 32)
    fill = -(-pairs * tiles // (SMS * 4 * WARPS))
    warp_tiles = min(8, max(fill, -(-tiles // (128 * WARPS))))
    chunks = -(-tiles // (WARPS * warp_tiles))
    t = -(-(-(-tiles // chunks)) // WARPS)
    chunks = -(-tiles // (t * WARPS))
    if tiles <= 16 * WARPS:  # one block may take all
        t = max(t, -(-tiles // WARPS))
    parts = 128 // (8 * eights(rows))
    return t, t + 1 + WARPS + -(-chunks // parts) + parts


def check(query, keys, mass, window, pairs, max_len, split):
    """query [rows / window, window, D] and keys [T, D] of one KV head, float64;
    mass [T] float32, zero before the call."""
    import torch

    D, T = keys.shape[1], keys.shape[0]
    rows = query.shape[0] * window
    s = torch.einsum("gwd,td->gwt", query, keys) / math.sqrt(D)
    hidden = torch.arange(T, device=s.device)[None] > torch.arange(T - window, T, device=s.device)[:, None]
    p = torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1)
    want = p.sum(dim=(0, 1))
    A = float(torch.einsum("gwd,td->gwt", query.abs(), keys.abs()).max()) / math.sqrt(D)
    B = float(query.abs().amax() * keys.abs().sum(dim=1).max()) / math.sqrt(D)
    t, R = rescalings(pairs, max_len, rows)
    E = (2 * D + 3) * U * A + (2.0 ** -22 * B if split else 0.0)
    rel = math.expm1(2 * E + (2 * R + 4) * U * A + (6 * R + 3 * t + eights(rows) + 16) * U)
    excess = (mass.double() - want).abs() - (rel * want + rows * 2.0 ** -126)
    assert float(excess.max()) <= 0.0, (float(excess.max()), rel)


def fill(device, lengths, H, D, seed=0):
    import torch

    blocks = sum(-(-n // 16) for n in lengths) + 1
    cache = make_cache(device, 1, H, D, 16, blocks, max_sequences=len(lengths),
                       max_blocks_per_sequence=max(-(-n // 16) for n in lengths))
    cache.track_attention()
    g = torch.Generator(device=device).manual_seed(seed)
    cache.key_codes.copy_(torch.randint(-127, 128, cache.key_codes.shape, generator=g, device=device))
    cache.key_scale_pages.copy_(torch.rand(cache.key_scale_pages.shape, generator=g, device=device) * 0.045 + 0.005)
    for s, n in enumerate(lengths):
        cache.create_sequence(s)
        cache.reserve([s], n)
    return cache


def of_sequence(cache, sequence, pages, head):
    import torch

    slots = torch.from_numpy(cache.page_table.slots_of(sequence, 0, cache.sequence_length(sequence))).to(pages.device)
    return pages[slots // 16, 0, head, slots % 16]


def keys_of(cache, sequence, head):
    return of_sequence(cache, sequence, cache.key_codes, head).double() * \
        of_sequence(cache, sequence, cache.key_scale_pages, head).double()[:, None]


def every_short_size():
    """Every number of rows and of tiles of one context that one block takes (and
    some that it does not), the smallest shared memory first within each
    kernel: no call raises the limit for a smaller one after it."""
    import torch

    from specdecode_b200.eviction import observe_rows

    device = torch.device("cuda", 0)
    for D in (64, 128):
        longest = 32 * 18
        cache = fill(device, [longest], 1, D)
        keys = keys_of(cache, 0, 0)
        tables, _, _ = cache.attention_inputs([0])
        for types in ((torch.bfloat16, torch.float16), (torch.float32,)):
            for n in (1, 2, 3):
                sizes = [(tiles * (64 * (n - 1) + 16 * -(-(rows - 8 * (n - 1)) // 2)), tiles, rows)
                         for rows in range(8 * n - 7, 8 * n + 1) for tiles in range(1, 19)]
                for _, tiles, rows in sorted(sizes):
                    T = 32 * tiles - (rows + tiles) % 32
                    lens = torch.full((1,), T, dtype=torch.int32, device=device)
                    for dtype in types:
                        q = (torch.randn((1, rows, 1, D), device=device) * 2).to(dtype)
                        cache.attention_mass.zero_()
                        observe_rows(cache, q, tables, lens, T, 0)
                        check(q[0].double(), keys[:T], of_sequence(cache, 0, cache.attention_mass, 0)[:T], 1, 1, T,
                              dtype == torch.float32)
        assert cache.status_bits() == 0
    print("every size")


def test_every_short_size_in_a_fresh_process(device):
    done = subprocess.run([sys.executable, str(Path(__file__).resolve())], capture_output=True, text=True, timeout=600)
    assert done.returncode == 0 and "every size" in done.stdout, done.stdout[-2000:] + done.stderr[-4000:]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("lengths, Hq, H, D, window", [
    ([700, 33], 8, 2, 64, 5),        # one launch or two
    ([1900], 1, 1, 128, 1),
    ([9000, 1200, 70], 12, 4, 128, 3),
    ([30011], 64, 1, 64, 1),         # 64 rows
    ([70001], 4, 1, 16, 1),          # chunks of five tiles a warp
    ([200003, 90000], 2, 1, 64, 3),  # more than 128 chunks
    ([8200], 5, 1, 32, 6),
    ([2500] * 40, 24, 8, 256, 2),
])
def test_within_the_bound_of_the_split(device, dtype, lengths, Hq, H, D, window):
    import torch

    from specdecode_b200.eviction import observe_attention

    cache = fill(device, lengths, H, D)
    kind = getattr(torch, dtype)
    q = (torch.randn((len(lengths), Hq, window, D), device=device) * 2).to(kind)
    observe_attention(cache, q, list(range(len(lengths))), 0)
    assert cache.status_bits() == 0
    group = Hq // H
    for s in range(len(lengths)):
        for h in range(H):
            check(q[s, h * group:(h + 1) * group].double(), keys_of(cache, s, h),
                  of_sequence(cache, s, cache.attention_mass, h), window, len(lengths) * H, max(lengths),
                  kind == torch.float32)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("D", [16, 32])
def test_every_number_of_rows_of_narrow_heads(device, D, dtype):
    """Rows of 16 elements share a warp with fifteen others, the last of which
    are not there for an odd number of eights."""
    import torch

    from specdecode_b200.eviction import observe_attention

    T, kind = 97, getattr(torch, dtype)
    cache = fill(device, [T], 1, D)
    keys = keys_of(cache, 0, 0)
    for rows in [*range(1, 34), 47, 63, 64]:
        # largest elements far apart from row to row: each row has its own scale
        q = torch.randn((1, rows, 1, D), device=device)
        q = (q * 2.0 ** (torch.arange(rows, device=device) % 7 - 5)[None, :, None, None]).to(kind)
        cache.attention_mass.zero_()
        observe_attention(cache, q, [0], 0)
        check(q[0].double(), keys, of_sequence(cache, 0, cache.attention_mass, 0), 1, 1, T, kind == torch.float32)
    assert cache.status_bits() == 0


if __name__ == "__main__":
    every_short_size()
