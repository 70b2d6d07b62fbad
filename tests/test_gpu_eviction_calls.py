"""Calls around an eviction: checkpoints taken before one, and a captured
decoding pass whose observation is switched on and off."""

from __future__ import annotations

import pytest

from gpu_helpers import make_cache

pytestmark = pytest.mark.gpu


def filled(device, lengths, L=1, H=2, D=64):
    import torch

    blocks = sum(-(-n // 16) for n in lengths) + 8
    cache = make_cache(device, L, H, D, 16, blocks, max_sequences=len(lengths), max_blocks_per_sequence=blocks)
    cache.track_attention().uniform_()
    for s, n in enumerate(lengths):
        cache.create_sequence(s)
        k, v = torch.randn((2, n, L, H, D), device=device)
        cache.append_tensor(s, k, v)
    return cache


def test_a_checkpoint_from_before_an_eviction_is_refused(device):
    import torch

    from specdecode_b200.eviction import compact_tokens, evict
    from specdecode_b200.kv_cache import KVCacheError

    cache = filled(device, [100, 20, 60])
    early = [cache.checkpoint(s) for s in range(3)]
    cache.truncate(0, 90)
    evict(cache, [0, 1], 50)
    codes = cache.key_codes.clone()
    with pytest.raises(KVCacheError, match="rewritten"):  # past the trimmed length
        cache.rollback(0, early[0])
    k, v = torch.randn((2, 70, 1, 2, 64), device=device)
    cache.append_tensor(0, k, v)  # 120 tokens: the checkpoint's count lies inside again
    with pytest.raises(KVCacheError, match="rewritten"):
        cache.rollback(0, early[0])
    assert cache.sequence_length(0) == 120
    # within its budget, sequence 1 was left as it was; sequence 2 was not listed
    cache.rollback(1, early[1])
    cache.rollback(2, early[2])
    # one taken since holds
    late = cache.checkpoint(0)
    cache.append_tensor(0, k[:5], v[:5])
    cache.rollback(0, late)
    assert cache.sequence_length(0) == 120
    # compaction alone rewrites too, and the next eviction ends the later checkpoint
    kept = torch.arange(1, 31, dtype=torch.int32, device=device).expand(1, 1, 2, 30)
    compact_tokens(cache, [2], kept)
    with pytest.raises(KVCacheError, match="rewritten"):
        cache.rollback(2, early[2])
    evict(cache, [0], 60)
    with pytest.raises(KVCacheError, match="rewritten"):
        cache.rollback(0, late)
    # a refused rollback changes nothing, and a truncation by count still works
    assert cache.sequence_length(2) == 60 and cache.sequence_length(0) == 60
    assert torch.equal(cache.key_codes[cache.block_table(1)[0]], codes[cache.block_table(1)[0]])
    cache.truncate(0, 10)
    cache.validate_invariants()
    # a sequence that is gone is unknown, whatever the checkpoint; one of the same name starts over
    gone = cache.checkpoint(0)
    cache.remove_sequence(0)
    with pytest.raises(KeyError):
        cache.rollback(0, gone)
    cache.create_sequence(0)
    cache.append_tensor(0, k[:9], v[:9])
    fresh = cache.checkpoint(0)
    cache.append_tensor(0, k[:9], v[:9])
    cache.rollback(0, fresh)
    assert cache.sequence_length(0) == 9
    # no checkpoint of its predecessor fits it, however often it is trimmed
    for budget in (8, 7, 6):
        evict(cache, [0], budget)
        cache.append_tensor(0, k[:9], v[:9])
        with pytest.raises(KVCacheError, match="rewritten"):
            cache.rollback(0, gone)


def test_rows_of_rolled_back_tokens(device):
    """Every observed row counts, also one whose token is rolled back afterwards;
    observing after the rollback counts the accepted rows alone."""
    import torch

    from specdecode_b200.eviction import observe_attention
    from test_gpu_observe_launch import check, fill, keys_of, of_sequence

    lengths, accepted, window, H = [41, 70, 38], [3, 1, 3], 5, 2
    cache = fill(device, lengths, H, 64)
    q = (torch.randn((3, 4, window, 64), device=device) * 2).to(torch.bfloat16)
    observe_attention(cache, q, [0, 1, 2], 0)
    every = [[of_sequence(cache, s, cache.attention_mass, h).clone() for h in range(H)] for s in range(3)]
    left = [n - window + a for n, a in zip(lengths, accepted)]
    cache.truncate_batch([0, 1, 2], left)
    for s in range(3):
        for h in range(H):  # the tokens before keep what the rejected rows gave them
            assert torch.equal(of_sequence(cache, s, cache.attention_mass, h), every[s][h][:left[s]])
    cache.attention_mass.zero_()
    for count in sorted(set(accepted)):  # one call per number of accepted rows
        ids = [s for s in range(3) if accepted[s] == count]
        observe_attention(cache, q[ids][:, :, :count], ids, 0)
    assert cache.status_bits() == 0
    for s in range(3):
        for h in range(H):
            check(q[s, 2 * h:2 * h + 2, :accepted[s]].double(), keys_of(cache, s, h),
                  of_sequence(cache, s, cache.attention_mass, h), accepted[s], 2 * H, max(left), False)
            assert bool((every[s][h][:left[s]] > of_sequence(cache, s, cache.attention_mass, h)).any())
