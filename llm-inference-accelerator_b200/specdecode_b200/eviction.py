"""Eviction from the paged cache by accumulated attention weight.

The reference's pool only grows and is cut at the tail
(src/specdecode/kv_cache.py:395-420); a context that outgrows its pages ends.
Here a sequence can be trimmed to a token budget and go on: every cached token
carries the softmax weight its key has received so far (its *mass*, one float32
per layer and KV head in pages beside the scales), and ``evict`` keeps, per
layer and head, the first tokens, the latest ones and the heaviest of the rest.

* ``observe_attention``: adds the weights one layer's queries give to the
  cached tokens -- the attention of ``paged_verify_attention`` seen from its
  keys; a ``PagedAttentionSession`` does it in its forward pass when its
  ``observe_attention`` is set;
* ``select_tokens``: the token indices a budget keeps;
* ``compact_tokens``: moves the kept tokens to the front of their pages;
* ``evict``: both, then the cache's ordinary rollback of the tail.

Every observed row counts, also one whose token is rolled back afterwards: the
rollback clears the discarded tokens' own mass, not what their queries gave to
the tokens before them.  A caller who verifies proposals and wants the accepted
rows alone observes after the rollback, when they are the sequence's last
positions: one call for the sequences with the same number of accepted rows,
with the queries of those rows.  A session observes in its forward pass, before
acceptance is known.

Every head keeps the same number of tokens, in order, but not the same ones:
after an eviction a cached index no longer names one token of the text, and a
sequence's length no longer is its next position.  Rotate new tokens by their
true positions (``rotary.norm_rotate_append``, or a model's ``position_ids``);
a checkpoint taken before an eviction is refused by the cache's ``rollback``, and
``BatchedSpeculativeDecoder``, which takes positions from cache lengths, does not
run over a trimmed cache.  ``PagedKVCache`` only: blocks that
``DevicePagedCache.fork`` shares cannot be moved.  Like the cache itself these
functions are not thread-safe; calls on one sequence belong on one stream.
"""

from __future__ import annotations

import ctypes
from collections.abc import Hashable, Sequence

from .kv_cache import PagedKVCache, _dtype_code, _torch, launch

__all__ = ["compact_tokens", "evict", "observe_attention", "select_tokens"]

# the most an observation takes for its scores; larger calls run in rounds
WORKSPACE_BYTES = 256 << 20


def _listed(cache, sequence_ids: Sequence[Hashable]):
    """(table rows, host lengths) of distinct sequences."""
    if not isinstance(cache, PagedKVCache):
        raise TypeError("cache must be a PagedKVCache")
    pages = cache.page_table
    known = pages.rows
    rows = [known[s] if s in known else pages.require(s) for s in sequence_ids]  # require raises
    if not rows:
        raise ValueError("at least one sequence is required")
    if len(set(rows)) != len(rows):
        raise ValueError("a sequence appears twice in one call")
    return rows, pages.lengths[rows].tolist()


def _inputs(cache, rows):
    """(table pointer, table stride, length pointer, what keeps them alive):
    the cache's own rows where they are consecutive, else a gathered copy."""
    tables, lens = cache.block_tables, cache.context_lens
    first, count, stride = rows[0], len(rows), tables.shape[1]
    if rows == list(range(first, first + count)):
        return tables.data_ptr() + first * stride * 4, stride, lens.data_ptr() + first * 4, None
    import torch

    index = torch.tensor(rows, dtype=torch.long, device=tables.device)
    tables, lens = tables.index_select(0, index), lens.index_select(0, index)
    return tables.data_ptr(), stride, lens.data_ptr(), (tables, lens)


def _tracked(cache):
    if cache.attention_mass is None:
        raise ValueError("the cache does not track attention (call its track_attention first)")
    return cache.attention_mass


def _budget(budget, recent, sinks) -> tuple[int, int, int]:
    values = []
    for name, value, least in (("budget", budget, 1), ("recent", recent, 0), ("sinks", sinks, 0)):
        if isinstance(value, bool) or not isinstance(value, int) or value < least:
            raise ValueError(f"{name} must be an integer of at least {least}")
        values.append(value)
    if recent + sinks > budget:
        raise ValueError("recent and sinks together exceed the budget")
    return tuple(values)


def observe_attention(cache: PagedKVCache, query, sequence_ids: Sequence[Hashable], layer: int):
    """Add the attention of ``query`` ``[B, query_heads, window, head_dim]``
    (bfloat16, float16 or float32) to the mass of the cached tokens.

    The window holds each sequence's last ``window`` cached positions, as in
    ``paged_verify_attention``: row i sees the tokens up to position ``length -
    window + i``, scores scaled by ``1 / sqrt(head_dim)``, and every visible
    token's mass of KV head h grows by the weights of that head's query rows
    (which stay when the window's tokens are rolled back).
    Query heads per KV head times window must not exceed 64; head_dim is 16,
    32, 64, 128 or 256.  Returns the mass pages.  A query row whose weights
    are not finite adds nothing and sets a bit of the cache's status word."""
    import torch

    rows, lengths = _listed(cache, sequence_ids)
    mass = _tracked(cache)
    shape = query.shape
    if len(shape) != 4 or shape[0] != len(rows) or shape[3] != cache.config.head_dim:
        raise ValueError("query must be [sequences, query_heads, window, head_dim]")
    if query.device != mass.device:
        raise ValueError("query must be on the cache's device")
    if query.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError("query dtype must be bfloat16, float16 or float32")
    if isinstance(layer, bool) or not 0 <= int(layer) < cache.config.num_layers:
        raise ValueError(f"layer {layer} outside the cache's {cache.config.num_layers} layers")
    if not 1 <= shape[2] <= min(lengths):
        raise ValueError("the window must hold between one token and the shortest sequence's length")
    _observe(cache, query, _inputs(cache, rows), max(lengths), int(layer))
    return mass


def observe_rows(cache: PagedKVCache, query, tables, lens, max_len: int, layer: int) -> None:
    """``observe_attention`` over the caller's device tables and lengths
    (``PagedKVCache.attention_inputs``), whose rows must not share blocks.  Its
    launches and workspace follow ``max_len``: a bound far above the lengths
    costs (64 contexts of 1000 tokens, 32 query heads of 64: 15 us under 1200, 199
    under 131072)."""
    _tracked(cache)
    if tables.stride(1) != 1:
        tables = tables.contiguous()
    _observe(cache, query, (tables.data_ptr(), tables.stride(0), lens.data_ptr(), (tables, lens)), int(max_len), layer)


def _observe(cache, query, inputs, max_len: int, layer: int) -> None:
    mass = cache.attention_mass
    tables, stride, lens, _ = inputs
    if not query.is_contiguous():
        query = query.contiguous()
    if query.data_ptr() % 16:
        query = query.clone()
    B, Hq, window, D = query.shape
    library = cache.library
    least, most = ctypes.c_size_t(), ctypes.c_size_t()
    library.check(library.handle.sdc_observe_workspace_size(
        B, Hq, cache.config.num_heads, D, window, max_len, least, most), "attention observation")
    size, workspace = 0, None
    if most.value:
        # a tensor of this call: freed behind its launches, and a captured graph's own
        size = max(least.value, min(most.value, WORKSPACE_BYTES))
        workspace = mass.new_empty(size, dtype=_torch().uint8)
    library.check(launch(mass.device, lambda stream: library.handle.sdc_observe_attention(
        cache.pool_desc, layer, mass.data_ptr(), query.data_ptr(), _dtype_code(query.dtype), B, Hq, window,
        tables, stride, lens, max_len, workspace.data_ptr() if size else None, size, cache._status.data_ptr(), stream)),
        "attention observation")


def select_tokens(cache: PagedKVCache, sequence_ids: Sequence[Hashable], budget: int, *, recent: int = 0,
                  sinks: int = 0):
    """int32 ``[B, layers, heads, budget]``: the cached indices each head
    keeps, ascending -- the first ``sinks``, the last ``recent``, and of the
    others the heaviest (equal masses: the lower index).  A sequence within
    the budget keeps all its tokens; the rest of its rows is -1."""
    rows, lengths = _listed(cache, sequence_ids)
    return _select(cache, rows, lengths, *_budget(budget, recent, sinks))


def _select(cache, rows, lengths, budget: int, recent: int, sinks: int):
    mass = _tracked(cache)
    c = cache.config
    kept = mass.new_empty((len(rows), c.num_layers, c.num_heads, budget), dtype=_torch().int32)
    tables, stride, lens, _keep = _inputs(cache, rows)
    longest = max(1, *lengths)
    library = cache.library
    library.check(launch(mass.device, lambda stream: library.handle.sdc_select_tokens(
        cache.pool_desc, mass.data_ptr(), len(rows), tables, stride, lens, longest, budget, recent, sinks,
        kept.data_ptr(), cache._status.data_ptr(), stream)), "token selection")
    return kept


def compact_tokens(cache: PagedKVCache, sequence_ids: Sequence[Hashable], kept) -> None:
    """Move token ``kept[b, layer, head, j]`` to index j (codes, scales and
    mass) in every sequence longer than ``kept``'s last dimension; the tokens
    from there on stay as they are until the caller truncates.  Rows must be
    strictly ascending indices of cached tokens; one that is not moves nothing
    and sets a bit of the cache's status word.  Call the cache's
    ``mark_rewritten`` after each replay of a captured compaction."""
    ids = list(sequence_ids)
    rows, lengths = _listed(cache, ids)
    _compact(cache, ids, rows, lengths, kept)


def _compact(cache, ids, rows, lengths, kept) -> None:
    import torch

    c = cache.config
    if not isinstance(kept, torch.Tensor) or kept.dtype != torch.int32:
        raise TypeError("kept must be an int32 tensor")
    shape = kept.shape
    if len(shape) != 4 or shape[:3] != (len(rows), c.num_layers, c.num_heads) or shape[3] < 1:
        raise ValueError("kept must be [sequences, num_layers, num_heads, budget]")
    if kept.device != cache.key_codes.device:
        raise ValueError("kept must be on the cache's device")
    kept = kept.contiguous()
    budget = shape[3]
    tables, stride, lens, _keep = _inputs(cache, rows)
    mass = cache.attention_mass
    library = cache.library
    library.check(launch(kept.device, lambda stream: library.handle.sdc_compact_tokens(
        cache.pool_desc, mass.data_ptr() if mass is not None else None, len(rows), tables, stride, lens,
        kept.data_ptr(), budget, cache._status.data_ptr(), stream)), "token compaction")
    cache.mark_rewritten([s for s, length in zip(ids, lengths) if length > budget])


def evict(cache: PagedKVCache, sequence_ids: Sequence[Hashable], budget: int, *, recent: int = 0, sinks: int = 0):
    """Trim every listed sequence longer than ``budget`` to its ``budget``
    kept tokens (``select_tokens``), releasing the blocks behind them; shorter
    ones are left as they are.  Returns the kept indices."""
    ids = list(sequence_ids)
    rows, lengths = _listed(cache, ids)
    kept = _select(cache, rows, lengths, *_budget(budget, recent, sinks))
    _compact(cache, ids, rows, lengths, kept)
    cache.truncate_batch(ids, [min(n, budget) for n in lengths])
    return kept
