"""Per-head normalisation, position rotation and append in one launch.

A model's attention layer normalises its query and key heads (where the model
has query / key norms), rotates them to their positions, and appends keys and
values to the cache.  The reference leaves the first two to the model and
quantizes what arrives (src/specdecode/hf_paged_cache.py:199-232);
``norm_rotate_append`` takes the projections themselves: queries come back in
the layout the paged attention reads, keys and values go straight into their
INT8 pages, the rotated key quantized without a 16-bit intermediate.

Positions are arguments, not cache lengths, because the two part once tokens
have been evicted (``eviction``): a sequence of 9000 tokens trimmed to 4096
appends its next token at slot 4096 and position 9000.

Usage::

    table = RotaryTable(128, 131072, base=500000.0, device=cache.device)
    pending = cache.reserve(ids, n)                       # slots for every layer
    for layer in range(layers):
        q, k, v = project(layer, hidden)                  # [B, n, heads, head_dim] views
        query = norm_rotate_append(cache, pending, layer, q, k, v, positions, table,
                                   query_weight=wq[layer], key_weight=wk[layer])
        out = attention(query, tables, lens, max_len, layer)
"""

from __future__ import annotations

from . import _lib
from .kv_cache import LayerwiseAppend, _dtype_code, launch

__all__ = ["RotaryTable", "norm_rotate_append"]


class RotaryTable:
    """Cosines and sines of ``position * frequency`` for the leading
    ``rotary_dim`` elements of a head, float32 ``[max_positions, rotary_dim /
    2, 2]`` on the device, computed in float64 (the angle of a far position
    has no correct digits left in float32).

    ``inv_freq`` gives the ``rotary_dim / 2`` frequencies of a scaled rotary
    embedding; by default they are ``base ** (-2 i / rotary_dim)``.  Both
    functions are multiplied by ``scaling`` (the attention factor some
    scaled embeddings carry).  ``interleaved`` pairs elements ``(2 i, 2 i +
    1)`` instead of ``(i, i + rotary_dim / 2)``."""

    def __init__(self, rotary_dim: int, max_positions: int, *, base: float = 10000.0, inv_freq=None,
                 scaling: float = 1.0, interleaved: bool = False, device=None) -> None:
        import torch

        if rotary_dim < 2 or rotary_dim % 2:
            raise ValueError("rotary_dim must be a positive even number")
        if max_positions < 1:
            raise ValueError("max_positions must be positive")
        device = torch.device(device if device is not None else "cuda")
        if inv_freq is None:
            inv_freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
        else:
            inv_freq = torch.as_tensor(inv_freq).to(device=device, dtype=torch.float64)
            if tuple(inv_freq.shape) != (rotary_dim // 2,):
                raise ValueError("inv_freq must hold rotary_dim / 2 frequencies")
        self.rotary_dim = int(rotary_dim)
        self.max_positions = int(max_positions)
        self.interleaved = bool(interleaved)
        self.values = torch.empty((max_positions, rotary_dim // 2, 2), dtype=torch.float32, device=device)
        rows = max(1, (1 << 24) // rotary_dim)  # float64 intermediates of at most 64 MB
        for start in range(0, max_positions, rows):
            stop = min(max_positions, start + rows)
            angles = torch.arange(start, stop, dtype=torch.float64, device=device)[:, None] * inv_freq
            self.values[start:stop, :, 0] = torch.cos(angles) * scaling
            self.values[start:stop, :, 1] = torch.sin(angles) * scaling

    @property
    def device(self):
        return self.values.device


def _heads(t, name: str, shape, dtype, device):
    """Projection heads ``shape`` with unit element stride, 16-byte aligned
    and strided (a view into a packed projection serves; others are copied)."""
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {list(shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must have the query's dtype {dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on the cache's device")
    s0, s1, s2, s3 = t.stride()
    if s3 != 1 or (t.data_ptr() | ((s0 | s1 | s2) * t.element_size())) & 15:
        # (contiguous() would keep the strides of dimensions of one element)
        import torch

        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _weight(w, name: str, head_dim: int, device):
    if w is None:
        return None
    if tuple(w.shape) != (head_dim,):
        raise ValueError(f"{name} must hold head_dim weights")
    if w.device != device:
        raise ValueError(f"{name} must be on the cache's device")
    if not w.is_contiguous() or w.data_ptr() % 16:
        w = w.clone()
    return w


def norm_rotate_append(cache, pending, layer: int, query, key, value, positions, table: RotaryTable, *,
                       query_weight=None, key_weight=None, eps: float = 1e-6, out=None):
    """Normalise and rotate ``query`` ``[B, n, query_heads, head_dim]`` and
    ``key`` ``[B, n, heads, head_dim]``, append ``key`` and ``value`` (the
    key's shape) to ``layer`` of ``cache`` and return the queries ``[B,
    query_heads, n, head_dim]`` (``out`` when given, which must not overlap the
    inputs), all in the query's dtype
    (float32, bfloat16 or float16; views into one packed projection are read
    in place).

    ``cache`` is a ``PagedKVCache`` with ``pending`` its reservation of n
    tokens for B sequences (``cache.reserve``), or a ``DevicePagedCache``
    with ``pending`` the slots its ``reserve`` returned: distinct slots, the
    first sequence's tokens first.  ``positions`` is int64 ``[B, n]`` (or
    ``[n]`` for every sequence).  Heads with a weight (``head_dim`` values)
    are normalised: ``x * weight / sqrt(mean(x**2) + eps)``; the arithmetic is
    float32 and rounds once.

    Launches on the current stream of the cache's device.  A position outside
    the table, a slot outside the pool and a non-finite key or value are bits
    of the cache's device status word; such a token's key or value is not
    written (a position fault also zeroes its queries)."""
    import torch

    config, device = cache.config, cache.key_codes.device
    H, D = config.num_heads, config.head_dim
    if query.dim() != 4:
        raise ValueError("query must use [batch, tokens, heads, head_dim] layout")
    B, n, Hq, _ = query.shape
    if Hq < 1 or Hq % H:
        raise ValueError("query heads must be a multiple of the cache's heads")
    if not 0 <= int(layer) < config.num_layers:
        raise ValueError(f"layer {layer} outside the cache's {config.num_layers} layers")
    if query.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("query dtype must be bfloat16, float16 or float32")
    q = _heads(query, "query", (B, n, Hq, D), query.dtype, device)
    k = _heads(key, "key", (B, n, H, D), query.dtype, device)
    v = _heads(value, "value", (B, n, H, D), query.dtype, device)
    slots = pending.slots if isinstance(pending, LayerwiseAppend) else pending
    if not isinstance(slots, torch.Tensor) or slots.dtype != torch.int64 or slots.dim() != 1:
        raise TypeError("pending must be a reservation or a 1-D int64 slot tensor")
    if slots.device != device:
        raise ValueError("the slots must be on the cache's device")
    count = pending.tokens if isinstance(pending, LayerwiseAppend) else int(slots.numel())
    if count != B * n:
        raise ValueError(f"the reservation holds {count} tokens, the projections {B * n}")
    slots = slots.contiguous()
    if positions.dtype != torch.int64:
        if positions.is_floating_point() or positions.dtype == torch.bool:
            raise TypeError("positions must be integers")
        positions = positions.long()
    if positions.device != device:
        raise ValueError("positions must be on the cache's device")
    if positions.dim() == 1:
        positions = positions.expand(B, -1)
    if positions.shape != (B, n):
        raise ValueError("positions must be [batch, tokens] or [tokens]")
    p0, p1 = positions.stride()
    if (n > 1 and p1 != 1) or (B > 1 and p0 < n):
        positions, p0 = positions.contiguous(), n
    if not isinstance(table, RotaryTable):
        raise TypeError("table must be a RotaryTable")
    if table.values.device != device:
        raise ValueError("the rotary table must be on the cache's device")
    if table.rotary_dim > D:
        raise ValueError(f"rotary_dim {table.rotary_dim} exceeds head_dim {D}")
    wq = _weight(query_weight, "query_weight", D, device)
    wk = _weight(key_weight, "key_weight", D, device)
    if wq is not None and wk is not None and wq.dtype != wk.dtype:
        wq, wk = wq.float(), wk.float()
    weight = wq if wq is not None else wk
    if weight is not None:
        if weight.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError("norm weights must be bfloat16, float16 or float32")
        if not 0.0 < float(eps) < float("inf"):
            raise ValueError("eps must be positive and finite")
    shape = (B, Hq, n, D)
    if out is None:
        out = query.new_empty(shape)
    elif out.shape != shape or out.dtype != query.dtype or out.device != device or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise ValueError(f"out must be a contiguous, 16-byte aligned {query.dtype} tensor of shape {list(shape)} on "
                         f"{device}")
    if B * n == 0:
        return out
    q0, q1, q2, _ = q.stride()
    k0, k1, k2, _ = k.stride()
    v0, v1, v2, _ = v.stride()
    batch = _lib.RotateBatch(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _dtype_code(query.dtype), B, n, Hq, q0, q1, q2, k0, k1, k2,
        v0, v1, v2, positions.data_ptr(), p0 if B > 1 else n, table.values.data_ptr(), table.max_positions,
        table.rotary_dim, table.interleaved, wq.data_ptr() if wq is not None else None,
        wk.data_ptr() if wk is not None else None, _dtype_code(weight.dtype) if weight is not None else 0, eps)
    library = cache.library
    library.check(launch(device, lambda stream: library.handle.sdc_norm_rotate_append(
        cache.pool_desc, int(layer), batch, slots.data_ptr(), out.data_ptr(), cache._status.data_ptr(), stream)),
        "rotated append")
    return out
