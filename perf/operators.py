"""The paged cache's long-context operators: what each is timed on, its plain
form and its definition in 64 bits.

* ``rotate``: one layer's packed query / key / value projections -> queries and
  keys normalised per head and rotated to their positions, queries in the
  attention's layout, keys and values quantized into their pages.
* ``observe``: the softmax weight that one layer's queries give to every cached
  token, added to the token's running sum in the pages.
* ``select``: the tokens a cache keeps under a budget, per layer and KV head:
  the first ones, the latest ones and those with the largest sums.
* ``compact``: the kept tokens moved, in order, to the front of the pages.

Shapes are those of the speculative pair this repository serves (a 16-layer
draft with head_dim 64, a 32-layer target with head_dim 128, both with 32 query
heads over 8 KV heads), of its 64-query-head long-context configuration, and
of its tests.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# -- cases -------------------------------------------------------------------
def listed():
    return [
        # one new token of one sequence of the draft: launch latency
        _rotate("rotate 1x1 32/8x64 bf16", 1, 1, 32, 8, 64, "bf16", norm=False, style="half", max_positions=16384),
        # a verify window of a full batch on the target
        _rotate("rotate 64x6 32/8x128 bf16 norm", 64, 6, 32, 8, 128, "bf16", norm=True, style="half",
                max_positions=131072),
        # a prefill chunk of a batch, pairs rotated side by side
        _rotate("rotate 16x512 32/8x128 f16 norm", 16, 512, 32, 8, 128, "f16", norm=True, style="interleaved",
                max_positions=131072),
        # one short sequence, one token: launch latency, and an odd length
        _observe("observe 1x131 32/8x64 f32", 1, 131, 131, 32, 8, 64, 1, "f32"),
        # a decode step of a batch on the draft
        _observe("observe 64x1100 32/8x64 bf16", 64, 1000, 1200, 32, 8, 64, 1, "bf16"),
        # a verify window of the target's batch, ragged contexts
        _observe("observe 32x8192 32/8x128 bf16 w5", 32, 1024, 8192, 32, 8, 128, 5, "bf16"),
        # one long context of the 64-query-head configuration
        _observe("observe 1x131071 64/8x128 f16 w3", 1, 131071, 131071, 64, 8, 128, 3, "f16"),
        # one sequence of the draft trimmed to a small budget
        _select("select 1x1021 to 256 16x8", 1, 1021, 1021, 16, 8, 256, 32, 4),
        # a batch of the target trimmed at once, ragged contexts
        _select("select 8x8192 to 2048 32x8", 8, 6000, 8192, 32, 8, 2048, 128, 4),
        # one long context trimmed once
        _select("select 1x131072 to 16384 8x8", 1, 131072, 131072, 8, 8, 16384, 1024, 16),
        # one sequence of the draft
        _compact("compact 1x1021 to 256 16x8x64", 1, 1021, 1021, 16, 8, 64, 256),
        # a batch of the target, eight of its layers
        _compact("compact 8x8192 to 4096 8x8x128", 8, 6000, 8192, 8, 8, 128, 4096),
    ]


def _rotate(name, batch, tokens, query_heads, kv_heads, head_dim, dtype, *, norm, style, max_positions):
    return {"name": name, "op": "rotate", "batch": batch, "tokens": tokens, "query_heads": query_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "norm": norm, "style": style,
            "max_positions": max_positions, "block_size": 16}


def _observe(name, batch, shortest, longest, query_heads, kv_heads, head_dim, window, dtype, block_size=16):
    return {"name": name, "op": "observe", "batch": batch, "shortest": shortest, "longest": longest,
            "query_heads": query_heads, "kv_heads": kv_heads, "head_dim": head_dim, "window": window,
            "dtype": dtype, "block_size": block_size}


def _select(name, batch, shortest, longest, layers, kv_heads, budget, recent, sinks, block_size=16):
    return {"name": name, "op": "select", "batch": batch, "shortest": shortest, "longest": longest,
            "layers": layers, "kv_heads": kv_heads, "budget": budget, "recent": recent, "sinks": sinks,
            "block_size": block_size}


def _compact(name, batch, shortest, longest, layers, kv_heads, head_dim, budget, block_size=16):
    return {"name": name, "op": "compact", "batch": batch, "shortest": shortest, "longest": longest,
            "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim, "budget": budget,
            "block_size": block_size}


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(("rotate", "observe", "select", "compact"))
    heads, head_dim = rng.choice(((8, 64), (8, 128), (4, 128), (2, 64)))
    group = rng.choice((1, 4, 8))
    if op == "rotate":
        batch = log(1, 64)
        case = _rotate("", batch, log(1, 8192 // batch), heads * min(group, 4), heads, head_dim,
                       rng.choice(("bf16", "f16", "f32")) if batch < 32 else rng.choice(("bf16", "f16")),
                       norm=rng.random() < 0.7, style=rng.choice(("half", "interleaved")),
                       max_positions=rng.choice((16384, 131072)))
    elif op == "observe":
        batch = log(1, 48)
        longest = log(16, min(131072, 200000 // batch))
        shortest = max(8, log(max(8, longest // 8), longest))
        case = _observe("", batch, shortest, longest, heads * group, heads, head_dim, rng.randint(1, 6),
                        rng.choice(("bf16", "f16", "f32")), rng.choice((8, 16, 32)))
    elif op == "select":
        batch = log(1, 8)
        longest = log(64, min(131072, 65536 // batch))
        budget = log(16, longest - 1)
        case = _select("", batch, log(max(16, longest // 2), longest), longest, rng.choice((4, 16, 32)), heads, budget,
                       rng.randint(0, budget // 4), rng.randint(0, 4), rng.choice((8, 16, 32)))
    else:
        batch = log(1, 8)
        longest = log(64, 65536 // batch)
        case = _compact("", batch, log(max(16, longest // 2), longest), longest, rng.choice((2, 4, 8)), heads,
                        head_dim, log(16, max(16, longest // 2)), rng.choice((8, 16, 32)))
    del case["name"]
    return case


# -- inputs ------------------------------------------------------------------
def _lengths(case):
    # the batch's lengths are part of the case: outputs keep their shapes
    rng = np.random.default_rng(case["shortest"] * 131 + case["longest"])
    return [int(n) for n in rng.integers(case["shortest"], case["longest"] + 1, size=case["batch"])]


def _tables(case, lengths, seed):
    """A shuffled pool just large enough, and each sequence's blocks in it."""
    bs = case["block_size"]
    counts = [-(-n // bs) for n in lengths]
    order = np.random.default_rng(seed + 1).permutation(sum(counts))
    tables = np.zeros((len(lengths), max(counts)), dtype=np.int64)
    at = 0
    for i, n in enumerate(counts):
        tables[i, :n] = order[at:at + n]
        at += n
    return order, tables


def _cache(case, layers, head_dim, lengths, order):
    """The framework's cache holding these sequences in these blocks."""
    import sys

    if "llm-inference-accelerator_b200" not in sys.path:
        sys.path.insert(0, "llm-inference-accelerator_b200")
    from specdecode_b200.kv_cache import KVCacheConfig, PagedKVCache

    bs = case["block_size"]
    cache = PagedKVCache(KVCacheConfig(layers, case["kv_heads"], head_dim, block_size=bs, num_blocks=len(order)),
                         block_order=order, max_sequences=len(lengths),
                         max_blocks_per_sequence=max(-(-n // bs) for n in lengths), check_status=False)
    for i, n in enumerate(lengths):
        cache.create_sequence(i)
        cache.reserve([i], n)
    return cache


def _pool(case, layers, head_dim, order, cache):
    """Codes and scales of a filled pool, [block, layer, head, offset(, dim)]."""
    shape = (len(order), layers, case["kv_heads"], case["block_size"], head_dim)
    if cache is not None:
        return {"keys": cache.key_codes, "values": cache.value_codes, "key_scales": cache.key_scale_pages,
                "value_scales": cache.value_scale_pages}
    return {"keys": torch.empty(shape, dtype=torch.int8, device="cuda"),
            "values": torch.empty(shape, dtype=torch.int8, device="cuda"),
            "key_scales": torch.empty(shape[:-1], device="cuda"),
            "value_scales": torch.empty(shape[:-1], device="cuda")}


def _fill(pool, gen):
    # codes as quantized Gaussian vectors have them, scales of unit-variance
    # heads with a spread from token to token
    for name in ("keys", "values"):
        codes = pool[name].view(-1)
        step = 1 << 28
        for at in range(0, codes.numel(), step):
            part = codes[at:at + step]
            if part.numel() <= 1 << 26:
                part.copy_((torch.randn(part.shape, generator=gen, device="cuda") * 45).clamp_(-127, 127).round_())
            else:
                part.random_(-127, 128, generator=gen)
        scales = pool[name[:-1] + "_scales"]
        scales.copy_(torch.rand(scales.shape, generator=gen, device="cuda") * 0.02 + 0.012)


def _mass(shape, gen):
    """Running sums as attention leaves them: a heavy tail, a twentieth of the
    tokens never looked at, and repeated values."""
    m = torch.exp(torch.randn(shape, generator=gen, device="cuda") * 2.0 - 3.0)
    r = torch.rand(shape, generator=gen, device="cuda")
    m = torch.where(r < 0.05, torch.zeros_like(m), m)
    return torch.where(r > 0.9, (m * 64).round() / 64, m)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "rotate":
        return _prepare_rotate(case, seed, gen)
    lengths = _lengths(case)
    order, tables = _tables(case, lengths, seed)
    layers = 2 if op == "observe" else case["layers"]
    D = 16 if op == "select" else case["head_dim"]
    cache = _cache(case, layers, D, lengths, order) if own else None
    state = {"case": case, "cache": cache, "ids": list(range(len(lengths))), "op": op,
             "tables": torch.from_numpy(tables).cuda(), "lengths": torch.tensor(lengths, device="cuda"),
             "longest": max(lengths)}
    if op != "select":
        state["pool"] = _pool(case, layers, D, order, cache)
        _fill(state["pool"], gen)
    shape = (len(order), layers, case["kv_heads"], case["block_size"])
    if own:
        state["mass"] = cache.track_attention()
    else:
        state["mass"] = torch.zeros(shape, device="cuda")
    state["mass"].copy_(_mass(shape, gen))
    if op == "observe":
        # a few steps' weights so far: each adds one per query row, spread over the context
        state["mass"] *= 4 * case["query_heads"] // case["kv_heads"] * case["window"] / max(lengths)
        q = torch.randn((case["batch"], case["query_heads"], case["window"], D), generator=gen, device="cuda")
        state["query"] = (q * 1.5).to(DTYPES[case["dtype"]])
        state["layer"] = 1
    if op == "compact":
        state["kept"] = _kept(case, lengths, gen)
    return state


def _kept(case, lengths, gen):
    """Ascending token indices per (sequence, layer, head): the first four, the
    latest eighth and a random choice between them; sequences within the budget keep all."""
    B, L, H, N = case["batch"], case["layers"], case["kv_heads"], case["budget"]
    T = torch.tensor(lengths, device="cuda")[:, None, None, None]
    longest = max(lengths)
    t = torch.arange(longest, device="cuda")
    rank = torch.rand((B, L, H, longest), generator=gen, device="cuda")
    rank = torch.where((t < min(4, N)) | (t >= T - N // 8), 2.0, rank)
    rank = torch.where(t < T, rank, -1.0)
    if longest < N:
        rank = torch.nn.functional.pad(rank, (0, N - longest), value=-1.0)
    kept = rank.argsort(dim=-1, descending=True, stable=True)[..., :N].sort(dim=-1).values
    short = torch.arange(N, device="cuda").expand(B, L, H, N)
    short = torch.where(short < T, short, -1)
    return torch.where(T > N, kept, short).to(torch.int32).contiguous()


def _prepare_rotate(case, seed, gen):
    B, n, Hq, Hk, D = (case[k] for k in ("batch", "tokens", "query_heads", "kv_heads", "head_dim"))
    dtype = DTYPES[case["dtype"]]
    # the projection of one layer: query, key and value heads side by side
    packed = torch.randn((B, n, Hq + 2 * Hk, D), generator=gen, device="cuda")
    packed *= torch.exp(torch.randn(D, generator=gen, device="cuda") * 0.5)
    packed = packed.to(dtype)
    # positions run past the cached length where tokens were evicted before
    rng = np.random.default_rng(seed)
    start = torch.from_numpy(rng.integers(0, case["max_positions"] - n, size=B)).cuda()
    positions = start[:, None] + torch.arange(n, device="cuda")
    weights = [torch.rand(D, generator=gen, device="cuda").add_(0.5).to(dtype) for _ in range(2)]
    base = 500000.0
    inv_freq = base ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    lengths = [n] * B
    order, tables = _tables(case, lengths, seed)
    cache = _cache(case, 2, D, lengths, order) if own else None
    state = {"case": case, "op": "rotate", "query": packed[:, :, :Hq], "key": packed[:, :, Hq:Hq + Hk],
             "value": packed[:, :, Hq + Hk:], "positions": positions, "inv_freq": inv_freq,
             "query_weight": weights[0] if case["norm"] else None, "key_weight": weights[1] if case["norm"] else None,
             "eps": 1e-6, "layer": 1, "cache": cache, "tables": torch.from_numpy(tables).cuda()}
    if own:
        from specdecode_b200.rotary import RotaryTable

        cache.truncate_batch(list(range(B)), [0] * B)
        state["pending"] = cache.reserve(list(range(B)), n)
        state["table"] = RotaryTable(D, case["max_positions"], base=base, interleaved=case["style"] == "interleaved",
                                     device=cache.device)
    else:
        angles = torch.arange(case["max_positions"], dtype=torch.float64, device="cuda")[:, None] * inv_freq
        state["cos"], state["sin"] = angles.cos().float(), angles.sin().float()
        state["pool"] = _pool(case, 2, D, order, None)
    return state


# -- one pass ----------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    return {"rotate": _plain_rotate, "observe": _plain_observe, "select": _plain_select,
            "compact": _plain_compact}[state["op"]](state)


def _run_own(state):
    op, cache = state["op"], state["cache"]
    if op == "rotate":
        from specdecode_b200.rotary import norm_rotate_append

        query = norm_rotate_append(cache, state["pending"], state["layer"], state["query"], state["key"],
                                   state["value"], state["positions"], state["table"],
                                   query_weight=state["query_weight"], key_weight=state["key_weight"],
                                   eps=state["eps"])
        keys, values = cache.gather_slots(state["pending"].slots, torch.bfloat16, layer_begin=state["layer"],
                                          layers=1)
        return query, keys, values
    from specdecode_b200.eviction import compact_tokens, observe_attention, select_tokens

    if op == "observe":
        return observe_attention(cache, state["query"], state["ids"], state["layer"])
    case = state["case"]
    if op == "select":
        return select_tokens(cache, state["ids"], case["budget"], recent=case["recent"], sinks=case["sinks"])
    compact_tokens(cache, state["ids"], state["kept"])
    return cache.key_codes, cache.value_codes, cache.key_scale_pages, cache.value_scale_pages, state["mass"]


def _plain_rotate(state):
    case, pool = state["case"], state["pool"]
    cos, sin = state["cos"][state["positions"]][:, :, None], state["sin"][state["positions"]][:, :, None]
    half = case["style"] == "half"

    def normed(x, weight):
        x = x.float()
        if weight is None:
            return x
        return x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + state["eps"]) * weight.float()

    def rotated(x):
        a, b = (x.chunk(2, dim=-1) if half else (x[..., 0::2], x[..., 1::2]))
        parts = (a * cos - b * sin, b * cos + a * sin)
        return torch.cat(parts, dim=-1) if half else torch.stack(parts, dim=-1).flatten(-2)

    query = rotated(normed(state["query"], state["query_weight"])).transpose(1, 2).to(state["query"].dtype)
    keys = rotated(normed(state["key"], state["key_weight"]))
    out = []
    n = case["tokens"]
    t = torch.arange(n, device="cuda")
    block, offset = state["tables"][:, t // case["block_size"]], (t % case["block_size"]).expand(case["batch"], n)
    for x, name in ((keys, "key"), (state["value"].float(), "value")):
        scale = x.abs().amax(dim=-1, keepdim=True) / 127
        safe = torch.where(scale > 0, scale, 1.0)
        codes = torch.sign(x) * torch.floor(x.abs() / safe + 0.5).clamp_(max=127)
        pool[name + "s"][block, state["layer"], :, offset] = codes.to(torch.int8)
        pool[name + "_scales"][block, state["layer"], :, offset] = scale[..., 0]
        out.append((codes * scale).to(torch.bfloat16).reshape(case["batch"] * n, 1, *x.shape[2:]))
    return query.contiguous(), out[0], out[1]


def _at(state, t):
    """(block, offset, live) of tokens t of every sequence, [B, T]."""
    bs = state["case"]["block_size"]
    block = state["tables"][:, t // bs]
    live = t < state["lengths"][:, None]
    return block, (t % bs).expand_as(block), live


def _plain_observe(state):
    case, pool, layer = state["case"], state["pool"], state["layer"]
    B, Hk, w, D = case["batch"], case["kv_heads"], case["window"], case["head_dim"]
    t = torch.arange(state["longest"], device="cuda")
    block, offset, live = _at(state, t)
    keys = pool["keys"][block, layer, :, offset].float() * pool["key_scales"][block, layer, :, offset][..., None]
    query = state["query"].float().reshape(B, Hk, -1, D)
    scores = torch.matmul(query, keys.permute(0, 2, 3, 1)) / math.sqrt(D)
    scores = scores.view(B, Hk, -1, w, state["longest"])
    last = state["lengths"][:, None] - w + torch.arange(w, device="cuda")
    scores = torch.where((t <= last[..., None])[:, None, None], scores, -math.inf)
    scores = scores - scores.amax(dim=-1, keepdim=True)
    weights = torch.exp(scores)
    weights = weights / weights.sum(dim=-1, keepdim=True)
    added = weights.sum(dim=(2, 3)).transpose(1, 2)
    mass = state["mass"]
    where = live.nonzero(as_tuple=True)
    mass[block[where], layer, :, offset[where]] += added[where]
    return mass


def _plain_select(state):
    case = state["case"]
    N, recent, sinks = case["budget"], case["recent"], case["sinks"]
    t = torch.arange(max(state["longest"], N), device="cuda")
    longest = state["longest"]
    block, offset, _ = _at(state, t[:longest])
    mass = state["mass"][block, :, :, offset].permute(0, 2, 3, 1)
    T = state["lengths"][:, None, None, None]
    rank = torch.where((t[:longest] < sinks) | (t[:longest] >= T - recent), math.inf, mass)
    rank = torch.where(t[:longest] < T, rank, -math.inf)
    if longest < N:
        rank = torch.nn.functional.pad(rank, (0, N - longest), value=-math.inf)
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :N].sort(dim=-1).values
    every = torch.where(t[:N] < T, t[:N], -1)
    return torch.where(T > N, kept, every).to(torch.int32)


def _plain_compact(state):
    case, pool, mass = state["case"], state["pool"], state["mass"]
    bs, N = case["block_size"], case["budget"]
    L, H = case["layers"], case["kv_heads"]
    move = (state["lengths"] > N).nonzero()[:, 0]
    if move.numel():
        kept = state["kept"][move].long()
        to = torch.arange(N, device="cuda").expand_as(kept)
        row = move[:, None, None, None]
        layer = torch.arange(L, device="cuda")[:, None, None].expand_as(kept)
        head = torch.arange(H, device="cuda")[:, None].expand_as(kept)
        src = (state["tables"][row, kept // bs], layer, head, kept % bs)
        dst = (state["tables"][row, to // bs], layer, head, to % bs)
        for pages in (pool["keys"], pool["values"], pool["key_scales"], pool["value_scales"], mass):
            pages[dst] = pages[src]
    return pool["keys"], pool["values"], pool["key_scales"], pool["value_scales"], mass


# -- what one pass cannot do without --------------------------------------------
def work(case):
    op, Hk = case["op"], case["kv_heads"]
    if op == "rotate":
        n, D, es = case["batch"] * case["tokens"], case["head_dim"], 4 if case["dtype"] == "f32" else 2
        per_token = (2 * case["query_heads"] + 2 * Hk) * D * es + 2 * Hk * (D + 4)  # in, queries out, codes and scales
        per_token += 8 + D * 4 + 8  # position, its angles' cosines and sines, slot
        back = 2 * Hk * (D * 3 + 4)  # the codes and scales read back as bf16 values
        return {"bytes": float(n * (per_token + back)), "flops": float(n * (case["query_heads"] + 2 * Hk) * D * 8)}
    tokens = case["batch"] * (case["shortest"] + case["longest"]) / 2
    if op == "observe":
        rows = case["query_heads"] // Hk * case["window"]
        es = 4 if case["dtype"] == "f32" else 2
        q = case["batch"] * case["query_heads"] * case["window"] * case["head_dim"] * es
        return {"bytes": tokens * Hk * (case["head_dim"] + 4 + 8) + q,
                "flops": tokens * Hk * rows * (2.0 * case["head_dim"] + 4)}
    vectors = case["layers"] * Hk
    kept = case["batch"] * min(case["budget"], (case["shortest"] + case["longest"]) / 2) * vectors
    if op == "select":
        return {"bytes": tokens * vectors * 4 + kept * 4, "flops": tokens * vectors}
    return {"bytes": kept * (2 * (2 * (case["head_dim"] + 4) + 4) + 4), "flops": 0}


# -- the definitions in 64 bits ------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op == "select":
        return None  # whole numbers
    state = prepare(case, seed)
    if op == "rotate":
        return _exact_rotate(case, state)
    if op == "observe":
        return _exact_observe(case, state)
    return _exact_compact(case, state)


def _exact_rotate(case, state):
    D = case["head_dim"]
    theta = state["positions"].double()[:, :, None, None] * state["inv_freq"]
    turn = torch.complex(theta.cos(), theta.sin())

    def head(x, weight):
        x = x.double()
        if weight is not None:
            x = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / D + state["eps"]) * weight.double()
        if case["style"] == "half":
            z = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn
            return torch.cat((z.real, z.imag), dim=-1)
        z = torch.view_as_complex(x.unflatten(-1, (D // 2, 2)).contiguous()) * turn
        return torch.view_as_real(z).flatten(-2)

    def stored(x):
        x = x.double()
        scale = (x.abs().max(-1, keepdim=True).values / 127).float().double()
        codes = torch.where(scale > 0, torch.trunc(x / scale.clamp_min(1e-300) + 0.5 * torch.sign(x)), 0.0)
        return (codes.clamp(-127, 127) * scale).flatten(0, 1).unsqueeze(1)

    return (head(state["query"], state["query_weight"]).permute(0, 2, 1, 3).contiguous(),
            stored(head(state["key"], state["key_weight"])), stored(state["value"]))


def _exact_observe(case, state):
    Hk, w, D, bs = case["kv_heads"], case["window"], case["head_dim"], case["block_size"]
    layer, pool = state["layer"], state["pool"]
    mass = state["mass"].double()
    for b, T in enumerate(state["lengths"].tolist()):
        blocks = state["tables"][b, :-(-T // bs)]
        k = pool["keys"][blocks, layer].double() * pool["key_scales"][blocks, layer].double()[..., None]
        k = k.transpose(0, 1).reshape(Hk, -1, D)[:, :T]
        q = state["query"][b].double().view(Hk, -1, D)
        s = torch.einsum("hrd,htd->hrt", q, k) * D ** -0.5
        row = torch.arange(q.shape[1], device="cuda") % w
        hidden = torch.arange(T, device="cuda") > (T - w + row)[:, None]
        s = s.masked_fill(hidden, -math.inf)
        p = torch.exp(s - torch.logsumexp(s, dim=-1, keepdim=True)).sum(dim=1)
        p = torch.nn.functional.pad(p, (0, blocks.numel() * bs - T)).view(Hk, -1, bs).transpose(0, 1)
        mass[blocks, layer] += p
    return mass


def _exact_compact(case, state):
    bs, N = case["block_size"], case["budget"]
    pool = {**state["pool"], "mass": state["mass"]}
    out = {name: pages.double() if pages.dtype != torch.int8 else pages.clone() for name, pages in pool.items()}
    for b, T in enumerate(state["lengths"].tolist()):
        if T <= N:
            continue
        table = state["tables"][b]
        dst = torch.arange(N, device="cuda")
        for layer in range(case["layers"]):
            for h in range(case["kv_heads"]):
                src = state["kept"][b, layer, h].long()
                for name, pages in pool.items():
                    out[name][table[dst // bs], layer, h, dst % bs] = \
                        pages[table[src // bs], layer, h, src % bs].to(out[name].dtype)
    return [out[name] for name in ("keys", "values", "key_scales", "value_scales", "mass")]
