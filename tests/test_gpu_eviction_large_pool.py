"""Selection, compaction and clearing over a pool whose offsets pass 32 bits in
every unit: three blocks 33 GiB apart, so that codes pass 64 GiB and scales
2^32 elements.  One buffer holds all of it, only the blocks' first pages are
touched, and what comes out is compared with indexing, bit by bit."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

L, H, D, BS = 2, 2, 64, 16
STRIDE = 33 << 30  # bytes from block to block


@pytest.fixture
def pages(device):
    import torch

    from specdecode_b200 import _lib

    need = 2 * STRIDE + (1 << 20)
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(device)[0] < need + (2 << 30):
        pytest.skip("needs 66 GiB of free device memory")
    buffer = torch.empty(need, dtype=torch.uint8, device=device)
    codes, scales = L * H * BS * D, L * H * BS * 4
    base = buffer.data_ptr()
    at = {"key_codes": 0, "value_codes": codes, "key_scales": 2 * codes, "value_scales": 2 * codes + scales,
          "mass": 2 * codes + 2 * scales}
    assert all(offset % 16 == 0 for offset in at.values()) and at["mass"] + scales <= 1 << 20
    pool = _lib.PagePool(base, base + at["value_codes"], base + at["key_scales"], base + at["value_scales"], 3, BS, L,
                         H, D, STRIDE, H * BS * D, BS * D, STRIDE // 4, H * BS, BS)

    def page(block, name):
        kind, nbytes = (torch.int8, codes) if name.endswith("codes") else (torch.float32, scales)
        start = block * STRIDE + at[name]
        shape = (L, H, BS, D) if name.endswith("codes") else (L, H, BS)
        return buffer[start:start + nbytes].view(kind).view(shape)

    g = torch.Generator(device=device).manual_seed(3)
    for block in range(3):
        for name in at:
            p = page(block, name)
            if p.dtype == torch.int8:
                p.copy_(torch.randint(-127, 128, p.shape, generator=g, device=device))
            else:
                p.copy_(torch.rand(p.shape, generator=g, device=device))
    yield pool, page, base + at["mass"], list(at)
    del buffer
    torch.cuda.empty_cache()


def test_pools_past_32_bit_offsets(device, pages):
    import torch

    from oracle.eviction import select_kept
    from specdecode_b200 import _lib

    pool, page, mass, names = pages
    library = _lib.load_library()
    stream = torch.cuda.current_stream(device).cuda_stream
    order, T, budget = [2, 0, 1], 45, 21
    table = torch.tensor([order], dtype=torch.int32, device=device)
    lens = torch.tensor([T], dtype=torch.int32, device=device)
    status = torch.zeros(1, dtype=torch.int32, device=device)

    def tokens(name):  # [L, H, 48, ...]
        return torch.cat([page(block, name) for block in order], dim=2)

    kept = torch.full((1, L, H, budget), -7, dtype=torch.int32, device=device)
    library.check(library.handle.sdc_select_tokens(
        ctypes.byref(pool), mass, 1, table.data_ptr(), 3, lens.data_ptr(), T, budget, 3, 2, kept.data_ptr(),
        status.data_ptr(), stream), "selection")
    weights = tokens("mass").cpu().numpy()
    for layer in range(L):
        for h in range(H):
            assert np.array_equal(kept[0, layer, h].cpu().numpy(), select_kept(weights[layer, h, :T], budget, 3, 2))

    before = {name: tokens(name) for name in names}
    library.check(library.handle.sdc_compact_tokens(
        ctypes.byref(pool), mass, 1, table.data_ptr(), 3, lens.data_ptr(), kept.data_ptr(), budget, status.data_ptr(),
        stream), "compaction")
    for name in names:
        want = before[name].clone()
        for layer in range(L):
            for h in range(H):
                want[layer, h, :budget] = before[name][layer, h, kept[0, layer, h].long()]
        assert torch.equal(tokens(name), want), name

    slots = torch.tensor([1 * BS + 12, 2 * BS + 5, 0], dtype=torch.int64, device=device)
    want = {block: page(block, "mass").clone() for block in range(3)}
    library.check(library.handle.sdc_clear_mass(ctypes.byref(pool), mass, slots.data_ptr(), 3, status.data_ptr(),
                                                stream), "clearing")
    for block, offset in ((1, 12), (2, 5), (0, 0)):
        want[block][:, :, offset] = 0.0
    assert all(torch.equal(page(block, "mass"), want[block]) for block in range(3))
    assert int(status.item()) == 0
