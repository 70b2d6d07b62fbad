"""Views the rotated append takes: whatever the strides, what reaches the
kernel lies on 16 bytes, dimensions of one element included."""

from __future__ import annotations

import numpy as np
import pytest

from gpu_helpers import make_cache


def views(device):
    """Inputs [B, n, H, D] whose strides no kernel can take as they are."""
    import torch

    def make(*shape):
        return torch.randn(shape, device=device).to(torch.bfloat16)

    return [
        make(1, 1, 1, 67)[..., :64],                            # one head vector of a padded row
        make(1, 5, 2, 64).as_strided((1, 5, 2, 64), (3, 128, 64, 1)),
        make(4, 1, 2, 64)[1:2].as_strided((1, 1, 2, 64), (7, 9, 64, 1)),
        make(3, 5, 1, 67)[..., :64],
        make(2, 3, 2, 128)[..., ::2],
        make(1, 2, 2, 72)[..., 1:65],
        make(2, 64, 2, 3).permute(0, 3, 2, 1),
    ]


@pytest.mark.parametrize("which", range(7))
def test_any_view_is_brought_to_16_bytes(which):
    import torch

    from specdecode_b200.rotary import _heads

    x = views(torch.device("cpu"))[which]
    y = _heads(x, "query", tuple(x.shape), x.dtype, x.device)
    assert torch.equal(x, y) and y.stride(3) == 1 and y.data_ptr() % 16 == 0
    assert all(s * y.element_size() % 16 == 0 for s in y.stride()[:3])
    # and what fits is read in place
    packed = torch.zeros(2, 3, 6, 64, dtype=torch.bfloat16)[:, :, 1:4]
    assert _heads(packed, "query", (2, 3, 3, 64), packed.dtype, packed.device).data_ptr() == packed.data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(7))
def test_views_give_what_their_copies_give(device, which):
    import torch

    from specdecode_b200.rotary import RotaryTable, norm_rotate_append

    x = views(device)[which]
    B, n, H, D = x.shape
    table = RotaryTable(D, 16, device=device)
    got = []
    for q in (x, x.clone(memory_format=torch.contiguous_format)):
        cache = make_cache(device, 1, H, D, 16, B, max_sequences=B)
        for s in range(B):
            cache.create_sequence(s)
        pending = cache.reserve(list(range(B)), n)
        out = norm_rotate_append(cache, pending, 0, q, q, q, torch.arange(n, device=device), table)
        assert cache.status_bits() == 0
        got.append((out, cache.key_codes, cache.value_codes, cache.key_scale_pages))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert np.count_nonzero(got[0][1].cpu().numpy())
