"""The observation switched on and off under captured decoding passes."""

from __future__ import annotations

import pytest

from gpu_helpers import make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graphs", [False, True])
def test_the_switch_holds_for_captured_passes(device, graphs):
    """Every verify pass adds its query rows' weights, one unit a row, exactly
    while the switch is on: the mass is read after each round."""
    import torch
    from transformers import LlamaConfig, LlamaForCausalLM

    from specdecode_b200.speculative import BatchedSpeculativeDecoder, DraftWindow

    torch.manual_seed(2)
    config = LlamaConfig(hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
                         num_key_value_heads=1, head_dim=64, vocab_size=100, max_position_embeddings=512)
    model = LlamaForCausalLM(config).to(device=device, dtype=torch.bfloat16).eval()
    B, P, new, window = 2, 9, 8, 4

    def cache():
        made = make_cache(device, 2, 1, 64, 16, 64, max_sequences=B)
        made.track_attention()
        return made

    decoder = BatchedSpeculativeDecoder(model, model, cache(), cache(), window=DraftWindow(window, dynamic=False),
                                        temperature=0.0, seed=1, cuda_graphs=graphs)
    grown = []
    target = decoder.target.cache
    original = decoder._graphed_forward if graphs else decoder._forward

    def watched(session, model, ids, tokens, keep):
        before = target.attention_mass.double().sum().item()
        out = original(session, model, ids, tokens, keep)
        if session is decoder.target and keep > 1:
            grown.append(target.attention_mass.double().sum().item() - before)
        return out

    if graphs:
        decoder._graphed_forward = watched
    else:
        decoder._forward = watched
    prompts = torch.randint(0, 100, (B, P))
    rows = 2 * B * 4 * (window + 1)  # layers x sequences x query heads x tokens of a verify pass
    with torch.no_grad():
        for on in (False, True, False, True):
            grown.clear()
            decoder.target.observe_attention = on
            decoder.generate(prompts, new)
            assert len(grown) >= 2
            # a row's weights sum to one within its roundings
            assert all(abs(g - (rows if on else 0)) <= 1e-4 * rows for g in grown), (on, grown)
