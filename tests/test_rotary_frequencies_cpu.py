"""Where rotary_frequencies and the attention layer's own embedding read a rope_scaling dictionary alike, and where they do not:
keys rotated for a layer's cache have to come from a dictionary of the first kind."""

import pytest
import torch

ALIKE = [None, dict(type="ntk", factor=4.0), dict(type="yarn", factor=16.0, original_max_position_embeddings=4096)]
APART = [dict(type="linear", factor=4.0), dict(type="llama3", factor=8.0),
         dict(type="dynamic_ntk", factor=2.0, original_max_position_embeddings=256), dict(rope_type="ntk", factor=4.0)]


def _both(scaling):
    import gsa_b200 as gsa

    emb = gsa.RotaryEmbedding(64, 4, 10000.0, scaling)
    return gsa.rotary_frequencies(64, 10000.0, scaling, seq_len=1000), emb.inv_freq.double()


@pytest.mark.parametrize("scaling", ALIKE)
def test_the_layer_reads_it_alike(scaling):
    (f, m), layer = _both(scaling)
    assert m == 1.0 and float((f / layer - 1).abs().max()) < 8 * 2.0 ** -24


@pytest.mark.parametrize("scaling", APART)
def test_the_layer_keeps_the_standard_frequencies(scaling):
    (f, _), layer = _both(scaling)
    standard = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert float((layer / standard - 1).abs().max()) < 8 * 2.0 ** -24
    assert float((f / layer - 1).abs().max()) > 0.1


def test_the_layer_has_no_attention_factor():
    import gsa_b200 as gsa

    scaling = dict(type="yarn", factor=16.0, attention_factor=1.25)
    assert gsa.rotary_frequencies(64, scaling=scaling)[1] == 1.25
    plain = gsa.RotaryEmbedding(64, 4, 10000.0, dict(type="yarn", factor=16.0))
    assert torch.equal(gsa.RotaryEmbedding(64, 4, 10000.0, scaling).cos_cached, plain.cos_cached)
