"""What of the models needs no GPU."""

import io

import torch


def test_models_saved_whole_before_packed_training():
    """A model that was saved as an object by a version without packed training has no such attribute on its instances."""
    from gsa_b200 import GSAConfig, GSALlamaForCausalLM

    cfg = GSAConfig(d_model=64, n_heads=2, n_kv_heads=1, d_indexer=16, n_indexer_heads=2, k_base=8, k_min=4, k_max=16, n_layers=1,
                    d_ffn=64, vocab_size=32, max_position_embeddings=32)
    m = GSALlamaForCausalLM(cfg)
    for module in (m.model, *m.model.layers):
        module.__dict__.pop("packed_training", None)
    buf = io.BytesIO()
    torch.save(m, buf)
    buf.seek(0)
    m = torch.load(buf, weights_only=False)
    assert m.model.packed_training is False and all(layer.packed_training is False for layer in m.model.layers)
    m.enable_packed_training()
    assert m.model.packed_training and all(layer.packed_training for layer in m.model.layers)
    assert not type(m.model).packed_training and not type(m.model.layers[0]).packed_training
