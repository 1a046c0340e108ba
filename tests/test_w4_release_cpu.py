"""What quantize_projections_ keeps of the bf16 weights, without a GPU: the rounding to 4 bits is left out."""

import gc
import weakref

import pytest
import torch


def tiny(**kw):
    from lastkv_b200.hf import LastKVConfig, LastKVForCausalLM

    cfg = LastKVConfig(**{**dict(hidden_size=128, intermediate_size=96, num_attention_heads=2, num_key_value_heads=1,
                                 num_hidden_layers=2, head_dim=64, vocab_size=32, chunk_size=32), **kw})
    return LastKVForCausalLM(cfg).to(torch.bfloat16).eval()


def projections(layer):
    a, m = layer.self_attn, layer.mlp
    return [a.q_proj, a.k_proj, a.v_proj, a.o_proj, m.gate_proj, m.up_proj, m.down_proj]


@pytest.mark.parametrize("fused", [False, True])
def test_release_lets_every_projection_weight_go(monkeypatch, fused):
    from lastkv_b200 import hf

    def of(linears, group, int8, release):
        """Frees the weights as QuantizedLinears.of does on the GPU."""
        for lin in linears:
            lin.weight = torch.nn.Parameter(lin.weight.new_empty((0, lin.in_features)), requires_grad=False)
        return torch.nn.Identity()

    monkeypatch.setattr(hf.QuantizedLinears, "of", staticmethod(of))
    monkeypatch.setattr(hf.QuantizedLinears, "check", staticmethod(lambda linears, group: None))
    model = tiny()
    if fused:
        model.fuse_projections_()
    held = []
    for layer in model.model.layers:
        held += [weakref.ref(lin.weight) for lin in projections(layer)]
        if fused:  # the tensors that the weights are views of
            held += [weakref.ref(layer.self_attn._qkv[0]), weakref.ref(layer.mlp._gate_up[0])]
    model.quantize_projections_(release=True)
    gc.collect()
    assert all(r() is None for r in held)
