"""Packed 4-bit projections move with their model and stay out of its state dict."""

import torch


def test_packed_weights_follow_the_module():
    from lastkv_b200 import ops
    from lastkv_b200.hf import LastKVConfig, LastKVForCausalLM, QuantizedLinears

    cfg = LastKVConfig(hidden_size=128, intermediate_size=96, num_attention_heads=2, num_key_value_heads=1,
                       num_hidden_layers=1, head_dim=64, vocab_size=32, chunk_size=32)
    model = LastKVForCausalLM(cfg).to(torch.bfloat16)
    keys, params = list(model.state_dict()), [n for n, _ in model.named_parameters()]
    bias = torch.zeros(32, dtype=torch.bfloat16)
    mlp = model.model.layers[0].mlp
    mlp._w4 = torch.nn.ModuleList(
        QuantizedLinears(ops.W4Weight(torch.zeros(2112, dtype=torch.uint8), 32, 128, 128), b, True) for b in (bias, None))
    assert list(model.state_dict()) == keys and [n for n, _ in model.named_parameters()] == params
    model.to("meta")
    for q in mlp._w4:
        assert q.weight.packed.device.type == "meta" and q.weight.packed.dtype == torch.uint8
        assert q.weight[1:] == (32, 128, 128)
    assert mlp._w4[0].bias.device.type == "meta" and mlp._w4[1].bias is None
