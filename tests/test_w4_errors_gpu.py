"""What goes wrong on the device in a 4-bit product of the model is seen by the cache's check_errors."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("activations", ["int8", "bf16"])
@pytest.mark.parametrize("tokens", [1, 200])  # 200 rows: bf16 activations either way
def test_every_product_reports_into_the_caches_error_word(monkeypatch, activations, tokens):
    from lastkv_b200 import ops
    from lastkv_b200.contract import RMarinBackendContractError
    from lastkv_b200.hf import LastKVConfig, LastKVForCausalLM
    from lastkv_b200.runner import init_random_

    cfg = LastKVConfig(hidden_size=512, intermediate_size=1024, num_attention_heads=8, num_key_value_heads=2,
                       num_hidden_layers=2, head_dim=64, vocab_size=512, chunk_size=256)
    model = LastKVForCausalLM(cfg).cuda().to(torch.bfloat16).eval()
    init_random_(model, seed=5)
    model.quantize_projections_(activations=activations)
    words, linear = [], ops.w4_linear

    def spy(x, weight, bias=None, *, out=None, error_word=None):
        words.append(error_word)
        return linear(x, weight, bias, out=out, error_word=error_word)

    monkeypatch.setattr(ops, "w4_linear", spy)
    cache = model.new_cache(1, 256)
    with torch.no_grad():
        model(torch.zeros((1, tokens), dtype=torch.int64, device="cuda"), cache)
    assert len(words) == 8 and all(w is cache.error_word for w in words)
    cache.check_errors()
    cache.error_word[0] = 1  # as a wait that gave up leaves it
    with pytest.raises(RMarinBackendContractError):
        cache.check_errors()
