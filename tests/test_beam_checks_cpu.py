"""Beam search that cannot be served is refused before it touches the cache."""

import pytest
import torch

from lastkv_b200.contract import RMarinBackendContractError as Refused
from lastkv_b200.hf import LastKVConfig, LastKVForCausalLM, PagedLastKVCache
from lastkv_b200.runner import GraphDecodeRunner


def _model(vocab=20):
    cfg = LastKVConfig(hidden_size=64, intermediate_size=96, num_attention_heads=4, num_key_value_heads=2,
                       num_hidden_layers=1, head_dim=64, vocab_size=vocab, chunk_size=32)
    return LastKVForCausalLM(cfg)


@pytest.mark.parametrize("vocab,beams,eos,word", [(100, 33, None, "32"), (20, 21, None, "20"), (100, 0, None, "beam"),
                                                  (100, 4, 100, "eos_token"), (100, 4, -1, "eos_token")])
def test_beams_that_the_selection_does_not_serve(vocab, beams, eos, word):
    model = _model(vocab)
    cache = PagedLastKVCache(model.config, max(beams, 1), 64, device="cpu", dtype=torch.float32)
    with pytest.raises(Refused, match=word):
        GraphDecodeRunner(model, cache, beams=beams, eos_token=eos)
    with pytest.raises(Refused, match=word):
        model.generate_beam(torch.zeros((1, 3), dtype=torch.int64), beams, 4, eos_token=eos, cache=cache)
    assert cache.seen_tokens == 0 and not cache.pool_k.any()


@pytest.mark.parametrize("beams", [None, 2])
def test_a_prompt_without_a_token(beams):
    model = _model()
    runner = object.__new__(GraphDecodeRunner)  # (the step's buffers need a GPU)
    runner.model, runner.beams, runner.B = model, beams, 2
    runner.cache = PagedLastKVCache(model.config, 2, 64, device="cpu", dtype=torch.float32)
    with pytest.raises(Refused, match="token"):
        runner.prefill(torch.zeros((2 if beams is None else 1, 0), dtype=torch.int64), 16)
    assert runner.cache.seen_tokens == 0
