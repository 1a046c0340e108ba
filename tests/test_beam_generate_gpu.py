"""Beam search through transformers' ``generate`` and through ``generate_beam`` on one model's weights."""

import pytest
import torch

from tests.test_beam_model_gpu import _model, _plain_beams, _prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,K,P,new", [(1, 4, 20, 30), (2, 3, 33, 40)])
def test_generate_with_beams_finds_the_same_sequences(B, K, P, new):
    """Without an end token both keep the K best sequences of a step.  Their totals are summed in another order, so the
    prompts are such that no step has candidates closer than 1e-5 (checked by the plain form, which runs every beam
    from its first token)."""
    from lastkv_b200.llm import CustomRecurrentMarinAKV254ReuseKVConfig, CustomRecurrentMarinAKV254ReuseKVForCausalLM

    torch.backends.cuda.matmul.allow_tf32 = False
    plain = _model(torch.float32, seed=3)
    c = plain.config
    cfg = CustomRecurrentMarinAKV254ReuseKVConfig(
        hidden_size=c.hidden_size, intermediate_size=c.intermediate_size, num_attention_heads=c.num_attention_heads,
        num_key_value_heads=c.num_key_value_heads, num_hidden_layers=c.num_hidden_layers, head_dim=c.head_dim,
        vocab_size=c.vocab_size, chunk_size=c.chunk_size, rms_norm_eps=c.rms_norm_eps, rope_theta=c.rope_theta,
        bos_token_id=1, eos_token_id=None, pad_token_id=0)
    model = CustomRecurrentMarinAKV254ReuseKVForCausalLM(cfg)
    model.load_state_dict(plain.state_dict(), strict=True)
    model.model._alpha = None
    model = model.cuda().eval()
    prompt = _prompt(B, P)
    seqs, _, _ = _plain_beams(plain, prompt, K, new)
    found = plain.generate_beam(prompt, K, new).sequences
    with torch.inference_mode():
        out = model.generate(prompt, max_new_tokens=new, do_sample=False, use_cache=True, num_beams=K,
                             num_return_sequences=K)
    assert torch.equal(found, seqs)
    assert torch.equal(out.view(B, K, -1), seqs)
