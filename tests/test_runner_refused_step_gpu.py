"""A step that is refused at a full cache leaves the cache as it was, its queued boundary commit included."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("device_plan", [False, True])
def test_the_queued_commit_survives(device_plan):
    from lastkv_b200.contract import RMarinBackendContractError
    from lastkv_b200.hf import LastKVConfig, LastKVForCausalLM
    from lastkv_b200.runner import GraphDecodeRunner, init_random_

    cfg = LastKVConfig(hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=2,
                       num_hidden_layers=2, head_dim=64, vocab_size=512, chunk_size=32)
    model = LastKVForCausalLM(cfg).cuda().to(torch.bfloat16).eval()
    init_random_(model, seed=3)
    prompt = torch.arange(120, device="cuda").view(2, 60)
    pools, last = [], []
    for refused in (False, True):
        cache = model.new_cache(2, 64)  # ends with a chunk
        runner = GraphDecodeRunner(model, cache, device_plan=device_plan)
        with torch.no_grad():
            runner.prefill(prompt, 60)
            runner.capture()
            for _ in range(4):
                runner.step()
            if refused:
                for _ in range(2):
                    with pytest.raises(RMarinBackendContractError):
                        runner.step()
                assert cache._pending is not None
            cache.reserve(80)  # flushes the commit
            logits, _ = model(prompt[:, :3], cache)
        pools.append((cache.pool_k.clone(), cache.pool_v.clone()))
        last.append(logits)
    assert torch.equal(*last)
    for a, b in zip(*pools):
        assert torch.equal(a, b)
