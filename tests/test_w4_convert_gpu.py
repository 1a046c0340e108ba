"""Converting a model's projections to 4 bits: what is freed, what is refused, what is left as it was."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def build(layers=2, **kw):
    from lastkv_b200.hf import LastKVConfig, LastKVForCausalLM
    from lastkv_b200.runner import init_random_

    cfg = LastKVConfig(**{**dict(hidden_size=512, intermediate_size=1032, num_attention_heads=8, num_key_value_heads=2,
                                 num_hidden_layers=layers, head_dim=64, vocab_size=512, chunk_size=32), **kw})
    model = LastKVForCausalLM(cfg).cuda().to(torch.bfloat16).eval()
    init_random_(model, seed=5)
    return model


def projections(layer):
    a, m = layer.self_attn, layer.mlp
    return [a.q_proj, a.k_proj, a.v_proj, a.o_proj, m.gate_proj, m.up_proj, m.down_proj]


@pytest.mark.parametrize("fused", [False, True])
def test_release_frees_the_bf16_weights(fused):
    """Fused projections first, as examples/w4_decode.py has them, or not."""
    model = build(hidden_size=1024, intermediate_size=4096, num_attention_heads=16)
    if fused:
        model.fuse_projections_()
    weights = sum(lin.weight.numel() * 2 for layer in model.model.layers for lin in projections(layer))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    model.quantize_projections_(release=True)
    torch.cuda.synchronize()
    # 4 bits and a bf16 scale per 128 columns take the place of 16 bits; 1 MB for the allocations' rounding
    assert torch.cuda.memory_allocated() - before <= weights * (4 + 16 / 128) / 16 - weights + 2 ** 20


@pytest.mark.parametrize("why", ["width", "type", "device", "released", "group"])
def test_a_refusal_leaves_the_model_as_it_was(why):
    """The last layer's down projection cannot be converted: no weight of the model is touched."""
    from lastkv_b200.contract import RMarinBackendContractError

    model = build(intermediate_size=1028 if why == "width" else 1032)
    group = 48 if why == "group" else 128
    down = model.model.layers[-1].mlp.down_proj
    if why == "type":
        down.weight.data = down.weight.data.float()
    elif why == "device":
        down.weight.data = down.weight.data.cpu()
    elif why == "released":
        down.weight = torch.nn.Parameter(down.weight.new_empty((0, down.in_features)), requires_grad=False)
    before = [[lin.weight for lin in projections(layer)] for layer in model.model.layers]
    kept = [[w.detach().clone() for w in layer] for layer in before]
    with pytest.raises(RMarinBackendContractError):
        model.quantize_projections_(group, release=True)
    for layer, weights, values in zip(model.model.layers, before, kept):
        assert layer.self_attn._w4 is None and layer.mlp._w4 is None
        for lin, w, v in zip(projections(layer), weights, values):
            assert lin.weight is w and torch.equal(w, v)


def test_a_quantized_model_moves():
    """To the host, where its products are refused, and back, where they are what they were."""
    import copy

    from lastkv_b200.contract import RMarinBackendContractError

    model = build(attention_bias=True).quantize_projections_(release=True)
    tokens = torch.arange(40, device="cuda")[None] % 512

    @torch.no_grad()
    def logits(m):
        return m(tokens, m.new_cache(1, 40))[0]

    want = logits(model)
    assert torch.equal(logits(copy.deepcopy(model)), want)
    cache = model.new_cache(1, 40)
    model.cpu()
    with pytest.raises(RMarinBackendContractError), torch.no_grad():
        model.model.layers[0].mlp(torch.zeros((1, 1, 512), dtype=torch.bfloat16, device="cuda"), cache.error_word)
    assert torch.equal(logits(model.cuda()), want)


def test_a_bf16_copy_prefills_for_the_quantized_model():
    """One cache: the prompt by the model with bf16 weights, the tokens behind it by its 4-bit copy."""
    import copy

    from lastkv_b200.runner import GraphDecodeRunner

    model = build().fuse_projections_()
    small = copy.deepcopy(model).quantize_projections_(release=True)
    prompt = torch.arange(120, device="cuda").view(2, 60)
    tokens, pools = [], []
    with torch.no_grad():
        for graph in (False, True):
            cache = small.new_cache(2, 80)
            logits, _ = model(prompt, cache, logits_to_keep=1)
            pools.append(cache.pool_k.clone())
            ids = logits[:, -1].float().argmax(-1, keepdim=True)
            out = [ids]
            if graph:
                runner = GraphDecodeRunner(small, cache, device_plan=True)
                runner.ids.copy_(ids)
                runner.capture()
                out += [runner.step().clone() for _ in range(10)]
            else:
                for _ in range(10):
                    logits, _ = small(out[-1], cache, logits_to_keep=1)
                    out.append(logits[:, -1].float().argmax(-1, keepdim=True))
            cache.check_errors()
            tokens.append(torch.cat(out, 1))
        alone = model.new_cache(2, 80)
        model(prompt, alone)
    assert torch.equal(tokens[0], tokens[1])
    assert torch.equal(pools[0], alone.pool_k) and torch.equal(pools[1], alone.pool_k)
