"""The model with 4-bit projections, and the graph runner that plans its steps on the device.

The 4-bit model is compared with the same model whose projection weights are the 4-bit values (each read back through
one-hot rows, exact before its rounding to bf16).  bf16 activations: the two differ by that rounding and by sums in
another order, a few bf16 roundings (2^-8) per projection: 2 % of the logits' norm.  int8 activations add a rounding
to steps of max / 127 per group of 128 normal values, about 0.7 % of an input's norm, at seven projections per layer
in three layers, in quadrature 3 %: 6 % with the bf16 part.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

LIMIT = {"bf16": 0.02, "int8": 0.06}


def build(seed=7, layers=3, **kw):
    from lastkv_b200.hf import LastKVConfig, LastKVForCausalLM
    from lastkv_b200.runner import init_random_

    cfg = LastKVConfig(**{**dict(hidden_size=512, intermediate_size=1032, num_attention_heads=8, num_key_value_heads=2,
                                 num_hidden_layers=layers, head_dim=64, vocab_size=512, chunk_size=32), **kw})
    model = LastKVForCausalLM(cfg).cuda().to(torch.bfloat16).eval()
    init_random_(model, seed=seed)
    if cfg.attention_bias:
        with torch.no_grad():
            for name, p in model.named_parameters():
                if name.endswith("bias"):
                    p.normal_(0.0, 0.1)
    return model


def four_bit_values(model, group):
    """Replace every projection's weight by its 4-bit values."""
    from lastkv_b200 import ops

    with torch.no_grad():
        for layer in model.model.layers:
            a, m = layer.self_attn, layer.mlp
            for lin in (a.q_proj, a.k_proj, a.v_proj, a.o_proj, m.gate_proj, m.up_proj, m.down_proj):
                eye = torch.eye(lin.in_features, device="cuda", dtype=torch.bfloat16)
                lin.weight.copy_(ops.w4_linear(eye, ops.w4_quantize(lin.weight, group)).T)
    return model


def run(model, tokens, segments):
    cache = model.new_cache(tokens.shape[0], tokens.shape[1])
    out, start = [], 0
    with torch.no_grad():
        for size in segments:
            logits, cache = model(tokens[:, start:start + size], cache)
            out.append(logits.float())
            start += size
    cache.check_errors()
    return torch.cat(out, 1)


@pytest.mark.parametrize("activations", ["bf16", "int8"])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("bias", [False, True])
def test_model_matches_its_four_bit_values(activations, group, bias):
    gen = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, 512, (2, 110), generator=gen, device="cuda")
    segments = [70] + [1] * 20 + [20]  # prefill spans and single tokens over three boundaries
    model = build(attention_bias=bias)
    got = run(model.quantize_projections_(group, activations), tokens, segments)
    torch.manual_seed(0)
    plain = build(attention_bias=bias)
    for (_, a), (_, b) in zip(model.named_parameters(), plain.named_parameters()):
        b.data.copy_(a.data)
    want = run(four_bit_values(plain, group), tokens, segments)
    off = float((got - want).norm() / want.norm())
    print(f"{activations} rows, groups of {group}: {off:.4f} of the logits' norm")
    assert off < LIMIT[activations]


@pytest.mark.parametrize("activations", ["bf16", "int8"])
def test_long_spans(activations):
    """Long spans run on bf16 activations; the compared model has the weights rounded to bf16."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    tokens = torch.randint(0, 512, (2, 600), generator=gen, device="cuda")
    segments = [590, 10]
    model = build(chunk_size=512)
    got = run(model.quantize_projections_(64, activations), tokens, segments)
    want = run(four_bit_values(build(chunk_size=512), 64), tokens, segments)
    off = float((got[:, :512] - want[:, :512]).norm() / want[:, :512].norm())
    print(f"{activations}: {off:.4f} of the logits' norm")
    assert off < LIMIT["bf16"]


def test_release_frees_the_weights_and_changes_nothing():
    gen = torch.Generator(device="cuda").manual_seed(2)
    tokens = torch.randint(0, 512, (1, 40), generator=gen, device="cuda")
    a = run(build().quantize_projections_(), tokens, [33, 1, 6])
    model = build().quantize_projections_(release=True)
    assert model.model.layers[0].mlp.down_proj.weight.numel() == 0
    torch.testing.assert_close(run(model, tokens, [33, 1, 6]), a, rtol=0, atol=0)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("batch", [1, 3])
def test_device_plan_decodes_the_same_tokens(quantized, batch):
    from lastkv_b200.runner import GraphDecodeRunner

    model = build()
    if quantized:
        model.quantize_projections_()
    else:
        model.fuse_projections_()
    gen = torch.Generator(device="cuda").manual_seed(3)
    prompt = torch.randint(0, 512, (batch, 45), generator=gen, device="cuda")
    steps = 60  # boundaries at 64 and 96
    runs = []
    for device_plan in (False, True):
        cache = model.new_cache(batch, 45 + steps + 1)
        runner = GraphDecodeRunner(model, cache, device_plan=device_plan)
        with torch.no_grad():
            runner.prefill(prompt, 45)
            runner.capture()
            got = [runner.ids.clone()]
            for _ in range(steps - 1):
                got.append(runner.step().clone())
        cache.flush_commit()
        cache.check_errors()
        assert cache.committed == 96 and cache.seen_tokens == 45 + steps - 1
        runs.append((torch.cat(got, 1).cpu(), cache.pool_k.cpu(), cache.pool_v.cpu()))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_device_plan_follows_the_cache():
    from lastkv_b200.contract import RMarinBackendContractError
    from lastkv_b200.runner import GraphDecodeRunner

    model = build(layers=2)
    gen = torch.Generator(device="cuda").manual_seed(4)
    prompt = torch.randint(0, 512, (2, 30), generator=gen, device="cuda")
    out = []
    for device_plan in (False, True):
        cache = model.new_cache(2, 48)
        runner = GraphDecodeRunner(model, cache, device_plan=device_plan)
        with torch.no_grad():
            runner.prefill(prompt, 30)
            runner.capture()
            ids = [runner.step().clone() for _ in range(4)]
            logits, _ = model(prompt[:, :3], cache, logits_to_keep=1)  # a span between two graph steps
            runner.ids.copy_(logits[:, -1].float().argmax(-1, keepdim=True))
            ids += [runner.step().clone() for _ in range(48 - 37)]
            with pytest.raises(RMarinBackendContractError):
                runner.step()  # the cache is full
            cache.reserve(80)
            if device_plan:
                with pytest.raises(RMarinBackendContractError):
                    runner.step()  # planned for the smaller cache
        out.append(torch.cat(ids, 1).cpu())
    assert torch.equal(*out)


def test_refusals():
    from lastkv_b200.contract import RMarinBackendContractError

    with pytest.raises(RMarinBackendContractError):
        build(layers=1).quantize_projections_(activations="fp8")
    with pytest.raises(RMarinBackendContractError):
        build(layers=1).quantize_projections_(group=48)
    with pytest.raises(RMarinBackendContractError):
        build(layers=1).float().quantize_projections_()
    with pytest.raises(RMarinBackendContractError):
        build(layers=1).cpu().quantize_projections_()
