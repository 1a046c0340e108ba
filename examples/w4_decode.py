"""Greedy decoding with 4-bit projection weights and steps planned on the device.

    python examples/w4_decode.py                    # a small model: 4-bit against bf16
    python examples/w4_decode.py --size 8b          # the 8B architecture, batch 8, 2048 prompt tokens

Random weights (no checkpoint is needed).  The same prompt is prefilled and decoded by the bf16 model (fused
projections, host-planned graph steps) and by the model with 4-bit projections (int8 rows between the kernels,
device-planned graph steps: one graph launch per token and nothing copied from the host).
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from lastkv_b200.hf import LastKVConfig, LastKVForCausalLM  # noqa: E402
from lastkv_b200.runner import GraphDecodeRunner, init_random_  # noqa: E402

SIZES = {
    "small": dict(hidden_size=768, intermediate_size=2048, num_attention_heads=12, num_key_value_heads=12,
                  num_hidden_layers=12, head_dim=64, vocab_size=32000, chunk_size=128),
    "8b": dict(hidden_size=4096, intermediate_size=14336, num_attention_heads=32, num_key_value_heads=8,
               num_hidden_layers=32, head_dim=128, vocab_size=128256, chunk_size=1024, rope_theta=500000.0),
}


def build(size: str) -> LastKVForCausalLM:
    with torch.device("meta"):
        model = LastKVForCausalLM(LastKVConfig(**SIZES[size]))
    model = model.to(torch.bfloat16).to_empty(device="cuda").eval()
    init_random_(model, seed=1)
    return model


@torch.no_grad()
def decode(model, prompt, steps: int, device_plan: bool):
    cache = model.new_cache(prompt.shape[0], prompt.shape[1] + steps + 8)
    runner = GraphDecodeRunner(model, cache, device_plan=device_plan)
    start, mid, end = (torch.cuda.Event(enable_timing=True) for _ in range(3))
    start.record()
    runner.prefill(prompt, 2048)
    mid.record()
    runner.capture()
    ids = [runner.ids.clone()]
    for _ in range(4):  # warm-up steps
        ids.append(runner.step().clone())
    torch.cuda.synchronize()
    prefill_ms = start.elapsed_time(mid)
    start.record()
    for _ in range(steps):
        ids.append(runner.step().clone())
    end.record()
    torch.cuda.synchronize()
    cache.check_errors()
    return torch.cat(ids, 1), prefill_ms, start.elapsed_time(end) / steps


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--size", choices=sorted(SIZES), default="small")
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--group", type=int, default=128)
    ap.add_argument("--activations", choices=["int8", "bf16"], default="int8")
    a = ap.parse_args()
    model = build(a.size)
    prompt = torch.randint(0, SIZES[a.size]["vocab_size"], (a.batch, a.prompt), device="cuda")
    model.fuse_projections_()
    decode(model, prompt, 2, False)  # loads the kernels
    ids, prefill, step = decode(model, prompt, a.steps, False)
    print(f"bf16:  prefill {prefill:8.2f} ms   step {step:7.3f} ms   {a.batch / step * 1e3:8.0f} tokens/s")
    model.quantize_projections_(a.group, a.activations, release=True)
    torch.cuda.empty_cache()
    decode(model, prompt, 2, True)
    ids4, prefill, step = decode(model, prompt, a.steps, True)
    print(f"4-bit: prefill {prefill:8.2f} ms   step {step:7.3f} ms   {a.batch / step * 1e3:8.0f} tokens/s   "
          f"({(ids == ids4).float().mean().item():.0%} of the tokens are the bf16 model's)")


if __name__ == "__main__":
    main()
