"""Greedy decoding and beam search over a history in 8 bits.

    python examples/q8_history.py                               # a small model
    python examples/q8_history.py --size 8b --batch 32 --prompt 8192

Random weights (no checkpoint is needed).  The same prompts are decoded greedily with a bf16 history and with one in
8 bits, and then by beam search, each prompt's beams sharing the pages of what they have in common.
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from examples.w4_decode import SIZES, build  # noqa: E402
from lastkv_b200.runner import GraphDecodeRunner  # noqa: E402


@torch.no_grad()
def decode(model, prompt, steps: int, *, history=None, beams: int | None = None):
    """(new tokens [rows, 5 + steps], GB of keys and values, prefill ms, ms per step)."""
    rows = prompt.shape[0] * (beams or 1)
    cache = model.new_cache(rows, prompt.shape[1] + steps + 8, history=history)
    held = [cache.pool_k, cache.pool_v] + (list(cache.q8) if cache.q8 is not None else [])
    runner = GraphDecodeRunner(model, cache, beams=beams)
    start, mid, end = (torch.cuda.Event(enable_timing=True) for _ in range(3))
    start.record()
    runner.prefill(prompt, 2048)
    mid.record()
    runner.capture()
    out = runner.ids.clone()
    for i in range(4 + steps):
        if i == 4:  # after the warm-up steps
            torch.cuda.synchronize()
            prefill_ms = start.elapsed_time(mid)
            start.record()
        ids = runner.step()
        out = torch.cat((out if beams is None else out[runner.choice.rows.view(-1)], ids), 1)
    end.record()
    torch.cuda.synchronize()
    cache.check_errors()
    return out, sum(t.nbytes for t in held) / 1e9, prefill_ms, start.elapsed_time(end) / steps


def main(argv=None) -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--size", choices=sorted(SIZES), default="small")
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--beams", type=int, default=4)
    a = ap.parse_args(argv)
    model = build(a.size)
    model.fuse_projections_()
    prompt = torch.randint(0, SIZES[a.size]["vocab_size"], (a.batch, a.prompt), device="cuda")
    few = prompt[: max(1, a.batch // a.beams)]
    decode(model, prompt[:1], 2)  # loads the kernels
    for history in (None, "int8"):
        _, gb, prefill, step = decode(model, prompt, a.steps, history=history)
        print(f"{history or 'bf16'} history: {gb:6.2f} GB   prefill {prefill:8.1f} ms   step {step:7.3f} ms   "
              f"{a.batch / step * 1e3:8.0f} tokens/s")
    for history in (None, "int8"):
        _, gb, prefill, step = decode(model, few, a.steps, history=history, beams=a.beams)
        print(f"{history or 'bf16'} history, {few.shape[0]} x {a.beams} beams: {gb:6.2f} GB   prefill {prefill:8.1f} ms   "
              f"step {step:7.3f} ms")


if __name__ == "__main__":
    main()
