"""Beam search and the 8-bit history inside the model: selection, shared pages, commits, captured steps."""

import numpy as np
import pytest
import torch

from lastkv_b200 import ops
from lastkv_b200.contract import RMarinBackendContractError as Refused
from lastkv_b200.hf import LastKVConfig, LastKVForCausalLM
from lastkv_b200.runner import GraphDecodeRunner, init_random_

pytestmark = pytest.mark.gpu


def _model(dtype, seed=3, **kw):
    cfg = LastKVConfig(**(dict(hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=2,
                               num_hidden_layers=3, head_dim=64, vocab_size=512, chunk_size=32) | kw))
    model = LastKVForCausalLM(cfg).cuda().to(dtype).eval()
    init_random_(model, std=0.06, seed=seed)
    return model


def _prompt(B, n, seed=1, vocab=512):
    return torch.randint(0, vocab, (B, n), generator=torch.Generator().manual_seed(seed)).cuda()


@torch.no_grad()
def _log_probs(model, seqs, **cache):
    """log p(next) at every position of [N, T] sequences, by one run without beams."""
    c = model.new_cache(seqs.shape[0], seqs.shape[1], **cache)
    logits, _ = model(seqs, c)
    c.check_errors()
    return torch.log_softmax(logits.double(), -1)


def _plain_beams(model, prompt, K, new, eos=None):
    """Beam search that runs every beam from its first token in each step, in fp32, with 64-bit totals."""
    B, P = prompt.shape
    seqs, scores, done = prompt[:, None], torch.zeros((B, 1), dtype=torch.float64, device="cuda"), None
    for _ in range(new):
        n = seqs.shape[1]
        logp = _log_probs(model, seqs.reshape(B * n, -1))[:, -1].view(B, n, -1)
        total = scores[..., None] + logp
        if done is not None and eos is not None:
            alone = torch.full_like(total, float("-inf"))
            alone[..., eos] = scores
            total = torch.where(done[..., None], alone, total)
        best, at = total.view(B, -1).sort(dim=-1, descending=True, stable=True)
        beam, token = at[:, :K] // total.shape[-1], at[:, :K] % total.shape[-1]
        gap = (best[:, :K] - best[:, 1:K + 1]).min().item()
        seqs = torch.cat((seqs.gather(1, beam[..., None].expand(-1, -1, seqs.shape[-1])), token[..., None]), -1)
        ended = token == (-1 if eos is None else eos)
        done = ended if done is None else ended | done.gather(1, beam)
        scores = best[:, :K]
        assert gap > 1e-5, "candidates too close for two orders of summation: another seed"
    return seqs, scores, done


@pytest.mark.parametrize("B,K,P,new", [(1, 4, 20, 30), (2, 3, 33, 40), (3, 2, 31, 36)])
def test_beam_search_matches_running_every_beam_from_the_start(B, K, P, new):
    """fp32, over several chunk boundaries (32 tokens): the same sequences; scores within the rounding of two ways to
    compute them (the fp32 model's logits agree to 1e-5 relative, and a score sums `new` of them)."""
    model = _model(torch.float32)
    prompt = _prompt(B, P, seed=K)
    want, scores, _ = _plain_beams(model, prompt, K, new)
    got = model.generate_beam(prompt, K, new)
    assert torch.equal(got.sequences, want)
    assert float((got.scores.double() - scores).abs().max()) <= 1e-4 * new


def test_beams_that_end():
    model = _model(torch.float32, seed=5)
    prompt = _prompt(2, 12, seed=9)
    first = model.generate_beam(prompt, 3, 6)
    eos = int(first.sequences[0, 0, 14])  # a token that beams do choose
    want, scores, done = _plain_beams(model, prompt, 3, 20, eos)
    got = model.generate_beam(prompt, 3, 20, eos_token=eos)
    n = got.sequences.shape[-1]
    assert torch.equal(got.sequences, want[..., :n]) and torch.equal(got.finished, done)
    assert bool(got.finished.any()) and (n == 32 or bool(got.finished.all()))
    assert float((got.scores.double() - scores).abs().max()) <= 1e-4 * 20


@pytest.mark.parametrize("history", [None, "int8"])
def test_scores_are_those_of_the_sequences(history):
    """bf16: a beam's score is the sum of its tokens' log-probabilities when its sequence is run alone, up to bf16
    logits of two batch sizes and kernels (a half step of logits below 8 is 2^-6; `new` tokens, each with two of them)."""
    model = _model(torch.bfloat16)
    prompt = _prompt(2, 45, seed=4)
    new, K = 60, 4
    cache = model.new_cache(2 * K, 45 + new, history=history)
    got = model.generate_beam(prompt, K, new, cache=cache)
    cache.check_errors()
    seqs = got.sequences.view(2 * K, -1)
    logp = _log_probs(model, seqs, history=history)
    own = logp[:, 44:-1].gather(-1, seqs[:, 45:, None])[..., 0].sum(-1).view(2, K)
    assert float((own - got.scores).abs().max()) <= new * 2 * 2.0 ** -6
    assert bool((got.scores[:, :-1] >= got.scores[:, 1:]).all())


@pytest.mark.parametrize("history", [None, "int8"])
def test_captured_steps_choose_what_eager_ones_do(history):
    """The runner's captured beam steps against the same steps run eagerly over an equal cache: same candidates."""
    model = _model(torch.bfloat16, seed=7)
    B, K, P, steps = 2, 4, 40, 70
    prompt = _prompt(B, P, seed=6)
    cache = model.new_cache(B * K, P + steps + 1, history=history)
    runner = GraphDecodeRunner(model, cache, beams=K, eos_token=7)
    with torch.no_grad():
        runner.prefill(prompt, 24)
        runner.capture()
        eager = model.new_cache(B * K, P + steps + 1, history=history)
        with eager.only_rows(np.arange(0, B * K, K)):
            for s in range(0, P, 24):
                logits, _ = model(prompt[:, s:s + 24], eager, logits_to_keep=1)
        best = ops.beam_select(logits[:, -1], torch.zeros((B, 1), device="cuda"), select=K, eos_token=7)
        eager.reorder_cache(np.repeat(np.arange(0, B * K, K), K))
        assert torch.equal(runner.ids, best.tokens.view(-1, 1))
        for step in range(steps):
            logits, _ = model(best.tokens.view(-1, 1), eager, logits_to_keep=1)
            best = ops.beam_select(logits[:, -1], best.scores, finished=best.finished, eos_token=7)
            eager.reorder_cache(best.rows)
            runner.step()
            assert torch.equal(runner.choice.rows, best.rows) and torch.equal(runner.choice.tokens, best.tokens), step
            assert torch.equal(runner.choice.scores, best.scores)
    cache.check_errors()
    eager.check_errors()


def test_8_bit_history_is_the_bf16_one_rounded():
    """Prefill spans and decode steps over several chunks.  Against a bf16 cache whose history pages are replaced by
    what the 8-bit ones stand for: the model's bf16 tolerance (relative L2 2e-2)."""
    model = _model(torch.bfloat16, seed=11, head_dim=128, num_attention_heads=4, num_key_value_heads=1)
    B, T = 3, 230
    tokens = _prompt(B, T, seed=12)
    q8, ref = model.new_cache(B, T, history="int8"), model.new_cache(B, T)
    ids = torch.arange(B * q8.pages_per_seq, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        at = 0
        for n in (50, 1, 30, 40, 3, 1, 1, 32, 60, 1, 1, 10):
            a, _ = model(tokens[:, at:at + n], q8)
            b, _ = model(tokens[:, at:at + n], ref)
            at += n
            if ref.committed:
                ref.flush_commit()
                pages = torch.from_numpy(ref.src_table[:, : ref.committed // 16].copy()).cuda()
                old = torch.from_numpy(q8.src_table[:, : ref.committed // 16].copy()).cuda()
                ops.dequantize_pages(q8.q8, old.reshape(-1), ref.pool_k, ref.pool_v, pages.reshape(-1))
            rel = float((a.double() - b.double()).norm() / b.double().norm())
            assert rel <= 2e-2, (at, rel)
    assert at == T and q8.committed == 224
    q8.check_errors()
    assert ids.numel() == q8.q8.num_pages


def test_rows_taken_in_turns_give_the_same():
    """A stage for all rows, for one, and for two at a time."""
    model = _model(torch.bfloat16, seed=13)
    tokens = _prompt(3, 150, seed=14)
    outs = []
    for limit in (1 << 30, 1, 2 * 2 * 2 * 16 * 2 * 64 * 6):
        cache = model.new_cache(3, 150, history="int8")
        cache.stage_bytes = limit
        with torch.no_grad():
            outs.append(model(tokens, cache)[0])
        cache.check_errors()
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


def test_8_bit_history_in_the_greedy_runner_and_after_growing():
    model = _model(torch.bfloat16, seed=15)
    prompt = _prompt(2, 70, seed=16)
    runs = []
    for tokens in (170, 80):
        cache = model.new_cache(2, tokens, history="int8")
        with torch.no_grad():
            if tokens == 80:
                model(prompt[:, :50], cache)
                cache.reserve(170)
                runner = GraphDecodeRunner(model, cache)
                runner.prefill(prompt[:, 50:], 64)
            else:
                runner = GraphDecodeRunner(model, cache)
                runner.prefill(prompt[:, :50], 64)
                runner.prefill(prompt[:, 50:], 64)
            runner.capture()
            out = [runner.ids.clone()]
            for _ in range(90):
                out.append(runner.step().clone())
        cache.check_errors()
        assert cache.committed == 160 or cache.committed == 128
        runs.append(torch.cat(out, 1))
    assert torch.equal(runs[0], runs[1])


def test_device_planned_steps_after_a_reorder():
    """A runner that plans on the device goes on with rows of their own after the cache was reordered, as one that
    plans on the host does with shared ones."""
    model = _model(torch.bfloat16, seed=17)
    prompt = _prompt(3, 50, seed=18)
    runs = []
    for device_plan in (False, True):
        cache = model.new_cache(3, 150)
        runner = GraphDecodeRunner(model, cache, device_plan=device_plan)
        with torch.no_grad():
            runner.prefill(prompt, 64)
            runner.capture()
            out = []
            for i in range(60):
                out.append(runner.step().clone())
                if i % 13 == 5:
                    order = torch.tensor([2, 0, 0], device="cuda")
                    cache.reorder_cache(order)
                    runner.ids.copy_(runner.ids[order])
        cache.check_errors()
        runs.append(torch.cat(out, 1))
    assert torch.equal(runs[0], runs[1])


@pytest.mark.parametrize("history", [None, "int8"])
def test_a_captured_step_is_refused_after_the_cache_has_grown(history):
    """The graphs hold the addresses of the memory that they were captured over."""
    model = _model(torch.bfloat16)
    cache = model.new_cache(2, 100, history=history)
    runner = GraphDecodeRunner(model, cache)
    with torch.no_grad():
        runner.prefill(_prompt(2, 40), 64)
        runner.capture()
        first = runner.step().clone()
        cache.reserve(110)  # the same number of pages
        with pytest.raises(Refused, match="grown"):
            runner.step()
        again = GraphDecodeRunner(model, cache)
        again.ids.copy_(first)
        again.capture()
        again.step()
    cache.check_errors()


def test_refused_calls():
    model = _model(torch.bfloat16)
    cache = model.new_cache(4, 64, history="int8")
    with pytest.raises(Refused, match="device"):
        GraphDecodeRunner(model, cache, device_plan=True)
    with pytest.raises(Refused, match="device"):
        GraphDecodeRunner(model, model.new_cache(4, 64), device_plan=True, beams=2)
    with pytest.raises(Refused, match="beams"):
        GraphDecodeRunner(model, cache, beams=3)
    with pytest.raises(Refused, match="rows"):
        model.generate_beam(_prompt(3, 4), 2, 5, cache=cache)
    with pytest.raises(Refused, match="a beam"):
        model.generate_beam(_prompt(2, 4), 0, 5)
    with pytest.raises(Refused, match="32 at most"):
        model.generate_beam(_prompt(1, 4), 33, 5)
    with pytest.raises(Refused, match="a prompt"):
        model.generate_beam(_prompt(2, 0), 2, 5)
    with pytest.raises(Refused, match="at least one"):
        model.generate_beam(_prompt(2, 4), 2, 0, cache=cache)
