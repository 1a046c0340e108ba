"""Host side of beam search's cache: shared tables, pages that rows write, refused calls."""

import numpy as np
import pytest
import torch

from lastkv_b200.contract import RMarinBackendContractError as Refused
from lastkv_b200.hf import LastKVConfig, PagedLastKVCache


def _cache(batch, tokens, **kw):
    cfg = LastKVConfig(hidden_size=64, intermediate_size=96, num_attention_heads=4, num_key_value_heads=2,
                       num_hidden_layers=2, head_dim=64, vocab_size=50, chunk_size=32)
    return PagedLastKVCache(cfg, batch, tokens, device="cpu", **({"dtype": torch.float32} | kw))


def _advance(cache, n, tag):
    """Write n tokens to every row the way the append kernel does, each with a number of its own in every place."""
    for _ in range(n):
        h = cache.plan_host(1)
        B = len(h["ring_tok"])
        flat = cache.pool_k.view(-1, cache.hkv, cache.d)
        for b in range(B):
            mark = tag(b, cache.seen_tokens)
            for l in range(cache.num_layers):
                flat[int(h["ring_tok"][b]) + int(cache.ring_base[l]) * 16] = mark
            flat[int(h["src_tok"][b])] = mark
        cache.advance(1)
        if cache.seen_tokens % cache.chunk_size == 0:
            cache.committed = cache.seen_tokens  # (no blend: the marks stay)


def _seen(cache, b):
    """What row b's attention would read in layer 1: the marks of all its keys."""
    h = cache.plan_host(1)
    flat = cache.pool_k.view(-1, cache.hkv, cache.d)
    marks = []
    for j in range(h["W"]):
        page = int(h["bt"][b, j]) + (int(cache.ring_base[1]) if j >= h["nsrc"] else 0)
        marks += flat[page * 16: page * 16 + 16, 0, 0].tolist()
    return marks[: h["seq_k"] - 1]


def test_rows_follow_their_parents():
    """Random reorders between random numbers of tokens, over several chunks: every row reads what its ancestors wrote."""
    rng = np.random.default_rng(0)
    B = 5
    cache = _cache(B, 200)
    history = [[] for _ in range(B)]
    step = 0
    while cache.seen_tokens < 190:
        n = int(rng.integers(1, 24))
        n = min(n, 190 - cache.seen_tokens)
        base = step * 1000
        first = cache.seen_tokens
        _advance(cache, n, lambda b, pos: base + b * 100 + (pos - first) % 100)
        for b in range(B):
            history[b] = history[b] + [float(base + b * 100 + i % 100) for i in range(n)]
        idx = rng.integers(0, B, B)
        cache.reorder_cache(torch.from_numpy(idx))
        history = [list(history[i]) for i in idx]
        step += 1
        if cache.seen_tokens < 200:
            for b in range(B):
                want = history[b]
                got = _seen(cache, b)
                assert got == want, (cache.seen_tokens, b)
    # a page is written by one row only
    h = cache.plan_host(1)
    assert len(set(h["ring_tok"].tolist())) == B and len(set(h["src_tok"].tolist())) == B


def test_unshare_gives_every_row_pages_of_its_own():
    cache = _cache(3, 120)
    _advance(cache, 50, lambda b, pos: b * 1000 + pos)
    before = [_seen(cache, b) for b in (2, 0, 0)]
    assert not cache.shared
    cache.reorder_cache(torch.tensor([2, 0, 0]))
    assert cache.shared
    _advance(cache, 7, lambda b, pos: 5000 + b * 1000 + pos)
    after = [_seen(cache, b) for b in range(3)]
    assert [a[:50] for a in after] == before
    cache.unshare_()
    assert not cache.shared and [_seen(cache, b) for b in range(3)] == after
    cache.reserve(300)
    assert [_seen(cache, b) for b in range(3)] == after


def test_spans_of_some_rows():
    cache = _cache(4, 100)
    with cache.only_rows([0, 2]):
        _advance(cache, 40, lambda b, pos: b * 1000 + pos)
        assert cache.plan_host(3)["bt"].shape[0] == 2
    cache.reorder_cache(np.array([0, 0, 2, 2]))
    got = [_seen(cache, b) for b in range(4)]
    assert got[0] == got[1] == [float(p) for p in range(40)] and got[2] == got[3] == [1000.0 + p for p in range(40)]


def test_8_bit_history_lays_out_its_raw_ring_in_front():
    cache = _cache(2, 100, dtype=torch.bfloat16, history="int8")
    assert cache.q8.num_pages == 2 * 7 and cache.src_pages == cache.ring_stride
    assert cache.num_pages == 3 * cache.ring_stride  # no bf16 page for the history
    h = cache.plan_host(5)
    assert h["src_tok"].tolist() == h["ring_tok"].tolist()
    cache.seen_tokens = 90
    h = cache.plan_host(2)
    assert h["nsrc"] == 2 and h["bt"][1, :2].tolist() == [7, 8]  # two finished chunks back: one chunk older
    codes = cache.q8.codes
    codes.copy_(torch.randint(1, 256, codes.shape).to(torch.uint8))
    was = [cache.q8.codes[cache.src_table[b]].clone() for b in range(2)]
    cache.reserve(300)
    assert cache.q8.num_pages == 2 * 19
    for b in range(2):
        assert torch.equal(cache.q8.codes[cache.src_table[b, :7]], was[b])


def test_refused_calls():
    with pytest.raises(Refused, match="history"):
        _cache(1, 32, history="int4", dtype=torch.bfloat16)
    with pytest.raises(Refused, match="bf16"):
        _cache(1, 32, history="int8")
    cache = _cache(4, 64)
    for idx in ([0, 1, 2], [0, 1, 2, 4], [-1, 0, 0, 0]):
        with pytest.raises(Refused, match="beam_idx"):
            cache.reorder_cache(torch.tensor(idx))
    for rows in ([], [0, 0], [4]):
        with pytest.raises(Refused, match="rows"):
            with cache.only_rows(rows):
                pass
