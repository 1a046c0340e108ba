"""Whether rows share pages is known without comparing tables for a cache that was never reordered."""

import numpy as np
import pytest
import torch

from lastkv_b200.hf import LastKVConfig, PagedLastKVCache


def _cache(**kw):
    cfg = LastKVConfig(hidden_size=64, intermediate_size=96, num_attention_heads=4, num_key_value_heads=2,
                       num_hidden_layers=2, head_dim=64, vocab_size=50, chunk_size=32)
    return PagedLastKVCache(cfg, 3, 150, device="cpu", **({"dtype": torch.float32} | kw))


@pytest.mark.parametrize("kw", [{}, {"dtype": torch.bfloat16, "history": "int8"}])
def test_no_table_is_compared_before_a_reorder(kw, monkeypatch):
    cache = _cache(**kw)
    cache.plan_host(20)
    cache.advance(20)
    compared = []
    equal = np.array_equal
    monkeypatch.setattr(np, "array_equal", lambda *a, **k: compared.append(a) or equal(*a, **k))
    assert not cache.shared
    cache.unshare_()
    cache.reserve(200)
    assert not cache.shared and not compared
    cache.reorder_cache([1, 1, 0])
    assert cache.shared and compared
    del compared[:]
    cache.unshare_()
    assert not cache.shared
    del compared[:]
    assert not cache.shared and not compared


def test_shared_ends_when_the_pages_do():
    """Rows that share pages of their rings alone (an 8-bit history before its first chunk is finished) no longer do
    when those have been written again."""
    cache = _cache(dtype=torch.bfloat16, history="int8")
    cache.plan_host(20)
    cache.advance(20)
    cache.reorder_cache([2, 0, 0])
    assert cache.shared  # one full page of the raw ring
    for n in (12, 32, 32, 32):
        cache.plan_host(n)
        cache.advance(n)
    assert not cache.shared
    cache.reserve(400)
    assert not cache.shared
