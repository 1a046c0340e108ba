"""What is not a number stays visible in the attention of spans, however the keys are split, and a token that sees no
key gives zeros."""

import pytest
import torch

from lastkv_b200 import ops
from tests.q8_helpers import random_cache

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
LENS, SPANS, NUM_Q8 = [1200, 500, 300], [3, 130, 300], [60, 31, 5]


def _case(seed=31, hq=4, hkv=2, d=64):
    t = random_cache(seed, LENS, NUM_Q8, hkv, d)
    cu = torch.tensor([0] + SPANS).cumsum(0).int().cuda()
    q = torch.randn((int(cu[-1]), hq, d), generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
    return t, q, cu


def _run(t, q, cu, splits, causal=True):
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")
    cache = ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])
    out = ops.prefill_paged_q8(q, cache, t["table"], t["seq_k"], cu, max(SPANS), num_q8=t["num_q8"], lse=lse,
                               pool_k=t["pool_k"], pool_v=t["pool_v"], causal=causal, kv_splits=splits, error_word=err)
    assert err.tolist() == [0, 0, 0, 0]
    return out, lse


@pytest.mark.parametrize("splits", [1, 2, 8])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("scales,value", [("ks", NAN), ("ks", INF), ("vs", NAN), ("vs", INF)])
def test_blocks_that_are_not_finite(splits, causal, scales, value):
    t, q, cu = _case()
    clean, clean_lse = _run(t, q, cu, splits, causal)
    assert bool(clean.isfinite().all()) and bool(clean_lse.isfinite().all())
    t[scales][int(t["table"][0, 2]), 1] = value  # tokens 40-47 of row 0, which all of its span sees
    t[scales][int(t["table"][1, 20]), 0] = value  # tokens 320-327 of row 1, likewise
    out, lse = _run(t, q, cu, splits, causal)
    assert bool(out[:133].isnan().all()) and bool(lse[:133].isnan().all())
    assert torch.equal(out[133:], clean[133:]) and torch.equal(lse[133:], clean_lse[133:])


@pytest.mark.parametrize("splits", [1, 2, 8])
def test_queries_and_bf16_values_that_are_not_numbers(splits):
    t, q, cu = _case()
    clean, clean_lse = _run(t, q, cu, splits)
    q[7, 2] = NAN  # one head of a token of row 1
    t["pool_v"][int(t["table"][0, 70]), 3] = NAN  # a value of row 0 that its span sees
    out, lse = _run(t, q, cu, splits)
    assert bool(out[:3].isnan().all())
    assert torch.equal(lse[:3], clean_lse[:3])  # the weights are numbers
    assert bool(out[7, 2].isnan().all()) and bool(lse[7, 2].isnan())
    rest = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    rest[:3], rest[7, 2] = False, False
    assert torch.equal(out[rest], clean[rest]) and torch.equal(lse[rest], clean_lse[rest])


@pytest.mark.parametrize("splits", [1, 4])
def test_bf16_pages_that_are_not_finite(splits):
    g = torch.Generator().manual_seed(5)
    pool_k, pool_v = (torch.randn((70, 16, 2, 64), generator=g).bfloat16().cuda() for _ in range(2))
    table = torch.randperm(70, generator=g).int().view(1, 70).cuda()
    q = torch.randn((40, 4, 64), generator=g).bfloat16().cuda()
    cu, seq = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 40], [1100]))
    pool_k[int(table[0, 9]), 5, 1] = NAN  # heads 2 and 3
    lse = torch.empty((40, 4), device="cuda")
    out = ops.prefill_paged(q, pool_k, pool_v, table, seq, cu, 40, causal=False, kv_splits=splits, lse=lse)
    assert bool(out[:, 2:].isnan().all()) and bool(lse[:, 2:].isnan().all())
    assert bool(out[:, :2].isfinite().all()) and bool(lse[:, :2].isfinite().all())


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("num_q8", [0, 9])
def test_tokens_that_see_no_key(splits, num_q8):
    """A causal span longer than its keys: the tokens in front see none, beside tokens of the same tile that do."""
    t = random_cache(33, [20], [num_q8], 2, 64)
    q = torch.randn((50, 4, 64), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    cu = torch.tensor([0, 50], dtype=torch.int32, device="cuda")
    cache = ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])
    lse = torch.empty((50, 4), device="cuda")
    out = ops.prefill_paged_q8(q, cache, t["table"], t["seq_k"], cu, 50, num_q8=t["num_q8"], pool_k=t["pool_k"],
                               pool_v=t["pool_v"], kv_splits=splits, lse=lse)
    assert bool((out[:30] == 0).all()) and bool((lse[:30] == -INF).all())
    assert bool((out[30:] != 0).any(-1).all()) and bool(lse[30:].isfinite().all())
    if not num_q8:
        out = ops.prefill_paged(q, t["pool_k"], t["pool_v"], t["table"], t["seq_k"], cu, 50, lse=lse)
        assert bool((out[:30] == 0).all()) and bool((lse[:30] == -INF).all())


@pytest.mark.parametrize("parts", [2, 5, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_merging_parts(parts, d):
    """A part whose log-sum-exp is NaN makes the row NaN; one of -inf counts for nothing, whatever it holds."""
    g = torch.Generator().manual_seed(parts)
    o = torch.randn((parts, 4, 2, d), generator=g).cuda()
    lse = torch.randn((parts, 4, 2), generator=g).cuda()
    got_lse = torch.empty((4, 2), device="cuda")
    clean = ops.merge_partials(o, lse)
    lse[1, 0, 1] = NAN
    lse[:, 1, 0] = -INF
    lse[0, 1, 0], o[0, 1, 0] = NAN, NAN      # nothing but NaN and parts without a key
    lse[0, 2, 1], o[0, 2, 1] = -INF, NAN
    lse[:, 3, 1] = -INF
    out = ops.merge_partials(o, lse, lse_out=got_lse)
    for row, head in ((0, 1), (1, 0)):
        assert bool(out[row, head].isnan().all()) and bool(got_lse[row, head].isnan())
    assert bool(out[2, 1].isfinite().all()) and bool(got_lse[2, 1].isfinite())
    assert bool((out[3, 1] == 0).all()) and float(got_lse[3, 1]) == -INF
    for row, head in ((0, 0), (1, 1), (2, 0), (3, 0)):
        assert torch.equal(out[row, head], clean[row, head])


@pytest.mark.parametrize("d", [64, 128])
def test_combining_ranks(d):
    """The combine of one rank is the merge of one part, also where that part is NaN."""
    rows = 4
    sizes = ops.cp_combine_sizes(rows, d, 1)
    o = torch.randn((rows, d), generator=torch.Generator().manual_seed(2)).cuda()
    lse = torch.tensor([0.5, NAN, -INF, 2.0], device="cuda")
    o[2] = NAN
    send = torch.zeros(sizes["send_floats"], device="cuda")
    send[: rows * d], send[rows * d: rows * (d + 1)] = o.flatten(), lse
    recv = torch.zeros(sizes["recv_words"], dtype=torch.int64, device="cuda")
    state = torch.zeros(2, dtype=torch.int32, device="cuda")
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    got = ops.cp_combine(send, [recv.data_ptr()], 0, 1, state, rows, d, 4, error_word=err).view(rows, d)
    assert bool(got[1].isnan().all()) and bool((got[2] == 0).all())
    assert torch.equal(got[[0, 3]], o[[0, 3]].bfloat16()) and err.tolist() == [0, 0, 0, 0]
