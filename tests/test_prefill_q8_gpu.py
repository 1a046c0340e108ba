"""Attention of spans of tokens over 8-bit and bf16 pages against its formula in 64 bits."""

import pytest
import torch

from lastkv_b200 import ops
from tests.q8_helpers import assert_within, attention, random_cache, row_keys

pytestmark = pytest.mark.gpu

# a quarter of the exponentials is a polynomial: relative error 7.5e-5 (ex2_poly2)
POLY = 7.5e-5


def _case(seed, lens, spans, num_q8, hq, hkv, d, **kw):
    t = random_cache(seed, lens, num_q8, hkv, d, **kw)
    g = torch.Generator().manual_seed(seed)
    cu = torch.tensor([0] + spans).cumsum(0).int().cuda()
    q = torch.randn((int(cu[-1]), hq, d), generator=g).bfloat16().cuda()
    return t, q, cu


def _run(t, q, cu, **kw):
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    cache = ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])
    top = int((cu[1:] - cu[:-1]).max())
    kw = dict(num_q8=t["num_q8"], pool_k=t["pool_k"], pool_v=t["pool_v"], error_word=err) | kw
    out = ops.prefill_paged_q8(q, cache, t["table"], t["seq_k"], cu, top, **kw)
    if kw["error_word"] is not None:
        assert err.tolist() == [0, 0, 0, 0]
    return out


def _check(t, q, cu, out, causal=True):
    c = cu.tolist()
    for b in range(len(c) - 1):
        k, v = row_keys(t, b)
        span = q[c[b]:c[b + 1]]
        ref, bound = attention(span, k, v, q.shape[2] ** -0.5, k.shape[0] - span.shape[0] if causal else None, POLY)
        assert_within(out[c[b]:c[b + 1]], ref, bound, f"row {b}")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (4, 2), (8, 2), (8, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_spans_over_both_kinds_of_pages(d, hq, hkv, causal):
    """Spans of one token to several tiles; pages that end inside; spans that end, begin and lie in 8-bit pages."""
    lens = [1, 40, 129, 300, 700, 333, 16, 530]
    spans = [1, 40, 1, 260, 37, 333, 0, 129]
    num_q8 = [0, 3, 2, 5, 43, 99, 1, 1]
    t, q, cu = _case(hq + d, lens, spans, num_q8, hq, hkv, d)
    _check(t, q, cu, _run(t, q, cu, causal=causal), causal)


def test_no_page_and_every_page_in_8_bits():
    for num_q8 in ([0, 0], [99, 99]):
        t, q, cu = _case(5, [200, 75], [100, 75], num_q8, 4, 2, 64)
        out = _run(t, q, cu)
        _check(t, q, cu, out)
        if num_q8[0]:
            assert torch.equal(out, _run(t, q, cu, num_q8=None, pool_k=None, pool_v=None))
        else:  # as the bf16 call, up to the exponentials that take the polynomial
            ref = ops.prefill_paged(q, t["pool_k"], t["pool_v"], t["table"], t["seq_k"], cu, 100)
            _check(t, q, cu, ref)


def test_stage_shared_by_calls_and_wider_than_needed():
    t, q, cu = _case(6, [400, 90], [64, 10], [20, 3], 8, 2, 128)
    W = t["table"].shape[1]
    stage = ops.StageQ8.empty(2, W + 5, 2, 128)
    a = _run(t, q, cu, stage=stage)
    _check(t, q, cu, a)
    b = _run(t, q.flip(1), cu, stage=stage, staged=True)
    _check(t, q.flip(1), cu, b)
    narrow = ops.StageQ8.empty(2, 20, 2, 128)
    assert torch.equal(a, _run(t, q, cu, stage=narrow))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("splits", [2, 3, 8])
def test_splits_of_the_keys(causal, splits):
    """Splits that end inside both kinds of pages, splits without a key that a token sees, rows of a single block."""
    t, q, cu = _case(13, [700, 40, 333, 1], [130, 40, 300, 1], [30, 1, 4, 0], 4, 2, 64)
    lse = torch.empty((471, 4), dtype=torch.float32, device="cuda")
    one = torch.empty_like(lse)
    out = _run(t, q, cu, causal=causal, kv_splits=splits, lse=lse)
    _check(t, q, cu, out, causal)
    _run(t, q, cu, causal=causal, kv_splits=1, lse=one)
    assert float((lse - one).abs().max()) <= 4 * POLY  # both have their weights' errors
    work = torch.empty((9, 471 * 4, 64), device="cuda"), torch.empty((9, 471 * 4), device="cuda")
    assert torch.equal(out, _run(t, q, cu, causal=causal, kv_splits=splits, partials=work))


def test_a_row_with_more_pages_than_the_stage_is_reported():
    t, q, cu = _case(7, [400, 90], [64, 10], [20, 3], 4, 2, 64)
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    cache = ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])
    out = ops.prefill_paged_q8(q, cache, t["table"], t["seq_k"], cu, 64, num_q8=t["num_q8"], pool_k=t["pool_k"],
                               pool_v=t["pool_v"], stage=ops.StageQ8.empty(2, 7, 2, 64), error_word=err)
    assert err[0] == 2 and bool(out.isfinite().all())
    _check({n: x[1:] if n in ("table", "num_q8", "seq_k") else x for n, x in t.items()}, q[64:], cu[1:] - 64, out[64:])


def test_blocks_that_a_token_does_not_see_leave_it_alone():
    """Infinite scales in 8-bit blocks behind a span's tokens: the tokens before them are as they were, and
    those that see them are not numbers."""
    t, q, cu = _case(8, [64, 160], [64, 64], [99, 99], 4, 2, 64)
    clean = _run(t, q, cu)
    page = int(t["table"][0, 2])  # tokens 40-47 of row 0, which are the span's own
    t["ks"][page, 1] = float("nan")
    dirty = _run(t, q, cu)
    assert torch.equal(dirty[:40], clean[:40]) and bool(dirty[40:64].isnan().all())
    assert torch.equal(dirty[64:], clean[64:])
    t["ks"][page, 1], t["vs"][page, 1] = 0.01, float("inf")
    dirty = _run(t, q, cu)
    assert torch.equal(dirty[:40], clean[:40]) and bool(dirty[40:64].isnan().all())


def test_blocks_behind_the_end_have_no_weight():
    t, q, cu = _case(9, [50, 23], [20, 23], [99, 99], 4, 1, 128)
    clean = _run(t, q, cu)
    t["ks"][int(t["table"][1, 1]), 1] = float("inf")  # tokens 24-31 of row 1
    t["vs"][int(t["table"][0, 3]), 1] = float("nan")  # tokens 56-63 of row 0
    assert torch.equal(clean, _run(t, q, cu))


def test_zero_scales_and_scales_far_apart():
    t, q, cu = _case(10, [300], [70], [15], 4, 2, 64)
    t["ks"][:4], t["vs"][3:7] = 0.0, 0.0
    t["vs"][7], t["vs"][8] = 1e-25, 3e4
    _check(t, q, cu, _run(t, q, cu))


@pytest.mark.parametrize("power", [-80, 90])
def test_values_of_any_size(power):
    t, q, cu = _case(13, [700, 90], [70, 20], [99, 99], 4, 2, 128)
    t["vs"] *= 2.0 ** power
    _check(t, q, cu, _run(t, q, cu))


def test_strides_lse_and_scales():
    t, q0, cu = _case(11, [90, 33], [50, 33], [4, 1], 8, 4, 64)
    wide = torch.zeros((83, 2, 8, 64), dtype=torch.bfloat16, device="cuda")
    wide[:, 1] = q0
    q, o = wide[:, 1], torch.full((83, 3, 8, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty((83, 8), dtype=torch.float32, device="cuda")
    f = torch.arange(1, 9, device="cuda").float() / 4
    out = _run(t, q, cu, out=o[:, 1], lse=lse, out_scale=f)
    _check(t, q, cu, out.double() / f.double()[:, None])
    assert bool((o[:, [0, 2]] == 3).all())
    k, _ = row_keys(t, 1)
    x = torch.einsum("lhd,nhd->lhn", q[50:].double(), k.repeat_interleave(2, 1)) / 8
    x = x.masked_fill(torch.ones((33, 33), device="cuda").triu(1).bool()[:, None], float("-inf"))
    # a weight's error of POLY is one of the sum's
    assert float((torch.logsumexp(x, -1) - lse[50:]).abs().max()) <= 2 * POLY


def test_refusals():
    from lastkv_b200.contract import RMarinBackendContractError as Refused

    t, q, cu = _case(12, [40], [10], [1], 4, 2, 64)
    with pytest.raises(Refused, match="staged"):
        _run(t, q, cu, staged=True)
    with pytest.raises(Refused, match="stage holds"):
        _run(t, q, cu, stage=ops.StageQ8.empty(1, 3, 2, 64)._replace(width=4))
    with pytest.raises(Refused, match="heads"):
        _run(t, q, cu, stage=ops.StageQ8.empty(1, 3, 1, 64))
    with pytest.raises(Refused, match="partials"):
        _run(t, q, cu, kv_splits=2, partials=(torch.empty((2, 40, 64), device="cuda"), torch.empty(2, 39, device="cuda")))
    with pytest.raises(Refused, match="unsupported"):
        _run(t, q, cu, kv_splits=9)
    with pytest.raises(Refused, match="cu_q"):
        _run(t, q, cu.long())
    with pytest.raises(Refused, match="together"):
        _run(t, q, cu, pool_v=None)
