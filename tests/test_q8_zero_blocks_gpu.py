"""Blocks of zeros beside large values: their tokens keep their weight, and only theirs."""

import pytest
import torch

from lastkv_b200 import ops
from tests.q8_helpers import FP32_HALF_STEP, assert_within, attention, random_cache, row_keys

pytestmark = pytest.mark.gpu

POLY = 7.5e-5  # the relative error of the exponentials that a polynomial takes


def _check_lse(lse, q, k, weight_error=0.0, causal_from=None):
    """Log-sum-exps [L, Hq] of one row: a weight's relative error is one of the sum's, a score's (a sum of D products,
    and its scaling) one of its exponential's; the sum itself has n roundings, the logarithm's last steps some of its size."""
    n, D = k.shape[0], q.shape[2]
    k = k.repeat_interleave(q.shape[1] // k.shape[1], 1)
    x = torch.einsum("lhd,nhd->lhn", q.double(), k) * D ** -0.5
    off = torch.einsum("lhd,nhd->lhn", q.double().abs(), k.abs()).amax(-1) * D ** -0.5
    if causal_from is not None:
        late = torch.arange(n, device=x.device)[None] > causal_from + torch.arange(x.shape[0], device=x.device)[:, None]
        x = x.masked_fill(late[:, None], float("-inf"))
    want = torch.logsumexp(x, -1)
    # the largest value scale goes through the running maximum and back: 128 at most as its logarithm
    tol = 2 * weight_error + (4 * D * off + 2 * n + 4 * want.abs() + 4 * 128) * FP32_HALF_STEP
    assert bool(((lse.double() - want).abs() <= tol).all()), float((lse.double() - want).abs().max())


def _cache(seed, lens, num_q8, power, d, low=0.0):
    """Values of about 2^power, every third half page of value scale `low`."""
    t = random_cache(seed, lens, num_q8, 2, d)
    t["vs"] *= 2.0 ** power
    t["pool_v"] = (t["pool_v"].float() * 2.0 ** power).bfloat16()
    half = torch.arange(t["vs"].shape[0] * 2, device="cuda").view(-1, 2) % 3 == 1
    t["vs"] = torch.where(half[..., None], low, t["vs"]).contiguous()
    return t


@pytest.mark.parametrize("power", [20, 40, 60, 90])
@pytest.mark.parametrize("lens,num_q8", [([300, 90], [9999, 9999]), ([9000, 20], [9999, 1]), ([700, 40], [20, 2])])
def test_single_tokens(power, lens, num_q8):
    t = _cache(51, lens, num_q8, power, 128)
    q = torch.randn((2, 4, 128), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    cache = ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])
    lse = torch.empty((2, 4), device="cuda")
    out = ops.decode_paged_q8(q, cache, t["table"], t["seq_k"], num_q8=t["num_q8"], pool_k=t["pool_k"],
                              pool_v=t["pool_v"], lse=lse)
    for b in range(2):
        k, v = row_keys(t, b)
        ref, bound = attention(q[b:b + 1], k, v, 128 ** -0.5)
        assert_within(out[b:b + 1], ref, bound, f"row {b}")
        _check_lse(lse[b:b + 1], q[b:b + 1], k)


@pytest.mark.parametrize("power", [20, 40, 60, 90])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("d", [64, 128])
def test_spans(power, splits, d):
    """Causal spans that end inside a block, so that most blocks have keys that a token does not see."""
    t = _cache(52, [700, 90, 333], [9999, 9999, 12], power, d)
    cu = torch.tensor([0, 70, 90, 390], dtype=torch.int32, device="cuda")
    q = torch.randn((390, 4, d), generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    cache = ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])
    lse = torch.empty((390, 4), device="cuda")
    out = ops.prefill_paged_q8(q, cache, t["table"], t["seq_k"], cu, 300, num_q8=t["num_q8"], pool_k=t["pool_k"],
                               pool_v=t["pool_v"], kv_splits=splits, lse=lse)
    c = cu.tolist()
    for b in range(3):
        k, v = row_keys(t, b)
        span = q[c[b]:c[b + 1]]
        n, L = k.shape[0], span.shape[0]
        ref, bound = attention(span, k, v, d ** -0.5, n - L, POLY)
        assert_within(out[c[b]:c[b + 1]], ref, bound, f"row {b}")
        _check_lse(lse[c[b]:c[b + 1]], span, k, POLY, n - L)


@pytest.mark.parametrize("span", [False, True])
def test_a_row_of_zero_blocks(span):
    """Nothing but zeros as values: zeros, and the log-sum-exp of the scores."""
    t = random_cache(53, [200], [9999], 2, 64)
    t["vs"].zero_()
    q = torch.randn((2 if span else 1, 4, 64), generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    cache = ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])
    lse = torch.empty(q.shape[:2], device="cuda")
    if span:
        cu = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
        out = ops.prefill_paged_q8(q, cache, t["table"], t["seq_k"], cu, 2, causal=False, lse=lse)
    else:
        out = ops.decode_paged_q8(q, cache, t["table"], t["seq_k"], lse=lse)
    k, _ = row_keys(t, 0)
    assert bool((out == 0).all())
    _check_lse(lse, q, k, POLY)


@pytest.mark.parametrize("behind", [-1.0, float("-inf"), float("nan"), 1e-40])
def test_what_lies_behind_a_zero_block(behind):
    """A zero block before the row's end, whatever the scales of the blocks behind it hold; an odd number of pages, so
    that the last one has no neighbour."""
    t = random_cache(54, [20, 72, 200], [9999] * 3, 2, 64)
    q = torch.randn((3, 4, 64), generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    for b, column, half in ((0, 1, 0), (1, 4, 0), (2, 12, 0)):  # the row's last tokens
        t["vs"][int(t["table"][b, column]), half] = 0
        t["vs"][int(t["table"][b, column]), 1 - half] = behind
    cache = ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    for out in (ops.decode_paged_q8(q, cache, t["table"], t["seq_k"]),
                ops.prefill_paged_q8(q, cache, t["table"], t["seq_k"], cu, 1)):
        for b in range(3):
            ref, bound = attention(q[b:b + 1], *row_keys(t, b), 64 ** -0.5, None, POLY)
            assert_within(out[b:b + 1], ref, bound, f"row {b}")


@pytest.mark.parametrize("power", [0, 30, 50, 90])
@pytest.mark.parametrize("zeros", ["first", "last"])
def test_pages_of_zeros_and_pages_of_large_values(power, zeros):
    """Hundreds of keys whose values are zeros, before or behind those whose values are not."""
    n, d = 1600, 64
    t = random_cache(55, [n], [9999], 2, d)
    t["vs"] *= 2.0 ** power
    pages = t["table"][0].long()
    t["vs"][pages[:60] if zeros == "first" else pages[-60:]] = 0
    q = torch.randn((3, 4, d), generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    cache = ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])
    k, v = row_keys(t, 0)
    ref, bound = attention(q, k, v, d ** -0.5, None, POLY)
    lse = torch.empty((3, 4), device="cuda")
    out = ops.decode_paged_q8(q, cache, t["table"].expand(3, -1), t["seq_k"].expand(3).contiguous(), lse=lse)
    assert_within(out, ref, bound, "tokens")
    _check_lse(lse, q, k)
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    for splits in (1, 3):
        out = ops.prefill_paged_q8(q, cache, t["table"], t["seq_k"], cu, 3, causal=False, kv_splits=splits, lse=lse)
        assert_within(out, ref, bound, f"span in {splits} parts")
        _check_lse(lse, q, k, POLY)
