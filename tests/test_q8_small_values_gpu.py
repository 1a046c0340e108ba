"""Small values: 8-bit pages beside bf16 pages whose values are as small keep their part of the result."""

import pytest
import torch

from lastkv_b200 import ops
from tests.q8_helpers import assert_within, attention, random_cache, row_keys

pytestmark = pytest.mark.gpu

POLY = 7.5e-5  # the relative error of the exponentials that a polynomial takes
LENS, NUM_Q8 = [700, 300, 2100, 90], [20, 18, 64, 2]


def _case(power, d, flat):
    """Values of about 2^power in both kinds of pages; flat: keys so small that every token has about the same weight."""
    t = random_cache(61, LENS, NUM_Q8, 2, d)
    t["vs"] *= 2.0 ** power
    t["pool_v"] = (t["pool_v"].float() * 2.0 ** power).bfloat16()
    if flat:
        t["ks"] *= 2.0 ** -6
        t["pool_k"] = (t["pool_k"].float() * 2.0 ** -6).bfloat16()
    return t, ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])


@pytest.mark.parametrize("flat", [False, True])
@pytest.mark.parametrize("power", [-50, -30, -20, -10, 0, 30])
@pytest.mark.parametrize("d", [64, 128])
def test_single_tokens(power, d, flat):
    t, cache = _case(power, d, flat)
    q = torch.randn((4, 4, d), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    out = ops.decode_paged_q8(q, cache, t["table"], t["seq_k"], num_q8=t["num_q8"], pool_k=t["pool_k"], pool_v=t["pool_v"])
    for b in range(4):
        ref, bound = attention(q[b:b + 1], *row_keys(t, b), d ** -0.5)
        assert_within(out[b:b + 1], ref, bound, f"row {b}")


@pytest.mark.parametrize("flat", [False, True])
@pytest.mark.parametrize("power", [-50, -30, -20, -10, 0, 30])
@pytest.mark.parametrize("d", [64, 128])
def test_spans(power, d, flat):
    """8-bit and bf16 pages in one block of 128 keys."""
    t, cache = _case(power, d, flat)
    spans = [10, 40, 3, 70]
    cu = torch.tensor([0] + spans).cumsum(0).int().cuda()
    q = torch.randn((int(cu[-1]), 4, d), generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    out = ops.prefill_paged_q8(q, cache, t["table"], t["seq_k"], cu, 70, num_q8=t["num_q8"], pool_k=t["pool_k"],
                               pool_v=t["pool_v"])
    c = cu.tolist()
    for b in range(4):
        k, v = row_keys(t, b)
        ref, bound = attention(q[c[b]:c[b + 1]], k, v, d ** -0.5, k.shape[0] - spans[b], POLY)
        assert_within(out[c[b]:c[b + 1]], ref, bound, f"row {b}")
