"""Rows of q that belong to no span (padding in front of the first and behind the last) leave the buffers alone."""

import pytest
import torch

from lastkv_b200 import ops
from tests.q8_helpers import random_cache

pytestmark = pytest.mark.gpu


def _buffers(T, hq, d):
    return (torch.full((T, hq, d), 3.0, dtype=torch.bfloat16, device="cuda"), torch.full((T, hq), 5.0, device="cuda"))


def _check(out, lse, one, one_lse, first, last, v):
    for t, was in ((out, 3.0), (lse, 5.0)):
        assert bool((t[:first] == was).all()) and bool((t[last:] == was).all())
    # either is off by its output's rounding and a half step of every weight (and a polynomial's error): of the values
    off = (out[first:last].double() - one[first:last].double()).abs()
    assert float(off.max()) <= 2 * (2.0 ** -8 * float(one[first:last].abs().max()) + (2.0 ** -8 + 2 * 7.5e-5) * v)
    assert bool(out[first:last].isfinite().all()) and bool(lse[first:last].isfinite().all())


@pytest.mark.parametrize("splits", [1, 2, 8])
@pytest.mark.parametrize("first", [0, 7])
@pytest.mark.parametrize("d", [64, 128])
def test_spans_over_8_bit_pages(splits, first, d):
    t = random_cache(71, [1100, 300], [60, 5], 2, d)
    cu = torch.tensor([first, first + 9, first + 49], dtype=torch.int32, device="cuda")
    T, last = first + 49 + 30, first + 49
    q = torch.randn((T, 4, d), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    cache = ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])
    got = []
    for s in (splits, 1):
        out, lse = _buffers(T, 4, d)
        nan = torch.full((s, T * 4, d), float("nan"), device="cuda"), torch.full((s, T * 4), float("nan"), device="cuda")
        ops.prefill_paged_q8(q, cache, t["table"], t["seq_k"], cu, 40, num_q8=t["num_q8"], pool_k=t["pool_k"],
                             pool_v=t["pool_v"], kv_splits=s, out=out, lse=lse, partials=nan)
        got += [out, lse]
    _check(*got, first, last, max(127 * float(t["vs"].max()), float(t["pool_v"].abs().max())))


@pytest.mark.parametrize("splits", [1, 4])
@pytest.mark.parametrize("first", [0, 3])
def test_spans_over_bf16_pages(splits, first):
    t = random_cache(72, [1100, 300], [0, 0], 2, 64)
    cu = torch.tensor([first, first + 9, first + 49], dtype=torch.int32, device="cuda")
    T, last = first + 49 + 30, first + 49
    q = torch.randn((T, 4, 64), generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    got = []
    for s in (splits, 1):
        out, lse = _buffers(T, 4, 64)
        nan = torch.full((s, T * 4, 64), float("nan"), device="cuda"), torch.full((s, T * 4), float("nan"), device="cuda")
        ops.prefill_paged(q, t["pool_k"], t["pool_v"], t["table"], t["seq_k"], cu, 40, causal=False, kv_splits=s,
                          out=out, lse=lse, partials=nan)
        got += [out, lse]
    _check(*got, first, last, float(t["pool_v"].abs().max()))
