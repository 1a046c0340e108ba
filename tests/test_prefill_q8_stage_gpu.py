"""The staged copy of 8-bit pages: calls of other table widths read it as it was written; tables without a column."""

import ctypes

import pytest
import torch

from lastkv_b200 import _capi, ops
from tests.q8_helpers import assert_within, attention, random_cache, row_keys

pytestmark = pytest.mark.gpu

POLY = 7.5e-5  # the relative error of the exponentials that a polynomial takes


def _case():
    t = random_cache(41, [400, 330, 90], [20, 18, 3], 2, 64)
    cu = torch.tensor([0, 64, 74, 100], dtype=torch.int32, device="cuda")
    q = torch.randn((100, 8, 64), generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    return t, q, cu, ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])


def _call(t, q, cu, cache, **kw):
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    out = ops.prefill_paged_q8(q, cache, t["table"], t["seq_k"], cu, 64, num_q8=t["num_q8"], pool_k=t["pool_k"],
                               pool_v=t["pool_v"], error_word=err, kv_splits=1, **kw)
    assert err.tolist() == [0, 0, 0, 0]
    return out


def _check(t, q, cu, out):
    c = cu.tolist()
    for b in range(len(c) - 1):
        k, v = row_keys(t, b)
        span = q[c[b]:c[b + 1]]
        ref, bound = attention(span, k, v, q.shape[2] ** -0.5, k.shape[0] - span.shape[0], POLY)
        assert_within(out[c[b]:c[b + 1]], ref, bound, f"row {b}")


@pytest.mark.parametrize("first,second", [(60, 25), (25, 60), (None, 25), (25, None)])
@pytest.mark.parametrize("width", [20, 33, 70])
def test_calls_of_other_widths_share_a_stage(first, second, width):
    """A table with room behind its rows, of which two calls see different numbers of columns."""
    t, q, cu, cache = _case()
    wide = torch.full((3, 60), -5, dtype=torch.int32, device="cuda")
    wide[:, :25] = t["table"][:, :25]
    small = dict(t, table=wide)
    stage = ops.StageQ8.empty(3, width, 2, 64)
    a = _call(small, q, cu, cache, stage=stage, max_pages=first)
    _check(t, q, cu, a)
    b = _call(small, q, cu, cache, stage=stage, max_pages=second, staged=True)
    assert torch.equal(a, b)


def test_a_table_without_columns():
    t, q, cu, cache = _case()
    empty = torch.zeros(3, dtype=torch.int32, device="cuda")
    narrow = torch.zeros((3, 0), dtype=torch.int32, device="cuda")
    for kw in (dict(max_pages=0), dict(table=narrow)):
        s = dict(t, seq_k=empty, table=kw.pop("table", t["table"]))
        out = _call(s, q, cu, cache, **kw)
        assert bool((out == 0).all())
        one = ops.decode_paged_q8(q[:3], cache, s["table"], empty, num_q8=t["num_q8"], pool_k=t["pool_k"],
                                  pool_v=t["pool_v"], **kw)
        assert bool((one == 0).all())


def test_a_stage_wider_than_the_table_through_the_c_entry():
    t, q, cu, cache = _case()
    want = _call(t, q, cu, cache)
    width = 99
    stage = ops.StageQ8.empty(3, width, 2, 64)
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    for staged in (2, 1):
        out = torch.empty_like(want)
        st = _capi.lib().lkv_prefill_paged_q8(
            q.data_ptr(), q.stride(0), cache.codes.data_ptr(), cache.scales.data_ptr(), cache.num_pages,
            stage.k.data_ptr(), stage.v.data_ptr(), width, staged, t["pool_k"].data_ptr(), t["pool_v"].data_ptr(),
            t["pool_k"].shape[0], t["table"].data_ptr(), t["table"].stride(0), t["num_q8"].data_ptr(),
            t["seq_k"].data_ptr(), cu.data_ptr(), out.data_ptr(), out.stride(0), None, None, 3, 100, 64, 8, 2, 64,
            t["table"].shape[1], 1, ctypes.c_float(64 ** -0.5), 1, None, None, err.data_ptr(),
            torch.cuda.current_stream().cuda_stream)
        assert st == 0 and torch.equal(out, want) and err.tolist() == [0, 0, 0, 0]
