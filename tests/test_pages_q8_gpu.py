"""Pages to 8 bits and back, and copies of pages, against their formulas."""

import pytest
import torch

from lastkv_b200 import ops
from tests.q8_helpers import FP32_HALF_STEP, quantized, values

pytestmark = pytest.mark.gpu


def _pool(seed, pages, hkv, d, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((pages, 16, hkv, d), generator=g) * spread
    x *= torch.where(torch.rand((hkv, d), generator=g) < 0.05, 8.0, 1.0)
    return x.bfloat16().cuda()


def _ids(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _check_codes(pages, codes, scale):
    """Scales as the formula has them; codes within the rounding of the quotient: x * (127 / max) has two
    roundings of half a step, at most 127 * 2 * 2^-24 off, so a code is at most that past its half-way point."""
    _, want = quantized(pages)
    assert torch.equal(scale.isnan(), want.isnan())
    assert torch.equal(scale.nan_to_num(nan=-1, posinf=-2), want.nan_to_num(nan=-1, posinf=-2))
    s = want.repeat_interleave(8, 1)[..., None].double()
    fine = s.isfinite() & (s > 0)
    assert bool((codes.double()[(~fine).expand_as(codes)] == 0).all())
    quotient = torch.where(fine, pages.double() / s, 0)
    # the scale itself is rounded once more than 127 / max
    slack = 127 * 4 * FP32_HALF_STEP
    assert float((codes.double() - quotient).abs().max()) <= 0.5 + slack
    assert int(codes.abs().max()) <= 127


@pytest.mark.parametrize("n,hkv,d", [(1, 1, 64), (1, 8, 128), (7, 3, 128), (33, 5, 64), (260, 8, 128)])
def test_quantize_and_back(n, hkv, d):
    k, v = _pool(n, n + 4, hkv, d), _pool(n + 1, n + 4, hkv, d, 30.0)
    g = torch.Generator().manual_seed(3)
    src = torch.randperm(n + 4, generator=g)[:n].int().cuda()
    dst = torch.randperm(n + 2, generator=g)[:n].int().cuda()
    cache = ops.PagesQ8.empty(n + 2, hkv, d)
    cache.codes.fill_(9)
    cache.scales.fill_(3.0)
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    ops.quantize_pages(k, v, src, cache, dst, error_word=err)
    ck, cv, ks, vs = cache.to_codes()
    at = dst.long()
    _check_codes(k[src.long()], ck[at], ks[at])
    _check_codes(v[src.long()], cv[at], vs[at])
    rest = [i for i in range(n + 2) if i not in at.tolist()]
    assert bool((cache.codes[rest] == 9).all()) and bool((cache.scales[rest] == 3).all())
    # back: bit for bit bf16(code * scale)
    bk, bv = torch.full_like(k, 5.0), torch.full_like(v, 5.0)
    ops.dequantize_pages(cache, dst, bk, bv, src, error_word=err)
    for back, codes, scale in ((bk, ck, ks), (bv, cv, vs)):
        want = (codes.float() * scale.repeat_interleave(8, 1)[..., None]).bfloat16()[at]
        assert torch.equal(back[src.long()], want)
        assert bool((back[[i for i in range(n + 4) if i not in src.tolist()]] == 5).all())
    assert err.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("d", [64, 128])
def test_pages_that_hold_fewer_tokens(d):
    hkv, counts = 3, [0, 1, 7, 8, 9, 15, 16, 20, -1]
    n = len(counts)
    k, v = _pool(1, n, hkv, d), _pool(2, n, hkv, d)
    k[:, 12:] = 1e30  # behind most pages' last token
    v[3, 8:] = float("nan")
    ids = _ids(*range(n))
    cache = ops.PagesQ8.empty(n, hkv, d)
    ops.quantize_pages(k, v, ids, cache, ids, tokens=_ids(*counts))
    ck, cv, ks, vs = cache.to_codes()
    tok = torch.arange(16, device="cuda")
    live = (tok < torch.tensor(counts, device="cuda")[:, None])[..., None, None]
    _check_codes(torch.where(live, k, 0), ck, ks)
    _check_codes(torch.where(live, v, 0), cv, vs)
    assert bool((ck[~live.expand_as(ck)] == 0).all())


@pytest.mark.parametrize("d", [64, 128])
def test_blocks_of_all_kinds_of_values(d):
    """Zeros, the smallest numbers, the largest, infinities and NaN, each in a block of 8 tokens of its own."""
    fills = [0.0, 1e-39, 9.2e-41, 2e-38, 1e-30, 3e38, -3e38]
    n = len(fills) + 4
    k, v = _pool(4, n, 2, d), _pool(5, n, 2, d)
    for i, f in enumerate(fills):
        k[i, :8], v[i, 8:] = f, f
        k[i, 3, 1, 5] = f / 2
    k[-4, 2, 0, 7], v[-4, 9, 1, 0] = float("inf"), float("-inf")
    k[-3, 15, 1, d - 1] = float("nan")
    v[-2, :, 0] = float("nan")
    ids = _ids(*range(n))
    cache = ops.PagesQ8.empty(n, 2, d)
    ops.quantize_pages(k, v, ids, cache, ids)
    ck, cv, ks, vs = cache.to_codes()
    _check_codes(k, ck, ks)
    _check_codes(v, cv, vs)
    back = torch.empty_like(k), torch.empty_like(v)
    ops.dequantize_pages(cache, ids, *back, ids)
    # a block that holds what is not finite reads as NaN, its neighbours as themselves
    assert bool(back[0][-4, :8, 0].isnan().all()) and bool(back[0][-4, 8:].isfinite().all())
    assert bool(back[0][-3, 8:, 1].isnan().all()) and bool(back[0][-3, :8].isfinite().all())
    assert bool(back[1][-2, :, 0].isnan().all()) and bool(back[1][-2, :, 1].isfinite().all())


def test_pages_outside_the_pools_are_skipped():
    k, v = _pool(1, 4, 2, 64), _pool(2, 4, 2, 64)
    cache = ops.PagesQ8.empty(3, 2, 64)
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    ops.quantize_pages(k, v, _ids(0, 4, -1, 2, 1), cache, _ids(0, 1, 1, 3, 2), error_word=err)
    assert err[0] == 2 and err[1] == 8
    assert bool((cache.codes[1] == 128).all()) and bool((cache.scales[1] == 0).all())
    _check_codes(k[[0, 1]], cache.to_codes()[0][[0, 2]], cache.to_codes()[2][[0, 2]])
    err.zero_()
    back = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    ops.dequantize_pages(cache, _ids(0, 3, -5, 2), *back, _ids(1, 0, 2, 4), error_word=err)
    assert err[0] == 2 and err[1] == 9
    assert bool((back[0][[0, 2, 3]] == 7).all()) and not bool((back[0][1] == 7).all())
    ops.quantize_pages(k, v, _ids(9), cache, _ids(0))  # without an error word
    ops.quantize_pages(k, v, _ids(), cache, _ids())    # nothing to do
    torch.cuda.synchronize()


def test_values_stand_for_the_codes():
    """from_codes, the kernels' order and dequantize_pages agree."""
    g = torch.Generator().manual_seed(8)
    for d in (64, 128):
        k, v = (torch.randint(-127, 128, (5, 16, 3, d), generator=g).to(torch.int8).cuda() for _ in range(2))
        ks, vs = (torch.rand((5, 2, 3), generator=g).cuda() for _ in range(2))
        cache = ops.PagesQ8.from_codes(k, v, ks, vs)
        back = torch.empty((5, 16, 3, d), dtype=torch.bfloat16, device="cuda"), \
            torch.empty((5, 16, 3, d), dtype=torch.bfloat16, device="cuda")
        ids = _ids(*range(5))
        ops.dequantize_pages(cache, ids, *back, ids)
        assert torch.equal(back[0], values(k, ks).float().bfloat16())
        assert torch.equal(back[1], values(v, vs).float().bfloat16())


# ---------------------------------------------------------------- copies of pages


def _expected(pool, src, dst, layers, stride):
    out = pool.clone()
    for l in range(layers):
        for s, d in zip(src, dst):
            out[d + l * stride] = pool[s + l * stride]
    return out


@pytest.mark.parametrize("n,layers", [(1, 1), (2, 3), (5, 1), (31, 2), (33, 4), (64, 2), (700, 1), (2048, 1)])
def test_reorder_permutes_pages(n, layers):
    """In place, among themselves, in pools of several types and page sizes."""
    g = torch.Generator().manual_seed(n)
    stride = n + 3
    ids = torch.randperm(n + 2, generator=g)[:n].tolist()
    src = [ids[i] for i in torch.randint(0, n, (n,), generator=g).tolist()]
    pools = [torch.randint(-2**30, 2**30, (layers * stride + 1, words), generator=g, dtype=torch.int32).cuda()
             for words in ((4, 12, 1028) if n > 64 else (4, 12, 8192))]
    pools.append(torch.randn((layers * stride + 1, 16, 2, 64), generator=g).bfloat16().cuda())
    want = [_expected(p, src, ids, layers, stride) for p in pools]
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    ops.reorder_pages(pools, _ids(*src), _ids(*ids), layers=layers, layer_stride=stride if layers > 1 else 0,
                      error_word=err)
    assert err.tolist() == [0, 0, 0, 0]
    for p, w in zip(pools, want):
        assert torch.equal(p, w)


def test_reorder_cycle_and_one_source():
    pool = torch.arange(6 * 64, dtype=torch.float32, device="cuda").view(6, 64)
    want = pool[[1, 2, 3, 4, 5, 0]].clone()
    ops.reorder_pages(pool, _ids(1, 2, 3, 4, 5, 0), _ids(0, 1, 2, 3, 4, 5))
    assert torch.equal(pool, want)
    ops.reorder_pages(pool, _ids(3, 3, 3, 3), _ids(0, 1, 3, 5))
    assert torch.equal(pool, want[[3, 3, 2, 3, 4, 3]])
    ops.reorder_pages(pool, _ids(), _ids())
    assert torch.equal(pool, want[[3, 3, 2, 3, 4, 3]])


def test_reorder_skips_pages_that_are_not_there():
    pool = torch.arange(8 * 64, dtype=torch.float32, device="cuda").view(8, 64)
    want = pool.clone()
    want[1] = pool[0]
    want[5] = pool[4]
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    # ids of one layer are below the stride; 4 and -1 are not
    ops.reorder_pages(pool, _ids(0, 4, 2, -1), _ids(1, 2, 4, 3), layers=2, layer_stride=4, error_word=err)
    assert err[0] == 2 and err[1] == 10
    assert torch.equal(pool, want)
    err.zero_()
    ops.reorder_pages(pool, _ids(8, 3), _ids(0, 6), error_word=err)
    assert err[0] == 2
    want[6] = want[3]
    assert torch.equal(pool, want)
