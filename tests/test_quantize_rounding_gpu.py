"""Codes of 8-bit pages are the fp32 quotients by the stored scale, rounded to nearest, ties to even: bit for bit."""

import pytest
import torch

from lastkv_b200 import ops
from tests.q8_helpers import quantized

pytestmark = pytest.mark.gpu


def _codes(x):
    ids = torch.arange(x.shape[0], dtype=torch.int32, device="cuda")
    cache = ops.PagesQ8.empty(x.shape[0], x.shape[2], x.shape[3])
    ops.quantize_pages(x, x.flip(0), ids, cache, ids)
    k, v, ks, vs = cache.to_codes()
    return (k, ks), (v.flip(0), vs.flip(0))


def _check(x):
    _, scale = quantized(x)
    s = scale.repeat_interleave(8, 1)[..., None]
    want = torch.where(s == 0, 0, torch.round(x.float() / s)).double()  # (two tensors: an fp32 division)
    for codes, got in _codes(x):
        assert torch.equal(got, scale)
        assert torch.equal(codes.double(), want), int((codes.double() != want).sum())


@pytest.mark.parametrize("d", [64, 128])
def test_random_values(d):
    g = torch.Generator().manual_seed(d)
    _check(torch.randn((300, 16, 4, d), generator=g).bfloat16().cuda())


@pytest.mark.parametrize("exponent", [0, 60, -60, -100, -106, -110, -120, -126, -130])
def test_values_half_way_between_two_codes(exponent):
    """Every mantissa as a block's largest value, with its half, quarter and so on, and random values below it;
    down to the numbers whose scales have few bits left."""
    g = torch.Generator().manual_seed(1)
    top = (128 + torch.arange(128)).double() * 2.0 ** (exponent - 7)
    parts = torch.randint(-254, 255, (128, 8 * 64), generator=g).double() / 254
    x = (top[:, None] * parts).bfloat16().double()
    x[:, 0], x[:, 7], x[:, 100], x[:, 301] = top, -top / 2, top / 2, top / 4
    x = x.bfloat16().view(64, 16, 1, 64).cuda()  # two blocks to a page
    _check(x)
