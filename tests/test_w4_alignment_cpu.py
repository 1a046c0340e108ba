"""Addresses that the products' loads and stores cannot take are refused before any CUDA call."""

import pytest


@pytest.fixture(scope="module")
def lib():
    from lastkv_b200 import _capi, build

    build.build()
    return _capi.load()


@pytest.mark.parametrize("y,bias,scale", [(17, None, 16), (16, 17, 16), (16, None, 18), (16, None, 17)])
def test_odd_addresses(lib, y, bias, scale):
    def bf16(y, bias):
        return lib.lkv_w4_linear(16, 128, 16, bias, y, 64, 1, 64, 128, 128, None, None)

    def int8(y, bias, scale):
        return lib.lkv_w4_linear_q8(8, 128, scale, 1, 16, bias, y, 64, 1, 64, 128, 128, None, None)

    assert int8(y, bias, scale) == 1
    if scale == 16:
        assert bf16(y, bias) == 1
