"""The reciprocal that quantising multiplies by, restated: x * inv is rounded as the fp32 x / scale is, for every bf16 x."""

import numpy as np

F = np.float32


def _inverse(top):
    """127 / top, a step away from the nearest where half of the largest value would go to the other side of 63.5 than
    it does by the stored scale."""
    scale = F(top) / F(127)
    inv = F(127) / F(top)
    by_scale = F(top) / F(2) / scale >= F(63.5)
    by_inv = float(top) * float(inv) - 127.0 >= 0  # exact in one fused multiply-add: 64 bits hold the product
    if by_scale and not by_inv:
        inv = np.nextafter(inv, F(np.inf))
    if not by_scale and by_inv:
        inv = np.nextafter(inv, F(0))
    return scale, float(inv)


def test_every_mantissa():
    for m in range(128, 256):
        top = float(m)
        scale, inv = _inverse(top)
        a = np.arange(128, 256, dtype=np.float64)
        x = (a[None, :] * 2.0 ** -np.arange(0, 12)[:, None]).reshape(-1)
        x = x[x <= top]
        # products of 8 and 24 bits are exact in 64
        assert np.array_equal(np.rint(x * inv), np.rint(x.astype(F) / scale)), m
        assert np.rint(top * inv) == 127
