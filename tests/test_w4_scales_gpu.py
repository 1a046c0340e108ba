"""int8 rows whose scales use all 24 bits, and scales at the ends of their ranges: equal results of either kernel.

One product per sum (a single 1 in a row, weights of code 1): x * w with w a power of two is exact in fp32 wherever
it is normal, and rounds once to bf16, so the outputs are those of the definition bit for bit.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

# (tokens, n): the streaming kernel, its widest calls, tiles of 64, 128 and 256 tokens, tiles with k in one split
SHAPES = [(4, 64), (32, 320), (60, 4000), (100, 3000), (300, 1000), (300, 6000)]


def weight(n, k, group, scales):
    """Codes 1 everywhere; `scales` [n] for each row's groups."""
    from lastkv_b200 import ops

    codes = torch.full((n, k // 2), 0x99, dtype=torch.uint8, device="cuda")
    return ops.w4_pack(codes, scales.bfloat16()[:, None].expand(n, -(-k // group)).contiguous(), group)


def rows(scales, k, group, at=3):
    """One 1 per row, in column `at`; the scales of the other groups are 1."""
    from lastkv_b200 import ops

    t = scales.numel()
    q = torch.zeros((t, k), dtype=torch.int8, device="cuda")
    q[:, at] = 1
    s = torch.ones((t, -(-k // group)), device="cuda")
    s[:, at // group] = scales
    return ops.Q8Rows(q, s, group)


@pytest.mark.parametrize("t,n", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_every_bit_of_a_scale_counts(t, n, group):
    """1 + 2^-8 lies between two bf16 values and goes to the even one, 1; any bit above it, up to the last of
    fp32's 24, sends it to 1 + 2^-7."""
    from lastkv_b200 import ops

    more = 2.0 ** torch.arange(-23, -8, device="cuda", dtype=torch.float32)
    scales = (1 + 2.0 ** -8 + more)[torch.arange(t, device="cuda") % more.numel()]
    scales[::7] = 1 + 2.0 ** -8
    assert bool((scales[1::7] > 1 + 2.0 ** -8).all())
    y = ops.w4_linear(rows(scales, 512, group, at=130), weight(n, 512, group, torch.ones(n, device="cuda")))
    want = torch.full((t, n), 1 + 2.0 ** -7, dtype=torch.bfloat16, device="cuda")
    want[::7] = 1
    assert torch.equal(y, want)


@pytest.mark.parametrize("t,n", SHAPES)
@pytest.mark.parametrize("group", [32, 128])
def test_scales_over_their_whole_range(t, n, group):
    """Every pair of a token's scale (fp32, subnormal to the largest binade) and a row's (bf16, likewise)."""
    from lastkv_b200 import ops

    xs = 2.0 ** torch.tensor([-149, -140, -127, -126, -107, -90, -30, 0, 30, 90, 100, 110, 124, 127], device="cuda",
                             dtype=torch.float64)
    ws = 2.0 ** torch.tensor([-133, -127, -126, -110, -60, 0, 60, 103, 104, 108, 112, 120, 127], device="cuda",
                             dtype=torch.float64)
    x = xs[torch.arange(t, device="cuda") * 5 % xs.numel()]
    w = ws[torch.arange(n, device="cuda") * 3 % ws.numel()]
    y = ops.w4_linear(rows(x.float(), group, group), weight(n, group, group, w.float()))
    exact = x[:, None] * w[None]
    want = exact.float().bfloat16()
    # a product below fp32's normal numbers may be rounded on its way: at most to its neighbour in bf16
    small = exact < 2.0 ** -126
    assert torch.equal(y[~small], want[~small])
    assert bool(((y.double() - exact).abs()[small] <= 2.0 ** -133).all())
