"""int8 rows with group scales (lkv_rmsnorm_q8, lkv_silu_mul_q8, lkv_quantize_q8, lkv_dequantize_q8) against
the definition in 64 bits.

Tolerances.  A scale is a chain of fp32 roundings: the sum of squares adds at most 64 products per thread and ten
tree levels, and the square root, division, products and the exponential (2 ulp) add less than 20 more half-ulps, so
it is within 100 * 2^-24 < 1e-5 of the 64-bit scale.  A value y then lies within that relative error too, and its
quotient by the scale, at most 127, within 127 * 2e-5 < 0.004: every int8 is within 0.504 of y / s.  The residual
sum is one fp32 addition and one rounding, as torch's bf16 addition: equal.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

REL = 1e-5
STEP = 0.504


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(sum(k * 7919 ** i for i, k in enumerate(key)) % (1 << 31))


def _check(rows, y, group):
    """rows against the 64-bit values y [T, K]."""
    T, K = y.shape
    G = -(-K // group)
    assert rows.q.shape == (T, K) and rows.scale.shape == (T, G)
    which = torch.arange(K, device=y.device) // group
    top = torch.zeros((T, G), dtype=torch.float64, device=y.device).scatter_reduce_(1, which.expand(T, K), y.abs(), "amax")
    want = top / 127
    assert bool(((rows.scale.double() - want).abs() <= REL * want).all())
    s = want[:, which]
    off = (y - rows.q.double() * s).abs()
    assert bool((off <= STEP * s).all()), float((off / s).max())
    assert int(rows.q.abs().max()) <= 127


def _norm64(h, w, eps):
    return h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


@pytest.mark.parametrize("rows,cols", [(1, 8), (1, 4096), (3, 72), (8, 4096), (37, 1544), (5, 8200), (2, 32768),
                                       (300, 768)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("with_residual", [False, True])
def test_rmsnorm(rows, cols, group, with_residual):
    from lastkv_b200 import ops

    g = _gen(rows, cols, group)
    x = torch.randn((rows, cols), generator=g, device="cuda").bfloat16()
    r = (torch.randn((rows, cols), generator=g, device="cuda") * 3).bfloat16()
    w = (torch.rand(cols, generator=g, device="cuda") + 0.5).bfloat16()
    if with_residual:
        h, out = ops.rmsnorm_q8(x, w, 1e-5, r, group=group)
        torch.testing.assert_close(h, x + r, rtol=0, atol=0)
        _check(out, _norm64(x.double() + r.double(), w, 1e-5), group)
    else:
        out = ops.rmsnorm_q8(x, w, 1e-5, group=group)
        _check(out, _norm64(x.double(), w, 1e-5), group)


@pytest.mark.parametrize("rows,cols", [(1, 8), (8, 14336), (33, 264), (400, 1544)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_silu_and_plain(rows, cols, group):
    from lastkv_b200 import ops

    g = _gen(rows, cols, group, 1)
    gu = (torch.randn((rows, 2 * cols), generator=g, device="cuda") * 4).bfloat16()
    d = gu.double()
    _check(ops.silu_mul_q8(gu, group=group), d[:, :cols] * torch.sigmoid(d[:, :cols]) * d[:, cols:], group)
    x = gu[:, :cols]  # rows of a wider tensor
    _check(ops.quantize_q8(x, group=group), x.double(), group)


def test_strided_outputs_and_dequantize():
    from lastkv_b200 import ops

    g = _gen(5)
    x = torch.randn((2, 3, 200), generator=g, device="cuda").bfloat16()
    rows = ops.quantize_q8(x, group=64)
    assert rows.q.shape == (6, 200) and rows.lead == (2, 3)
    back = ops.dequantize_q8(rows)
    assert back.shape == x.shape
    want = (rows.q.float() * rows.scale.repeat_interleave(64, 1)[:, :200]).bfloat16().view(x.shape)
    torch.testing.assert_close(back, want, rtol=0, atol=0)
    # caller's buffers: int8 rows inside a wider tensor, scales with a longer row, output rows likewise
    q = torch.full((6, 256), 99, dtype=torch.int8, device="cuda")
    s = torch.full((6, 9), -1.0, device="cuda")
    mine = ops.quantize_q8(x, group=64, out=ops.Q8Rows(q[:, 8:208], s[:, :4], 64))
    torch.testing.assert_close(mine.q, rows.q, rtol=0, atol=0)
    torch.testing.assert_close(mine.scale, rows.scale, rtol=0, atol=0)
    assert bool((q[:, :8] == 99).all()) and bool((q[:, 208:] == 99).all()) and bool((s[:, 4:] == -1).all())
    wide = torch.zeros((6, 320), dtype=torch.bfloat16, device="cuda")
    ops.dequantize_q8(mine, out=wide[:, 16:216])
    torch.testing.assert_close(wide[:, 16:216], want.view(6, 200), rtol=0, atol=0)
    assert not bool(wide[:, :16].any()) and not bool(wide[:, 216:].any())


def test_residual_in_place_and_no_rows():
    from lastkv_b200 import ops

    g = _gen(6)
    x = torch.randn((16, 512), generator=g, device="cuda").bfloat16()
    r = torch.randn((16, 512), generator=g, device="cuda").bfloat16()
    w = torch.ones(512, device="cuda", dtype=torch.bfloat16)
    want = x + r
    h, _ = ops.rmsnorm_q8(x, w, 1e-6, r, residual_out=r)
    assert h.data_ptr() == r.data_ptr()
    torch.testing.assert_close(r, want, rtol=0, atol=0)
    none = ops.quantize_q8(x[:0])
    assert none.q.shape == (0, 512) and ops.dequantize_q8(none).shape == (0, 512)


def test_zeros_tiny_and_non_finite_values():
    from lastkv_b200 import ops

    x = torch.zeros((4, 256), dtype=torch.bfloat16, device="cuda")
    x[0, :128] = 1e-38      # a scale near the smallest normal number: the reciprocal would overflow
    x[0, 5] = -3e-38
    x[1, 130] = float("inf")
    x[2, 0] = float("nan")
    x[3, 7] = 3e38
    rows = ops.quantize_q8(x, group=128)
    v = ops.dequantize_q8(rows)
    assert rows.q[0, 5] == -127 and bool((rows.q[0, :5] == 42).all())
    assert rows.scale[0, 1] == 0 and not bool(rows.q[0, 128:].any())
    assert bool(torch.isnan(v[1, 128:]).all()) and not bool(v[1, :128].any())
    assert bool(torch.isnan(v[2, :128]).all()) and not bool(v[2, 128:].any())
    assert rows.q[3, 7] == 127 and bool(torch.isfinite(v[3]).all())
    w = torch.ones(256, dtype=torch.bfloat16, device="cuda")
    n = ops.dequantize_q8(ops.rmsnorm_q8(x, w, 1e-6))
    assert bool(torch.isnan(n[1, 128:]).all()) and bool(torch.isnan(n[2]).all())


def test_refusals():
    from lastkv_b200 import ops
    from lastkv_b200.contract import RMarinBackendContractError

    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: ops.quantize_q8(x, group=48),
                 lambda: ops.quantize_q8(x.float()),
                 lambda: ops.quantize_q8(x.cpu()),
                 lambda: ops.quantize_q8(x[:, :12]),             # not a multiple of 8
                 lambda: ops.quantize_q8(x[:, 1:33]),            # rows off the 16-byte grid
                 lambda: ops.quantize_q8(x.t()),
                 lambda: ops.quantize_q8(x, out=ops.Q8Rows.empty_for(x[:3], 64, 128)),
                 lambda: ops.silu_mul_q8(x[:, :24]),             # 12 columns
                 lambda: ops.rmsnorm_q8(x, w[:32], 1e-6),
                 lambda: ops.rmsnorm_q8(x, w.float(), 1e-6),
                 lambda: ops.rmsnorm_q8(x, w, 1e-6, x[:2]),
                 lambda: ops.rmsnorm_q8(torch.zeros((1, 32776), dtype=torch.bfloat16, device="cuda"),
                                        torch.zeros(32776, dtype=torch.bfloat16, device="cuda"), 1e-6),
                 lambda: ops.dequantize_q8(ops.quantize_q8(x), out=x[:2])):
        with pytest.raises(RMarinBackendContractError):
            call()


def test_rows_must_be_q8rows():
    from lastkv_b200 import ops
    from lastkv_b200.contract import RMarinBackendContractError

    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    for call in (lambda: ops.dequantize_q8(x), lambda: ops.quantize_q8(x, out=x)):
        with pytest.raises(RMarinBackendContractError):
            call()
