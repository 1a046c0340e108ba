"""SiLU-and-mul int8 rows over the gates' whole range, against the definition in 64 bits.

Tolerances as for the other int8 rows: the scale within 1e-5 (a chain of fewer than 100 fp32 roundings), every int8
within 0.504 of y / s.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def check(gate, up, group=32):
    from lastkv_b200 import ops

    rows = ops.silu_mul_q8(torch.cat((gate, up), 1), group=group)
    g, u = gate.double(), up.double()
    y = (g * torch.sigmoid(g) * u).view(gate.shape[0], -1, group)
    scale = y.abs().amax(-1, keepdim=True) / 127
    s = rows.scale.double()[..., None]
    q = rows.q.double().view(y.shape)
    assert bool(((s - scale).abs() <= 1e-5 * scale).all())
    assert bool(((y - q * scale).abs() <= 0.504 * scale).all())


@pytest.mark.parametrize("low", [-80.0, -87.0, -88.0, -88.5, -89.0, -95.0, -104.0, -120.0, -150.0])
def test_far_gates_of_large_ups(low):
    """silu is small there, but a large up makes the product an ordinary number."""
    g = torch.Generator(device="cuda").manual_seed(int(-low))
    gate = (low - torch.rand((4, 128), generator=g, device="cuda") * 4).bfloat16()
    up = ((torch.rand((4, 128), generator=g, device="cuda") + 0.5) * 2.0 ** 126).bfloat16()
    check(gate, up)
    check(gate, -up)


def test_ordinary_gates():
    """Gates whose products stay fp32's normal numbers, in order and mixed."""
    g = torch.Generator(device="cuda").manual_seed(1)
    gate = torch.linspace(-70, 100, 4096, device="cuda").bfloat16().view(4, 1024)
    up = ((torch.rand((4, 1024), generator=g, device="cuda") + 0.5) * 3).bfloat16()
    check(gate, up)
    check(gate[:, torch.randperm(1024, generator=g, device="cuda")], -up)


def test_non_finite_gates_and_ups():
    """Infinite and NaN products make their own group NaN, and no other."""
    from lastkv_b200 import ops

    inf, nan = float("inf"), float("nan")
    gate = torch.full((8, 128), 1.5, dtype=torch.bfloat16, device="cuda")
    up = torch.full((8, 128), -2.0, dtype=torch.bfloat16, device="cuda")
    for i, (a, b) in enumerate([(inf, 1.0), (-inf, 1.0), (nan, 1.0), (1.0, inf), (1.0, nan), (-100.0, -inf), (0.0, inf),
                                (inf, 0.0)]):
        gate[i, 40], up[i, 40] = a, b
    v = ops.dequantize_q8(ops.silu_mul_q8(torch.cat((gate, up), 1), group=32))
    assert bool(torch.isnan(v[:, 32:64]).all())
    assert bool(torch.isfinite(v[:, :32]).all()) and bool(torch.isfinite(v[:, 64:]).all())
    want = -2.0 * 1.5 / (1 + torch.exp(torch.tensor(-1.5, dtype=torch.float64)))
    assert bool(((v[:, 64:].double() - want).abs() <= 0.01 * abs(want)).all())
