"""int8 rows whose inputs the call just before wrote: every input is read after that call has finished."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden", [512, 4096, 16384])
@pytest.mark.parametrize("maker", ["dequantize", "product"])
def test_norm_weight_from_the_call_before(hidden, maker):
    """A [1, H] result of the library as the norm's weight, as in a conditional norm, in buffers that hold
    another weight until then."""
    from lastkv_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(hidden)
    x = torch.randn((3, hidden), generator=g, device="cuda").bfloat16()
    weights = [(torch.rand((1, hidden), generator=g, device="cuda") + 0.5).bfloat16() for _ in range(2)]
    if maker == "dequantize":
        rows = [ops.quantize_q8(w) for w in weights]

        def make(i, out):
            ops.dequantize_q8(rows[i], out=out)
    else:
        cond = [torch.randn((1, 256), generator=g, device="cuda").bfloat16() for _ in range(2)]
        w4 = ops.w4_quantize(torch.randn((hidden, 256), generator=g, device="cuda").bfloat16())

        def make(i, out):
            ops.w4_linear(cond[i], w4, out=out)
    weight = torch.empty((1, hidden), dtype=torch.bfloat16, device="cuda")
    want = []
    for i in range(2):
        make(i, weight)
        torch.cuda.synchronize()
        want.append(ops.rmsnorm_q8(x, weight, 1e-5))
    torch.cuda.synchronize()
    assert not torch.equal(want[0].q, want[1].q)
    got = []
    for i in range(200):
        make(i % 2, weight)
        got.append(ops.rmsnorm_q8(x, weight, 1e-5))
    for i, rows_ in enumerate(got):
        assert torch.equal(rows_.q, want[i % 2].q) and torch.equal(rows_.scale, want[i % 2].scale), i
