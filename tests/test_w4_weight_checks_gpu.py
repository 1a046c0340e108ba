"""w4_linear refuses a packed weight, or an error word, that its kernels would read or write out of range."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("tokens", [4, 200])
def test_refusals(tokens, int8):
    from lastkv_b200 import ops
    from lastkv_b200.contract import RMarinBackendContractError

    g = torch.Generator(device="cuda").manual_seed(1)
    w = ops.w4_quantize(torch.randn((64, 256), generator=g, device="cuda").bfloat16())
    x = torch.randn((tokens, 256), generator=g, device="cuda").bfloat16()
    x = ops.quantize_q8(x) if int8 else x
    want = ops.w4_linear(x, w)
    bad = [w._replace(packed=w.packed.cpu()), w._replace(packed=w.packed[:-16]), w._replace(n=96),
           w._replace(packed=w.packed.view(torch.int8)), w._replace(packed=w.packed.repeat(2)[::2]),
           w._replace(group=64), tuple(w)]
    for weight in bad:
        with pytest.raises(RMarinBackendContractError):
            ops.w4_linear(x, weight)
    for word in (torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32, device="cuda"),
                 torch.zeros(4, dtype=torch.float32, device="cuda")):
        with pytest.raises(RMarinBackendContractError):
            ops.w4_linear(x, w, error_word=word)
    copy = w._replace(packed=w.packed.clone())
    torch.cuda.synchronize()  # a packed weight that w4_pack did not write is read early (see W4Weight)
    assert torch.equal(ops.w4_linear(x, copy), want)
