"""w4_linear looks at the packed weight and the error word before it launches anything; these checks need no GPU."""

import pytest
import torch


@pytest.fixture(scope="module", autouse=True)
def built():
    from lastkv_b200 import build

    build.build()


def packed(nbytes, dtype=torch.uint8, device="cpu"):
    return torch.zeros(nbytes, dtype=dtype, device=device)


@pytest.mark.parametrize("tensor,n,k,group", [
    (packed(2112 - 1), 32, 128, 128),           # a byte short
    (packed(2 * 2112), 32, 128, 128),           # another weight's
    (packed(2112), 33, 128, 128),               # n past the packed rows
    (packed(2112), 32, 256, 128),               # k past the packed columns
    (packed(2112), 32, 128, 64),                # fewer scales than the groups need
    (packed(2112, torch.int8), 32, 128, 128),
    (packed(2 * 2112)[::2], 32, 128, 128),
    (packed(0), 0, 128, 128),
    (packed(0), 32, 12, 128)])
def test_packed_bytes_must_be_the_weights(tensor, n, k, group):
    from lastkv_b200 import ops
    from lastkv_b200.contract import RMarinBackendContractError

    w = ops.W4Weight(tensor, n, k, group)
    rows = ops.Q8Rows(torch.zeros((2, k), dtype=torch.int8), torch.zeros((2, -(-k // group))), group)
    for x in (torch.zeros((2, k), dtype=torch.bfloat16), rows):
        with pytest.raises(RMarinBackendContractError, match="weight.packed must be the"):
            ops.w4_linear(x, w)


def test_packed_weight_must_be_on_the_rows_gpu():
    from lastkv_b200 import ops
    from lastkv_b200.contract import RMarinBackendContractError

    for device in ("cpu", "meta"):
        with pytest.raises(RMarinBackendContractError, match="on x's GPU"):
            ops.w4_linear(torch.zeros((2, 128), dtype=torch.bfloat16), ops.W4Weight(packed(2112, device=device), 32, 128, 128))
    with pytest.raises(RMarinBackendContractError, match="W4Weight"):
        ops.w4_linear(torch.zeros((2, 128), dtype=torch.bfloat16), (packed(2112), 32, 128, 128))


def test_error_word_is_four_device_words():
    from lastkv_b200 import ops
    from lastkv_b200.contract import RMarinBackendContractError

    assert ops._err_ptr(None) is None
    for bad in (torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int64, device="meta"),
                torch.zeros(3, dtype=torch.int32, device="meta")):
        with pytest.raises(RMarinBackendContractError):
            ops._err_ptr(bad)
