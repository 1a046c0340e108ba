"""Which calls of 4-bit projections take int8 rows."""

import pytest
import torch


@pytest.mark.parametrize("group", [32, 64, 128])
def test_int8_rows_up_to_a_groups_width(group):
    from lastkv_b200 import ops
    from lastkv_b200.hf import QuantizedLinears

    w = ops.W4Weight(torch.zeros(2048 + 64 * (128 // group), dtype=torch.uint8), 32, 128, group)
    took = [rows for rows in range(1, 300) if QuantizedLinears(w, None, True).takes_int8(rows)]
    assert took == list(range(1, group + 1))
    assert not any(QuantizedLinears(w, None, False).takes_int8(rows) for rows in range(1, 300))
