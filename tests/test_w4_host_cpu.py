"""Argument checks of the int8 rows, the 4-bit products and the step plan that need no GPU."""

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from lastkv_b200 import _capi, build

    build.build()
    return _capi.load()


def test_packed_sizes(lib):
    # 32 x 128 blocks of 2048 bytes of codes and 64 bytes of scales per group of columns
    assert lib.lkv_w4_bytes(32, 128, 128) == 2112
    assert lib.lkv_w4_bytes(33, 136, 128) == 4 * 2112
    assert lib.lkv_w4_bytes(1, 8, 64) == 2048 + 128
    assert lib.lkv_w4_bytes(1, 8, 32) == 2048 + 256
    assert lib.lkv_w4_bytes(28672, 4096, 128) == 896 * 32 * 2112
    for bad in ((0, 128, 128), (32, 0, 128), (32, 12, 128), (32, 128, 16), (-1, 128, 128)):
        assert lib.lkv_w4_bytes(*bad) == 0


def test_products_validate_before_any_cuda_call(lib):
    def bf16(tokens=1, n=64, k=128, group=128, x=16, packed=16, y=16, x_row=128, y_row=64):
        return lib.lkv_w4_linear(x, x_row, packed, None, y, y_row, tokens, n, k, group, None, None)

    def int8(tokens=1, scale=16, scale_row=1, q=8, q_row=128):
        return lib.lkv_w4_linear_q8(q, q_row, scale, scale_row, 16, None, 16, 64, tokens, 64, 128, 128, None, None)

    assert bf16(tokens=0) == 0
    assert bf16(group=48) == 2
    assert bf16(tokens=-1) == 1 and bf16(k=12) == 1 and bf16(n=0) == 1
    assert bf16(x=None) == 1 and bf16(packed=None) == 1 and bf16(y=None) == 1
    assert bf16(x=8) == 1 and bf16(packed=8) == 1           # off the 16-byte grid
    assert bf16(tokens=2, x_row=120) == 1 and bf16(tokens=2, y_row=63) == 1 and bf16(tokens=2, x_row=132) == 1
    assert int8(tokens=0) == 0
    assert int8(scale=None) == 1 and int8(q=4) == 1 and int8(tokens=2, q_row=132) == 1
    assert int8(tokens=2, scale_row=0) == 1
    assert lib.lkv_w4_pack(None, 64, 16, 1, 32, 128, 128, 16, None) == 1
    assert lib.lkv_w4_pack(16, 64, 16, 1, 32, 128, 96, 16, None) == 2
    assert lib.lkv_w4_pack(16, 60, 16, 1, 32, 128, 128, 16, None) == 1


def test_rows_validate_before_any_cuda_call(lib):
    def plain(rows=2, cols=64, group=32, x=16, x_row=64, q=8, q_row=64, scale=4, scale_row=2):
        return lib.lkv_quantize_q8(x, x_row, q, q_row, scale, scale_row, rows, cols, group, None)

    assert plain(rows=0) == 0
    assert plain(group=16) == 2 and plain(rows=1 << 30, cols=1 << 20) == 2
    assert plain(rows=-1) == 1 and plain(cols=12) == 1 and plain(cols=0) == 1
    assert plain(x=None) == 1 and plain(q=None) == 1 and plain(scale=None) == 1
    assert plain(x=8) == 1 and plain(q=4) == 1 and plain(x_row=56) == 1 and plain(x_row=68) == 1
    assert plain(scale_row=1) == 1
    assert lib.lkv_silu_mul_q8(16, 96, 8, 64, 4, 2, 2, 64, 32, None) == 1  # a row holds gate and up
    assert lib.lkv_rmsnorm_q8(16, 32776, None, 0, None, 0, 16, 1e-6, 8, 32776, 4, 257, 1, 32776, 128, None) == 2
    assert lib.lkv_rmsnorm_q8(16, 64, 16, 64, None, 0, 16, 1e-6, 8, 64, 4, 2, 1, 64, 32, None) == 1  # no residual_out
    assert lib.lkv_dequantize_q8(8, 64, 4, 2, None, 64, 2, 64, 32, None) == 1


def test_plan_validates_before_any_cuda_call(lib):
    def plan(batch=1, stride=7, slots=2, most=100, chunk=32, layers=1, width=11, tokens=1, ptr=16):
        return lib.lkv_plan_step(ptr, ptr, ptr, batch, ptr, stride, slots, most, chunk, ptr, layers, 1, 1, width,
                                 tokens, *([ptr] * 9), None, None)

    assert plan(batch=0) == 0
    assert plan(ptr=None) == 1
    for bad in (dict(batch=-1), dict(stride=6), dict(slots=0), dict(most=0), dict(chunk=24), dict(chunk=0),
                dict(layers=0), dict(width=6), dict(tokens=-1)):
        assert plan(**bad) == 1, bad


def test_wrappers_refuse_cpu_tensors():
    from lastkv_b200 import ops
    from lastkv_b200.contract import RMarinBackendContractError

    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    rows = ops.Q8Rows(torch.zeros((2, 64), dtype=torch.int8), torch.zeros((2, 1)), 128)
    w = ops.W4Weight(torch.zeros(2112, dtype=torch.uint8), 32, 64, 128)
    for call in (lambda: ops.rmsnorm_q8(x, x[0], 1e-6), lambda: ops.silu_mul_q8(x), lambda: ops.quantize_q8(x),
                 lambda: ops.dequantize_q8(rows), lambda: ops.w4_linear(x, w), lambda: ops.w4_linear(rows, w),
                 lambda: ops.w4_pack(torch.zeros((32, 32), dtype=torch.uint8), x[:, :1]),
                 lambda: ops.w4_quantize(x), lambda: ops.w4_quantize(x[:, :12]), lambda: ops.w4_quantize(x, 16),
                 lambda: ops.StepPlan(1, 1, torch.zeros((1, 4), dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                                      chunk_size=16, max_sequence_tokens=64, scratch_src_page=0,
                                      scratch_ring_page=0)):
        with pytest.raises(RMarinBackendContractError):
            call()
