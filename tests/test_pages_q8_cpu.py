"""8-bit pages, their attention and beam search: the codes' layout and the calls that are refused."""

import ctypes

import pytest
import torch

from lastkv_b200 import ops
from lastkv_b200.contract import RMarinBackendContractError

Refused = RMarinBackendContractError


@pytest.mark.parametrize("d", [64, 128])
def test_codes_layout_round_trip(d):
    g = torch.Generator().manual_seed(d)
    n, h = 3, 2
    k, v = (torch.randint(-127, 128, (n, 16, h, d), generator=g).to(torch.int8) for _ in range(2))
    ks, vs = torch.rand((n, 2, h), generator=g), torch.rand((n, 2, h), generator=g)
    c = ops.PagesQ8.from_codes(k, v, ks, vs)
    assert (c.num_pages, c.num_kv_heads, c.head_dim) == (n, h, d)
    for a, b in zip(c.to_codes(), (k, v, ks, vs)):
        assert torch.equal(a, b)
    raw = c.codes.int() - 128
    for r in range(16):
        for x in range(d):  # the order that include/lastkv_b200.h gives
            half, tile = r // 8, x // 16
            at = tile // 2 * 512 + (4 * (r % 8) + x // 2 % 4) * 16 + (tile % 2 * 2 + half) * 4 + 2 * (x % 2) + x // 8 % 2
            assert torch.equal(raw[:, :, 0, at], k[:, r, :, x].int())
            at = tile // 2 * 512 + (4 * (x % 8) + r // 2 % 4) * 16 + (tile % 2 * 2 + half) * 4 + 2 * (r % 2) + x // 8 % 2
            assert torch.equal(raw[:, :, 1, at], v[:, r, :, x].int())
    assert torch.equal(c.scales[..., 0], ks[:, 0]) and torch.equal(c.scales[..., 3], vs[:, 1])


def _pages(d=64, pages=2, h=2):
    return ops.PagesQ8.empty(pages, h, d, device="cpu")


def test_wrong_pages_are_refused():
    with pytest.raises(Refused, match="head_dim"):
        ops.PagesQ8.empty(2, 2, 96, device="cpu")
    k = torch.zeros((2, 16, 2, 64), dtype=torch.int8)
    s = torch.zeros((2, 2, 2))
    with pytest.raises(Refused, match="codes"):
        ops.PagesQ8.from_codes(k.short(), k, s, s)
    with pytest.raises(Refused, match="codes"):
        ops.PagesQ8.from_codes(k[:, :8], k[:, :8], s, s)
    with pytest.raises(Refused, match="scales"):
        ops.PagesQ8.from_codes(k, k, s[:1], s)


def test_calls_off_the_gpu_are_refused():
    """Every tensor has to be on the current device; nothing reaches a kernel otherwise."""
    pool = torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16)
    ids = torch.zeros(1, dtype=torch.int32)
    q = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    table = torch.zeros((1, 2), dtype=torch.int32)
    for call in (lambda: ops.quantize_pages(pool, pool, ids, _pages(), ids),
                 lambda: ops.dequantize_pages(_pages(), ids, pool, pool, ids),
                 lambda: ops.decode_paged_q8(q, _pages(), table, ids),
                 lambda: ops.prefill_paged_q8(q, _pages(), table, ids, torch.zeros(2, dtype=torch.int32), 1),
                 lambda: ops.reorder_pages(pool, ids, ids),
                 lambda: ops.beam_select(torch.zeros((2, 8)), torch.zeros((1, 2)))):
        with pytest.raises(Refused, match="CUDA"):
            call()


def _lib():
    from lastkv_b200 import _capi, build

    build.build()
    return _capi.load()


def _buf(n=4096):
    """A host address that is never dereferenced, aligned to 256 bytes."""
    b = ctypes.create_string_buffer(n + 256)
    return b, (ctypes.addressof(b) + 255) & ~255


def test_page_calls_check_their_arguments_on_the_host():
    lib = _lib()
    keep, a = _buf()
    quant = lib.lkv_q8_quantize_pages
    assert quant(a, a, 4, a, None, a, a, 4, a, 1, 2, 96, None, None) == 2     # head_dim
    assert quant(a, a, 4, a, None, a, a, 4, a, 1, 0, 64, None, None) == 1     # no heads
    assert quant(a, None, 4, a, None, a, a, 4, a, 1, 2, 64, None, None) == 1  # no values
    assert quant(a + 8, a, 4, a, None, a, a, 4, a, 1, 2, 64, None, None) == 1  # alignment
    assert quant(a, a, 4, None, None, a, a, 4, a, 1, 2, 64, None, None) == 1  # no list
    assert quant(a, a, 4, a, None, a, a, 4, a, -1, 2, 64, None, None) == 1
    assert quant(a, a, 4, None, None, a, a, 4, None, 0, 2, 64, None, None) == 0  # nothing to do
    back = lib.lkv_q8_dequantize_pages
    assert back(a, a, 4, a, a, a, 4, a, 1, 300, 64, None, None) == 1
    assert back(a, a + 4, 4, a, a, a, 4, a, 1, 2, 64, None, None) == 1
    assert back(a, a, 4, None, a, a, 4, None, 0, 2, 64, None, None) == 0
    pools, sizes, counts = (ctypes.c_void_p * 1)(a), (ctypes.c_int64 * 1)(64), (ctypes.c_int64 * 1)(4)
    move = lib.lkv_reorder_pages
    assert move(pools, sizes, counts, 0, a, a, 1, 1, 0, None, None) == 1
    assert move(pools, sizes, counts, 9, a, a, 1, 1, 0, None, None) == 1
    assert move(pools, sizes, counts, 1, a, a, 2049, 1, 0, None, None) == 2
    assert move(pools, sizes, counts, 1, a, a, 1, 2, 0, None, None) == 1       # layers without a stride
    assert move(pools, sizes, counts, 1, None, a, 1, 1, 0, None, None) == 1
    assert move(pools, (ctypes.c_int64 * 1)(24), counts, 1, a, a, 1, 1, 0, None, None) == 1
    assert move((ctypes.c_void_p * 1)(a + 8), sizes, counts, 1, a, a, 1, 1, 0, None, None) == 1
    assert move(pools, sizes, counts, 1, None, None, 0, 1, 0, None, None) == 0


def test_attention_calls_check_their_arguments_on_the_host():
    lib = _lib()
    keep, a = _buf()

    def decode(q=a, q_row=256, codes=a, out=a, out_row=256, hq=4, hkv=2, d=64, pool=None, pages=0, ws=a, ws_bytes=4096,
               batch=1, width=2, num_q8=None):
        return lib.lkv_decode_paged_q8(q, q_row, codes, a, 4, pool, pool, pages, a, width, num_q8, a, out, out_row,
                                       None, None, batch, hq, hkv, d, width, 1.0, ws, ws_bytes, 0, None)

    assert decode(d=96) == 2
    assert decode(hq=6) == 2 and decode(hq=5) == 1
    assert decode(q=None) == 1 and decode(codes=None) == 1 and decode(out=None) == 1
    assert decode(q=a + 2) == 1 and decode(q_row=255) == 1 and decode(out_row=128) == 1 and decode(codes=a + 8) == 1
    assert decode(ws=None) == 6 and decode(ws=a + 16) == 6 and decode(ws_bytes=256) == 6
    assert decode(width=-1) == 1 and decode(batch=-1) == 1
    assert decode(batch=0) == 0

    def prefill(stage=a, width=2, codes=a, scales=a, q=a, q_row=256, batch=1, total=1, d=64, hq=4, staged=0, splits=1):
        return lib.lkv_prefill_paged_q8(q, q_row, codes, scales, 4, stage, stage, width, staged, None, None, 0, a, 2,
                                        None, a, a, a, 256, None, None, batch, total, 1, hq, 2, d, 2, 1, 1.0, splits, None,
                                        None, None, None)

    assert prefill(d=96) == 2 and prefill(hq=6) == 2
    assert prefill(stage=None) == 1 and prefill(width=0) == 1 and prefill(scales=None) == 1
    assert prefill(codes=None) == 1 and prefill(codes=a + 8) == 1 and prefill(width=3) == 1  # wider than the table
    assert prefill(q=a + 4) == 1 and prefill(q_row=252) == 1
    assert prefill(splits=2) == 1 and prefill(splits=9) == 2  # no partials; too many
    assert prefill(batch=0) == 0 and prefill(total=0) == 0


def test_beam_select_checks_its_arguments_on_the_host():
    lib = _lib()
    keep, a = _buf()

    def select(logits=a, fp32=0, finished=None, eos=-1, batch=1, beams=2, vocab=8, n=2, scores=a):
        return lib.lkv_beam_select(logits, vocab, fp32, scores, finished, eos, batch, beams, vocab, n, a, a, a, a, a,
                                   4096, None)

    assert select(n=0) == 1 and select(n=9) == 1 and select(beams=0) == 1 and select(vocab=0) == 1
    assert select(vocab=100, n=33) == 2 and select(beams=65) == 2 and select(batch=40000) == 2
    assert select(logits=None) == 1 and select(logits=a + 1) == 1 and select(logits=a + 2, fp32=1) == 1
    assert select(scores=None) == 1
    assert select(finished=a) == 1 and select(finished=a, eos=8) == 1
    assert select(batch=0) == 0
    assert lib.lkv_beam_workspace_bytes(0, 4) == 0 and lib.lkv_beam_workspace_bytes(4, 0) == 0
    assert lib.lkv_beam_workspace_bytes(4, 4) >= 4 * (4 * 8 + 8)
