"""Attention of single tokens over 8-bit and bf16 pages against its formula in 64 bits."""

import pytest
import torch

from lastkv_b200 import ops
from tests.q8_helpers import assert_within, attention, random_cache, row_keys

pytestmark = pytest.mark.gpu


def _cache(t):
    return ops.PagesQ8.from_codes(t["k"], t["v"], t["ks"], t["vs"])


def _q(seed, B, hq, d):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((B, hq, d), generator=g).bfloat16().cuda()


def _check(t, q, out, *, scale=None, out_scale=None, lse=None, what=""):
    for b in range(q.shape[0]):
        k, v = row_keys(t, b)
        s = q.shape[2] ** -0.5 if scale is None else scale
        ref, bound = attention(q[b:b + 1], k, v, s)
        if out_scale is not None:
            ref, bound = ref * out_scale[:, None], bound * out_scale.abs()[:, None] * (1 + 2 ** -20)
        assert_within(out[b:b + 1], ref, bound, f"{what} row {b}")
        if lse is not None:
            if not k.shape[0]:
                assert bool((lse[b] == float("-inf")).all())
                continue
            G = q.shape[1] // k.shape[1]
            x = torch.einsum("hd,nhd->hn", q[b].double(), k.repeat_interleave(G, 1)) * s
            # a score's rounding as in `attention`, a sum of n terms, the last multiplication
            off = torch.einsum("hd,nhd->hn", q[b].double().abs(), k.abs().repeat_interleave(G, 1)).amax(-1) * s
            want = torch.logsumexp(x, -1)
            tol = (4 * q.shape[2] * off + 2 * k.shape[0] + 4 * want.abs() + 16) * 2.0 ** -24
            assert bool(((lse[b].double() - want).abs() <= tol).all()), (lse[b], want)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (6, 3), (8, 2), (16, 2)])
def test_lengths_and_kinds_of_pages(d, hq, hkv):
    """One token to thousands; pages that end inside; none, an odd number, all and more than all pages in 8 bits."""
    lens = [1, 0, 16, 17, 31, 32, 33, 100, 257, 1000, 1000, 2049, 700]
    num_q8 = [1, 3, 0, 1, 1, 2, 2, 3, 17, 5, 62, 0, 1000]
    t = random_cache(hq * d, lens, num_q8, hkv, d)
    q = _q(1, len(lens), hq, d)
    lse = torch.empty((len(lens), hq), dtype=torch.float32, device="cuda")
    ws = ops.Workspace.for_decode(len(lens), hq, d, t["table"].shape[1])
    out = ops.decode_paged_q8(q, _cache(t), t["table"], t["seq_k"], num_q8=t["num_q8"], pool_k=t["pool_k"],
                              pool_v=t["pool_v"], workspace=ws, lse=lse)
    assert ws.error() == [0, 0, 0, 0]
    _check(t, q, out, lse=lse)


@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 4), (128, 8, 2)])
def test_every_page_in_8_bits_without_a_pool(d, hq, hkv):
    lens = [5, 0, 640, 1999]
    t = random_cache(7, lens, [10 ** 6] * 4, hkv, d)
    q = _q(2, 4, hq, d)
    out = ops.decode_paged_q8(q, _cache(t), t["table"], t["seq_k"])
    _check(t, q, out)
    again = ops.decode_paged_q8(q, _cache(t), t["table"], t["seq_k"], num_q8=t["num_q8"])
    assert torch.equal(out, again)


def test_splits_of_one_long_row():
    """A single row of 40000 keys: many splits, then one split by a workspace that holds no more."""
    t = random_cache(9, [40000], [2300], 2, 128)
    q, cache = _q(3, 1, 8, 128), _cache(t)
    args = (q, cache, t["table"], t["seq_k"])
    kw = dict(num_q8=t["num_q8"], pool_k=t["pool_k"], pool_v=t["pool_v"])
    lse = torch.empty((1, 8), dtype=torch.float32, device="cuda")
    _check(t, q, ops.decode_paged_q8(*args, **kw, lse=lse), lse=lse)
    small = ops.Workspace(256 + 8 * 129 * 4 + 256)
    _check(t, q, ops.decode_paged_q8(*args, **kw, lse=lse, workspace=small), lse=lse)
    a, b = ops.decode_paged_q8(*args, **kw), ops.decode_paged_q8(*args, **kw, l2_keep=True)
    assert torch.equal(a, b)


def test_strides_scales_and_buffers():
    """q and out as slices of wider rows, tables wider than they are used, a scale per head, another softmax scale."""
    B, hq, hkv, d = 5, 8, 4, 64
    t = random_cache(11, [40, 300, 64, 15, 500], [1, 9, 4, 0, 20], hkv, d)
    wide_q = torch.zeros((B, 3, hq, d), dtype=torch.bfloat16, device="cuda")
    wide_q[:, 1] = _q(4, B, hq, d)
    q = wide_q[:, 1]
    wide_o = torch.full((B, 2, hq, d), 3.0, dtype=torch.bfloat16, device="cuda")
    table = torch.full((B + 2, t["table"].shape[1] + 9), -7, dtype=torch.int32, device="cuda")
    table[:B, :t["table"].shape[1]] = t["table"]
    f = torch.tensor([0.5, -2.0, 1.0, 3.0, 0.0, 1.5, 0.25, 8.0], device="cuda")
    out = ops.decode_paged_q8(q, _cache(t), table, t["seq_k"], num_q8=t["num_q8"], pool_k=t["pool_k"],
                              pool_v=t["pool_v"], out=wide_o[:, 1], out_scale=f, softmax_scale=0.3,
                              max_pages=t["table"].shape[1])
    assert out.data_ptr() == wide_o[:, 1].data_ptr()
    _check(t, q, out, scale=0.3, out_scale=f.double())
    assert bool((wide_o[:, 0] == 3).all())


def test_what_lies_behind_the_end_has_no_weight():
    """NaN and infinities in 8-bit blocks (their scales) and bf16 rows past a row's last token."""
    hkv, d = 2, 64
    lens, num_q8 = [20, 24, 40, 53, 3], [2, 2, 1, 2, 1]
    t = random_cache(13, lens, num_q8, hkv, d)
    q = _q(5, len(lens), 4, d)
    args = lambda: dict(num_q8=t["num_q8"], pool_k=t["pool_k"], pool_v=t["pool_v"])  # noqa: E731
    clean = ops.decode_paged_q8(q, _cache(t), t["table"], t["seq_k"], **args())
    page = lambda b, j: int(t["table"][b, j])  # noqa: E731
    for b, j, half in ((1, 1, 1), (4, 0, 1)):  # tokens 24-31 of row 1, 8-15 of row 4
        t["ks"][page(b, j), half], t["vs"][page(b, j), half] = float("nan"), float("inf")
    t["ks"][page(0, 1), 1] = float("inf")
    t["pool_k"][page(2, 2), 8:], t["pool_v"][page(2, 2), 8:] = float("inf"), float("nan")
    t["pool_v"][page(3, 3), 5:] = float("nan")
    dirty = ops.decode_paged_q8(q, _cache(t), t["table"], t["seq_k"], **args())
    assert torch.equal(clean, dirty)
    _check(t | {"ks": t["ks"].nan_to_num(1, posinf=1), "vs": t["vs"].nan_to_num(1, posinf=1)}, q, clean)


def test_a_value_that_is_not_a_number_is_seen():
    t = random_cache(15, [600, 600], [20, 20], 1, 128)
    q = _q(6, 2, 4, 128)
    t["vs"][int(t["table"][1, 7]), 0] = float("nan")
    out = ops.decode_paged_q8(q, _cache(t), t["table"], t["seq_k"], num_q8=t["num_q8"], pool_k=t["pool_k"],
                              pool_v=t["pool_v"])
    assert bool(out[0].isfinite().all()) and bool(out[1].isnan().all())
    t["ks"][int(t["table"][0, 3]), 1] = float("inf")  # 0 * inf in the scores
    out = ops.decode_paged_q8(q, _cache(t), t["table"], t["seq_k"], num_q8=t["num_q8"], pool_k=t["pool_k"],
                              pool_v=t["pool_v"])
    assert bool(out.isnan().all())


def test_large_scores_and_zero_blocks():
    """Scores far apart (weights that underflow), blocks whose scale is zero."""
    t = random_cache(17, [300, 90], [12, 5], 2, 64, spread=40.0)
    t["ks"][:3], t["vs"][2:5] = 0.0, 0.0
    q = _q(7, 2, 2, 64)
    out = ops.decode_paged_q8(q, _cache(t), t["table"], t["seq_k"], num_q8=t["num_q8"], pool_k=t["pool_k"],
                              pool_v=t["pool_v"])
    _check(t, q, out)


@pytest.mark.parametrize("lens", [[300, 90], [9000, 20]])
@pytest.mark.parametrize("power", [-80, 90])
def test_values_of_any_size(lens, power):
    """Scales from 2^-90 up: the weights carry them, the sum of weights does not."""
    t = random_cache(27, lens, [10000, 10000], 2, 128)
    t["vs"] *= 2.0 ** power
    q = _q(8, 2, 4, 128)
    out = ops.decode_paged_q8(q, _cache(t), t["table"], t["seq_k"], num_q8=t["num_q8"])
    _check(t, q, out)


def test_pages_that_are_not_there_read_as_zeros():
    hkv, d = 2, 128
    t = random_cache(19, [100, 100], [4, 4], hkv, d)
    q = _q(8, 2, 4, d)
    ws = ops.Workspace.for_decode(2, 4, d, t["table"].shape[1])
    good = ops.decode_paged_q8(q, _cache(t), t["table"], t["seq_k"], num_q8=t["num_q8"], pool_k=t["pool_k"],
                               pool_v=t["pool_v"], workspace=ws)
    assert ws.error()[0] == 0
    bad = t["table"].clone()
    bad[1, 1], bad[1, 5] = t["k"].shape[0], -3
    out = ops.decode_paged_q8(q, _cache(t), bad, t["seq_k"], num_q8=t["num_q8"], pool_k=t["pool_k"],
                              pool_v=t["pool_v"], workspace=ws)
    e = ws.error()
    assert e[0] == 2 and e[1] == 11 and e[3] in (t["k"].shape[0], -3)
    assert torch.equal(out[0], good[0])
    z = {n: x.clone() for n, x in t.items()}
    z["ks"][int(t["table"][1, 1])] = z["vs"][int(t["table"][1, 1])] = 0
    z["pool_k"][int(t["table"][1, 5])] = z["pool_v"][int(t["table"][1, 5])] = 0
    _check(z, q, out)
    ws.clear_error()
    # bf16 columns without a pool
    out = ops.decode_paged_q8(q, _cache(t), t["table"], t["seq_k"], num_q8=t["num_q8"], workspace=ws)
    assert ws.error()[0] == 2 and bool(out.isfinite().all())


def test_pages_past_4_gib():
    """Codes at byte offsets over 2^32."""
    hkv, d = 8, 128
    page = hkv * 2 * 16 * d
    pages = 2 ** 32 // page + 64
    codes = torch.zeros((pages, hkv, 2, 16 * d), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((pages, hkv, 4), device="cuda")
    t = random_cache(21, [500], [32], hkv, d, extra=0)
    small = _cache(t)
    first = pages - small.num_pages
    codes[first:], scales[first:] = small.codes, small.scales
    q = _q(9, 1, 16, d)
    a = ops.decode_paged_q8(q, small, t["table"], t["seq_k"])
    b = ops.decode_paged_q8(q, ops.PagesQ8(codes, scales), t["table"] + first, t["seq_k"])
    assert torch.equal(a, b)
    _check(t, q, a)


def test_captured_and_replayed_with_new_lengths():
    """A captured call follows the lengths, tables and pages that are there when it is replayed."""
    t = random_cache(23, [900, 900, 900], [30, 30, 30], 2, 128)
    q, cache = _q(10, 3, 8, 128), _cache(t)
    ws = ops.Workspace.for_decode(3, 8, 128, t["table"].shape[1])
    seq, nq, out = t["seq_k"].clone(), t["num_q8"].clone(), torch.empty_like(q)

    def call():
        ops.decode_paged_q8(q, cache, t["table"], seq, num_q8=nq, pool_k=t["pool_k"], pool_v=t["pool_v"], out=out,
                            workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([900, 1, 0], [17, 480, 481], [899, 33, 500]):
        seq.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        _check(t | {"seq_k": seq}, q, out)


def test_refusals():
    from lastkv_b200.contract import RMarinBackendContractError as Refused

    t = random_cache(25, [40], [1], 2, 64)
    q, cache = _q(11, 1, 4, 64), _cache(t)

    def call(**kw):
        a = dict(q=q, cache=cache, block_table=t["table"], seq_k=t["seq_k"], num_q8=t["num_q8"], pool_k=t["pool_k"],
                 pool_v=t["pool_v"]) | kw
        return ops.decode_paged_q8(a.pop("q"), a.pop("cache"), a.pop("block_table"), a.pop("seq_k"), **a)

    call()
    for kw, word in ((dict(q=q.float()), "q must"), (dict(q=_q(1, 1, 6, 64)), "GQA"), (dict(q=_q(1, 1, 4, 128)), "head_dim"),
                     (dict(pool_k=None), "together"), (dict(pool_k=t["pool_k"].float()), "bf16"),
                     (dict(block_table=t["table"].long()), "block_table"), (dict(max_pages=99), "max_pages"),
                     (dict(seq_k=t["seq_k"].long()), "seq_k"), (dict(num_q8=t["num_q8"][:0]), "num_q8"),
                     (dict(seq_k=t["seq_k"].cpu()), "CUDA"), (dict(out=q.float()), "out"),
                     (dict(out_scale=torch.ones(3, device="cuda")), "out_scale"),
                     (dict(lse=torch.ones(3, device="cuda")), "lse"),
                     (dict(cache=cache._replace(scales=cache.scales[:1])), "scales"),
                     (dict(cache=cache._replace(codes=cache.codes[:, :, :, ::2])), "codes"),
                     (dict(cache=tuple(cache)), "PagesQ8"), (dict(workspace=ops.Workspace(0)), "workspace")):
        with pytest.raises(Refused, match=word):
            call(**kw)
