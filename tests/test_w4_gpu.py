"""Products with 4-bit weights (lkv_w4_pack, lkv_w4_linear, lkv_w4_linear_q8) against the definition in 64 bits.

Tolerance per output: one rounding to bf16 (2^-8 of the result) and the fp32 sums.  Every product x * c is exact in
fp32 (bf16 x 4 bits, or int8 x 4 bits summed in int32); the tensor cores add at least eight products at a time, and
each step and each scaled group rounds or truncates once, so the sums are off by at most
(K / 8 + 4 K / G + 32) * 2^-23 of sum |x| |w|.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def make_weight(n, k, group, g):
    u = torch.randint(0, 16, (n, k), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    scales = ((torch.rand((n, -(-k // group)), generator=g, device="cuda") + 0.5) * 0.05).bfloat16()
    codes = u[:, 0::2] | (u[:, 1::2] << 4)
    dense = (u.double() - 8) * scales.double().repeat_interleave(group, 1)[:, :k]
    return codes, scales, dense


def make_x(t, k, group, int8, g):
    from lastkv_b200 import ops

    if not int8:
        x = torch.randn((t, k), generator=g, device="cuda").bfloat16()
        return x, x.double()
    pitch = -(-k // 16) * 16
    q = torch.randint(-127, 128, (t, pitch), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)[:, :k]
    s = torch.rand((t, -(-k // group)), generator=g, device="cuda") + 0.1
    return ops.Q8Rows(q, s, group), q.double() * s.double().repeat_interleave(group, 1)[:, :k]


def check(y, x64, w64, group, bias=None):
    K = x64.shape[1]
    ref = x64 @ w64.T
    size = x64.abs() @ w64.abs().T
    if bias is not None:
        ref = ref + bias.double()
        size = size + bias.double().abs()
    tol = 2.0 ** -8 * ref.abs() + (K / 8 + 4 * K / group + 32) * 2.0 ** -23 * size
    off = (y.double() - ref).abs()
    assert bool((off <= tol).all()), f"worst {float((off / tol.clamp(min=1e-30)).max()):.2f} of the tolerance"


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(sum(k * 7919 ** i for i, k in enumerate(key)) % (1 << 31))


SHAPES = [(1, 64, 128), (1, 1, 8), (3, 100, 72), (8, 768, 768), (8, 4096, 4096), (9, 130, 1544), (16, 2055, 264),
          (17, 64, 4096), (33, 1003, 1544), (40, 4096, 136), (64, 6144, 512), (65, 300, 2048), (128, 129, 1160),
          (200, 1000, 776), (256, 768, 2048), (300, 2048, 768), (1030, 520, 392), (70, 3000, 1544),
          (100, 2055, 392), (50, 5000, 136), (400, 1500, 8), (129, 2600, 4096), (2000, 257, 264)]


@pytest.mark.parametrize("t,n,k", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("int8", [False, True])
def test_matches_definition(t, n, k, group, int8):
    from lastkv_b200 import ops

    g = _gen(t, n, k, group, int8)
    codes, scales, w64 = make_weight(n, k, group, g)
    x, x64 = make_x(t, k, group, int8, g)
    w = ops.w4_pack(codes, scales, group)
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    check(ops.w4_linear(x, w, error_word=err), x64, w64, group)
    assert err.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("t,n", [(1, 203), (8, 203), (20, 203), (90, 203), (300, 203),
                                 (60, 2403), (100, 2402), (300, 2403), (290, 2402)])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("off", [8, 16])
def test_bias_strides_and_untouched_neighbours(t, n, int8, off):
    from lastkv_b200 import ops

    k, group = 1032, 64
    g = _gen(t, int8, n, off)
    codes, scales, w64 = make_weight(n, k, group, g)
    wide_c = torch.zeros((n, k // 2 + 7), dtype=torch.uint8, device="cuda")
    wide_c[:, : k // 2] = codes
    w = ops.w4_pack(wide_c[:, : k // 2], scales, group)  # codes in a wider tensor
    bias = torch.randn(n, generator=g, device="cuda").bfloat16()
    x, x64 = make_x(t, k, group, int8, g)
    if int8:
        q = torch.full((t, k + 40), 55, dtype=torch.int8, device="cuda")
        q[:, off:k + off] = x.q
        s = torch.full((t, x.scale.shape[1] + 3), float("nan"), device="cuda")
        s[:, :-3] = x.scale
        x = ops.Q8Rows(q[:, off:k + off], s[:, :-3], group)
    else:
        xw = torch.full((t, k + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
        xw[:, off:k + off] = x
        x = xw[:, off:k + off]
    out = torch.full((t + 1, n + 5), 7.0, dtype=torch.bfloat16, device="cuda")
    y = ops.w4_linear(x, w, bias, out=out[:t, 1:n + 1])
    check(y, x64, w64, group, bias)
    assert bool((out[t] == 7).all()) and bool((out[:, 0] == 7).all()) and bool((out[:, n + 1:] == 7).all())


@pytest.mark.parametrize("t,n", [(1, 80), (12, 80), (100, 80), (60, 4000), (100, 3000), (264, 1200)])
def test_every_code_and_column_is_its_own(t, n):
    """One-hot rows read single weights: code, scale and place of each."""
    from lastkv_b200 import ops

    k, group = 264, 32
    g = _gen(t, 3)
    codes, scales, w64 = make_weight(n, k, group, g)
    w = ops.w4_pack(codes, scales, group)
    cols = torch.arange(t, device="cuda") * 37 % k
    x = torch.zeros((t, k), dtype=torch.bfloat16, device="cuda")
    x[torch.arange(t, device="cuda"), cols] = 1.0
    want = w64[:, cols].T.bfloat16()
    torch.testing.assert_close(ops.w4_linear(x, w), want, rtol=0, atol=0)
    q = ops.Q8Rows((x * 1).to(torch.int8), torch.ones((t, -(-k // group)), device="cuda"), group)
    torch.testing.assert_close(ops.w4_linear(q, w), want, rtol=0, atol=0)


@pytest.mark.parametrize("t,n", [(2, 192), (40, 192), (130, 192), (60, 3000), (130, 2000), (300, 1000)])
def test_non_finite_rows_stay_their_own(t, n):
    from lastkv_b200 import ops

    g = _gen(t, 4, n)
    codes, scales, w64 = make_weight(n, 512, 128, g)
    w = ops.w4_pack(codes, scales, 128)
    x, x64 = make_x(t, 512, 128, False, g)
    x[0, 3] = float("nan")
    x[1, 200] = float("inf")
    y = ops.w4_linear(x, w)
    assert bool(torch.isnan(y[0]).all())
    c = w64[:, 200]
    assert bool((y[1][c > 0] == float("inf")).all()) and bool((y[1][c < 0] == float("-inf")).all())
    assert bool(torch.isnan(y[1][c == 0]).all())
    if t > 2:
        check(y[2:], x64[2:], w64, 128)
    rows = ops.quantize_q8(x)
    y = ops.w4_linear(rows, w)
    assert bool(torch.isnan(y[:2]).all()) and bool(torch.isfinite(y[2:]).all())


@pytest.mark.parametrize("scale", [1e-30, 1e33])
@pytest.mark.parametrize("t,n", [(4, 64), (300, 1000)])
def test_scales_far_from_one(scale, t, n):
    """int8 rows whose values reach the ends of bf16's range, times weights that bring them back."""
    from lastkv_b200 import ops

    g = _gen(t, 9)
    codes, scales, w64 = make_weight(n, 512, 128, g)
    unit = 1e-4 if scale > 1 else 1.0
    w = ops.w4_pack(codes, (scales.float() * unit).bfloat16())
    w64 = (w64 / scales.double().repeat_interleave(128, 1)) * (scales.float() * unit).bfloat16().double().repeat_interleave(128, 1)
    x, x64 = make_x(t, 512, 128, True, g)
    x = ops.Q8Rows(x.q, x.scale * scale, 128)
    x64 = x.q.double() * x.scale.double().repeat_interleave(128, 1)
    check(ops.w4_linear(x, w), x64, w64, 128)


@pytest.mark.parametrize("t", [1, 8, 50, 200])
@pytest.mark.parametrize("int8", [False, True])
def test_deterministic_graph_and_other_stream(t, int8):
    from lastkv_b200 import ops

    g = _gen(t, 5, int8)
    codes, scales, w64 = make_weight(1024, 4096, 128, g)
    w = ops.w4_pack(codes, scales)
    x, x64 = make_x(t, 4096, 128, int8, g)
    a = ops.w4_linear(x, w)
    out = torch.empty_like(a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.w4_linear(x, w, out=out)
    torch.cuda.current_stream().wait_stream(s)
    torch.testing.assert_close(out, a, rtol=0, atol=0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.w4_linear(x, w, out=out)
    (x.q if int8 else x)[:, :128].zero_()
    graph.replay()
    torch.testing.assert_close(out, ops.w4_linear(x, w), rtol=0, atol=0)
    assert not torch.equal(out, a)


def test_quantize_rounds_to_four_bits():
    from lastkv_b200 import ops

    g = _gen(11)
    w = torch.randn((70, 200), generator=g, device="cuda").bfloat16()
    w[3, :32] = 0
    q = ops.w4_quantize(w, 32)
    eye = torch.eye(200, device="cuda").bfloat16()
    back = ops.w4_linear(eye, q).T.double()
    top = torch.nn.functional.pad(w.double().abs(), (0, -200 % 32)).view(70, -1, 32).amax(-1)
    s = (top / 7).repeat_interleave(32, 1)[:, :200]
    # half a step, the scale's and the result's rounding to bf16 (7 steps of 2^-8 each)
    assert bool(((back - w.double()).abs() <= s * (0.5 + 14 * 2.0 ** -8) + 1e-30).all())
    assert not bool(back[3, :32].any())


def test_no_rows_and_refusals():
    from lastkv_b200 import ops
    from lastkv_b200.contract import RMarinBackendContractError

    g = _gen(12)
    codes, scales, _ = make_weight(64, 256, 128, g)
    w = ops.w4_pack(codes, scales)
    x = torch.zeros((4, 256), dtype=torch.bfloat16, device="cuda")
    assert ops.w4_linear(x[:0], w).shape == (0, 64)
    assert ops.w4_linear(x.view(2, 2, 256), w).shape == (2, 2, 64)
    for call in (lambda: ops.w4_linear(x[:, :128], w),
                 lambda: ops.w4_linear(x.float(), w),
                 lambda: ops.w4_linear(x.cpu(), w),
                 lambda: ops.w4_linear(torch.zeros((4, 264), dtype=torch.bfloat16, device="cuda")[:, 4:260], w),
                 lambda: ops.w4_linear(ops.quantize_q8(x, group=64), w),
                 lambda: ops.w4_linear(x, w, out=torch.empty((4, 65), dtype=torch.bfloat16, device="cuda")),
                 lambda: ops.w4_linear(x, w, out=torch.empty((4, 64), device="cuda")),
                 lambda: ops.w4_linear(x, w, bias=torch.zeros(63, dtype=torch.bfloat16, device="cuda")),
                 lambda: ops.w4_pack(codes, scales, 64),
                 lambda: ops.w4_pack(codes, scales.float()),
                 lambda: ops.w4_pack(codes[:, :6], scales[:, :1], 128),  # 12 columns
                 lambda: ops.w4_pack(codes, scales, 256),
                 lambda: ops.w4_quantize(x[:, :12]),
                 lambda: ops.w4_quantize(codes)):
        with pytest.raises(RMarinBackendContractError):
            call()


@pytest.mark.parametrize("t,n,k,group,int8", [
    (20, 10075, 9992, 128, False), (32, 28672, 4096, 128, False), (45, 1508, 8400, 64, False), (14, 18754, 11568, 32, True),
    (8, 28672, 4096, 128, True), (141, 24819, 1032, 128, True), (141, 24819, 1032, 32, True), (256, 6144, 4096, 32, True),
    (141, 24819, 1032, 64, False), (300, 6144, 4096, 128, False), (300, 28672, 4096, 128, True)])
def test_many_blocks_in_flight(t, n, k, group, int8):
    """Weights past the rings' depth, over and over: each call gives the first one's bits, and those are right."""
    from lastkv_b200 import ops

    g = _gen(t, n, k, group)
    codes, scales, w64 = make_weight(n, k, group, g)
    x, x64 = make_x(t, k, group, int8, g)
    w = ops.w4_pack(codes, scales, group)
    err = torch.zeros(4, dtype=torch.int32, device="cuda")
    first = ops.w4_linear(x, w, error_word=err)
    check(first, x64, w64, group)
    for _ in range(60):
        assert torch.equal(ops.w4_linear(x, w, error_word=err), first)
    assert err.tolist() == [0, 0, 0, 0]
