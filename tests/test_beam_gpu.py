"""Beam search's selection against sorting all totals in 64 bits."""

import pytest
import torch

from lastkv_b200 import ops

pytestmark = pytest.mark.gpu

INF = float("inf")


def _plain(logits, scores, n, finished=None, eos=-1):
    """(totals fp64, rows, tokens, finished), ties by beam and token; what is not a number counts as -inf."""
    B, K = scores.shape
    V = logits.shape[1]
    x = logits.cpu().double().view(B, K, V)
    c = scores.cpu().double()
    total = c[..., None] + torch.log_softmax(x, -1)
    lse = torch.logsumexp(x, -1)
    if finished is not None:
        done = finished.cpu()
        alone = torch.full((B, K, V), -INF, dtype=torch.float64)
        alone[..., eos] = c
        total = torch.where(done[..., None], alone, total)
        lse = torch.where(done, 0.0, lse)
    total = torch.where(c.isfinite()[..., None] & lse.isfinite()[..., None] & ~total.isnan(), total, -INF)
    best, at = total.view(B, K * V).sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    beam, token = at // V, at % V
    ended = token == eos
    if finished is not None:
        ended = ended | finished.cpu().gather(1, beam)
    return best, beam + torch.arange(B)[:, None] * K, token, ended


def _tolerance(best):
    """Of a total: a term of the sum has its argument's rounding (|x - max| log2 e half steps) and the exponential's
    2^-22; sums of up to 2^18 terms, in chunks of 32 to a thread, then pairwise, are below 64 half steps off; the
    total's own rounding and the score's."""
    return (64 + 32) * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -24 * (best.abs() + 64)


def _check(logits, scores, n=None, finished=None, eos=None, permuted=False):
    """``permuted``: the rows hold the same values in different orders, or the same values plus a constant.  Their
    sums of exponentials are then equal numbers (but for the rounding of the logits themselves, a half step of 2^-19 below
    64), and so are totals of different rows; which of them is larger is a matter of how the sums round (in 64 bits
    as well), so any candidate whose total is the rank's within the totals' tolerance is right."""
    n = scores.shape[1] if n is None else n
    r = ops.beam_select(logits, scores, select=n, finished=finished, eos_token=eos)
    best, rows, tokens, ended = _plain(logits, scores, n, finished, -1 if eos is None else eos)
    if permuted:
        total = scores.cpu().double().view(-1, 1) + torch.log_softmax(logits.cpu().double(), -1)
        chosen = total[r.rows.cpu(), r.tokens.cpu()]
        assert bool(((chosen - best).abs() <= 2 * _tolerance(best)).all())
        assert all(len(set(zip(a, b))) == n for a, b in zip(r.rows.tolist(), r.tokens.tolist()))
    else:
        assert torch.equal(r.rows.cpu(), rows) and torch.equal(r.tokens.cpu(), tokens)
    assert torch.equal(r.finished.cpu(), ended)
    assert r.scores.dtype == torch.float32
    got, fine = r.scores.cpu().double(), best.isfinite()
    assert torch.equal(got[~fine], best[~fine])
    assert bool(((got[fine] - best[fine]).abs() <= _tolerance(best[fine])).all())
    return r


def _logits(seed, rows, V, dtype=torch.float32, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, V), generator=g) * spread).to(dtype).cuda()


def _scores(seed, B, K):
    return -torch.rand((B, K), generator=torch.Generator().manual_seed(seed)).cuda() * 4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 1, 1), (1, 1, 33, 32), (2, 3, 7, 7), (3, 4, 100, 8), (1, 4, 8192, 4),
                                     (2, 2, 8193, 5), (1, 5, 50001, 10), (16, 8, 1000, 16), (1, 64, 3001, 32),
                                     (2, 4, 128256, 8), (1, 2, 300000, 32)])
def test_sizes(dtype, B, K, V, n):
    _check(_logits(V + n, B * K, V, dtype), _scores(V, B, K), n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_any_stride_and_alignment(dtype):
    for pad, off in ((1, 0), (5, 1), (8, 3), (3, 7)):
        wide = _logits(pad, 6, 20000 + pad + off, dtype)
        _check(wide[:, off: off + 20000], _scores(2, 2, 3), 6)
    row = _logits(3, 1, 9000, dtype)
    _check(row.expand(4, 9000), _scores(4, 1, 4), 4)  # one row of logits for all beams


def test_equal_values_go_by_beam_and_token():
    for V in (50, 9000, 40000):
        for n in (1, 4, 32):
            x = torch.zeros((4, V), device="cuda")
            _check(x, torch.zeros((1, 4), device="cuda"), n)
            _check(x.bfloat16(), torch.zeros((2, 2), device="cuda"), n)
    x = torch.randint(-2, 3, (6, 30000), generator=torch.Generator().manual_seed(1)).float().cuda()
    _check(x, torch.zeros((2, 3), device="cuda"), 6)
    x = torch.tensor([[0.0, -0.0] * 20000], device="cuda")  # -0 equals 0
    _check(x, torch.zeros((1, 1), device="cuda"), 16)


@pytest.mark.parametrize("n", [1, 8, 32])
def test_sorted_rows(n):
    """Every tile beats the ones before it, or none does."""
    up = torch.arange(40000, device="cuda").float() / 1000
    x = torch.stack((up, up.flip(0), up.roll(12345), -(up - 20).abs()))
    _check(x.contiguous(), torch.zeros((1, 4), device="cuda"), n, permuted=True)
    _check(x.bfloat16(), torch.zeros((2, 2), device="cuda"), n, permuted=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [2, 8, 32])
def test_large_values_in_few_threads(dtype, n):
    """A tile whose large values all lie with a few threads of each warp but one, in bands: more of them reach the
    raised bar than the list holds, and they are taken out one by one."""
    per = 16 // torch.tensor([], dtype=dtype).element_size()  # values of a thread's 16-byte piece
    at = torch.arange(8192)
    thread = at // per % 256
    lane, warp = thread % 32, thread // 32
    band = torch.where((lane < 31) & (warp < 7), 31 - lane, 0).float()
    fine = torch.rand(8192, generator=torch.Generator().manual_seed(n)) * 0.9
    x = torch.where(band > 0, band + fine, torch.full_like(fine, -50.0) + fine)
    rows = torch.stack((x, x.flip(0), x + 1)).to(dtype).cuda()
    _check(rows, torch.zeros((1, 3), device="cuda"), n, permuted=True)
    for i in range(3):
        _check(rows[i:i + 1], torch.zeros((1, 1), device="cuda"), n)


def test_masked_vocabularies():
    V = 30011
    x = _logits(5, 6, V)
    x[0] = -INF
    x[0, 12345] = 1.0
    x[1, 100:] = -INF
    x[2, ::2] = -INF
    x[3] = torch.finfo(torch.float32).min
    x[4] = -INF  # nothing left at all
    for n in (3, 6, 32):
        _check(x, _scores(6, 1, 6), n)
        _check(x, _scores(7, 2, 3), n)
    y = _logits(8, 2, 200).bfloat16()
    y[0] = torch.finfo(torch.bfloat16).min
    y[1, 3:] = torch.finfo(torch.bfloat16).min
    _check(y, _scores(9, 1, 2), 8)


def test_beams_that_are_out():
    """Scores of -inf (the beams of a first step), of -1e9, of NaN; rows with NaN or infinity."""
    x = _logits(10, 8, 5000)
    s = torch.full((2, 4), -INF, device="cuda")
    s[:, 0] = 0
    r = _check(x, s, 4)
    assert r.rows.tolist() == [[0] * 4, [4] * 4]
    s[:, 1:] = -1e9
    _check(x, s, 8)
    s[0, 0], s[1, 2] = float("nan"), INF
    _check(x, s, 8)
    x[1, 77], x[5, 4000], x[6, 0] = float("nan"), INF, -INF
    x[2] = float("nan")
    _check(x, _scores(11, 2, 4), 8)
    dead = torch.full((1, 3), -INF, device="cuda")
    r = _check(_logits(12, 3, 9000), dead, 5)
    assert r.tokens.tolist() == [[0, 1, 2, 3, 4]] and r.rows.tolist() == [[0] * 5]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_finished_beams(dtype):
    V, eos = 20003, 2
    x, s = _logits(13, 12, V, dtype), _scores(14, 3, 4)
    done = torch.tensor([[True, False, False, True], [False] * 4, [True] * 4], device="cuda")
    r = _check(x, s, 8, done, eos)
    assert bool(r.finished[2, :4].all())
    _check(x, s, 4, done, V - 1)
    x[4, eos] = 60.0  # a beam that ends now
    r = _check(x, s, 4, done, eos)
    assert bool(r.finished[r.tokens == eos].all())
    x[0] = float("nan")  # a finished beam's logits do not matter
    _check(x, s, 4, done, eos)


def test_captured_steps():
    """Buffers of a captured step, replayed with new logits; two captures, one after the other."""
    x, s = torch.zeros((8, 30000), device="cuda"), torch.zeros((2, 4), device="cuda")
    outs = [ops.BeamChoice.empty(2, 4) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.beam_select(x, s, out=outs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            ops.beam_select(x, s, out=o)
        graphs.append(g)
    for seed in range(3):
        x.copy_(_logits(seed, 8, 30000))
        s.copy_(_scores(seed, 2, 4))
        for g, o in zip(graphs, outs):
            g.replay()
            best, rows, tokens, _ = _plain(x, s, 4)
            assert torch.equal(o.rows.cpu(), rows) and torch.equal(o.tokens.cpu(), tokens)


@pytest.mark.parametrize("B,K", [(1, 1), (3, 7), (5, 32)])
def test_results_in_the_place_of_scores_and_finished(B, K):
    g = torch.Generator().manual_seed(B)
    logits = torch.randn((B * K, 3001), generator=g).cuda()
    scores, done = -torch.rand((B, K), generator=g).cuda() * 5, (torch.rand((B, K), generator=g) < 0.4).cuda()
    want = ops.beam_select(logits, scores, finished=done, eos_token=9)
    out = ops.BeamChoice.empty(B, K)._replace(scores=scores, finished=done)
    ops.beam_select(logits, scores, finished=done, eos_token=9, out=out)
    for a, b in zip(out, want):
        assert torch.equal(a, b)


def test_same_result_every_time():
    x, s = _logits(15, 32, 128256).bfloat16(), _scores(16, 4, 8)
    first = ops.beam_select(x, s, select=16)
    for _ in range(5):
        for a, b in zip(first, ops.beam_select(x, s, select=16)):
            assert torch.equal(a, b)


def test_refusals():
    from lastkv_b200.contract import RMarinBackendContractError as Refused

    x, s = _logits(17, 6, 40), _scores(18, 2, 3)
    for args, kw, word in (((x.half(), s), {}, "logits"), ((x[:5], s), {}, "logits"), ((x.t(), s), {}, "logits"),
                           ((x, s.double()), {}, "scores"), ((x, s.t()), {}, "scores"), ((x, s), dict(select=0), "select"),
                           ((x, s), dict(select=33), "select"), ((x[:, :4], s), dict(select=5), "select"),
                           ((x, s), dict(finished=s > -2), "eos_token"),
                           ((x, s), dict(finished=s > -2, eos_token=40), "eos_token"),
                           ((x, s), dict(finished=(s > -2).int(), eos_token=1), "finished"),
                           ((x, s), dict(out=ops.BeamChoice.empty(2, 4)), "out")):
        with pytest.raises(Refused, match=word):
            ops.beam_select(*args, **kw)
