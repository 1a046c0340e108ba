"""The device step plan (lkv_plan_step) against the host plan of the same pool, element for element."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _pool(slots, max_tokens, chunk, layers, seed=0):
    from lastkv_b200.vllm_backend import SharedKVPool

    pages = -(-max_tokens // 16)
    return SharedKVPool(num_layers=layers, num_slots=slots, max_sequence_tokens=max_tokens, chunk_size=chunk,
                        num_kv_heads=1, head_dim=64, page_order=np.random.default_rng(seed).permutation(slots * pages))


def _device_plan(pool, batch, tokens, **kw):
    from lastkv_b200 import ops

    table = torch.from_numpy(pool.src_table).cuda()
    return ops.StepPlan(batch, tokens, table, pool.ring_base_dev, chunk_size=pool.chunk_size,
                        max_sequence_tokens=pool.max_sequence_tokens, scratch_src_page=pool.scratch_src_page,
                        scratch_ring_page=pool.scratch_ring_page, **kw)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _check(pool, plan, spans, padded):
    from lastkv_b200.vllm_backend import SharedKVFastPath

    batch = len(spans) + padded
    fast = SharedKVFastPath(pool, max_batch=batch, max_tokens=max(batch, sum(s.num_query_tokens for s in spans)),
                            num_q_heads=1)
    for s in spans:  # as a session that has run up to here: the chunk before its span's is committed
        done = s.num_computed_tokens // pool.chunk_size * pool.chunk_size
        pool.committed[s.slot] = done - pool.chunk_size if s.num_computed_tokens == done and done else done
    want = fast.plan_rows(spans, batch if padded else None)
    plan.run(_i32([s.num_computed_tokens for s in spans] + [77] * padded),
             _i32([s.num_query_tokens for s in spans] + [5] * padded), _i32([s.slot for s in spans] + [-1] * padded))
    T, B = want["tokens"], want["batch"]
    assert plan.error_word.tolist() == [0, 0, 0, 0]
    np.testing.assert_array_equal(plan.cu_q.cpu().numpy(), want["cu"])
    np.testing.assert_array_equal(plan.seq_k.cpu().numpy(), want["seqk"])
    np.testing.assert_array_equal(plan.positions[:T].cpu().numpy(), want["pos"])
    np.testing.assert_array_equal(plan.ring_slots[:T].cpu().numpy(), want["ring"])
    np.testing.assert_array_equal(plan.src_slots[:T].cpu().numpy(), want["src"])
    assert not bool(plan.positions[T:].any())
    assert bool((plan.ring_slots[T:] == pool.scratch_ring_page * 16).all())
    assert bool((plan.src_slots[T:] == pool.scratch_src_page * 16).all())
    j = np.arange(fast.W)[None, :]
    base = pool.ring_base_host[:, None, None]
    tables = np.where(j[None] < want["nsrc"][None, :, None], want["bt"][None], want["bt"][None] + base)
    np.testing.assert_array_equal(plan.block_tables.cpu().numpy(), tables)
    k = len(want["commits"])
    assert plan.commit_count.tolist() == [k]
    if k:
        raw, ring = fast._commit_pages(want["commits"])
        np.testing.assert_array_equal(plan.commit_raw[:k].cpu().numpy(), raw)
        np.testing.assert_array_equal(plan.commit_ring[:k].cpu().numpy(), ring)
    assert not bool(plan.commit_raw[k:].any()) and not bool(plan.commit_ring[k:].any())


@pytest.mark.parametrize("chunk,max_tokens,layers", [(16, 100, 1), (32, 1000, 3), (128, 5000, 2), (1024, 9000, 4)])
@pytest.mark.parametrize("padded", [0, 2])
def test_decode_steps(chunk, max_tokens, layers, padded):
    from lastkv_b200.vllm_backend import Span

    pool = _pool(7, max_tokens, chunk, layers)
    plan = _device_plan(pool, 5 + padded, 5 + padded)
    edges = [0, 1, chunk - 1, chunk, chunk + 1, 2 * chunk - 1, 2 * chunk, 3 * chunk, max_tokens - 1]
    for i in range(len(edges)):
        pos = [min(e, max_tokens - 1) for e in (edges[i:] + edges[:i])[:5]]
        _check(pool, plan, [Span((3 * b + i) % 7, p, 1) for b, p in enumerate(pos)], padded)


@pytest.mark.parametrize("seed", range(6))
def test_spans(seed):
    from lastkv_b200.vllm_backend import Span

    rng = np.random.default_rng(seed)
    chunk, max_tokens = [(64, 2000), (256, 3000), (512, 700)][seed % 3]
    rows = [1, 3, 40, 300, 2, 17][seed]
    pool = _pool(rows, max_tokens, chunk, 2, seed)
    spans = []
    for slot in rng.permutation(rows):
        p0 = int(rng.integers(0, max_tokens))
        if rng.random() < 0.4:
            p0 = p0 // chunk * chunk
        room = min(chunk - p0 % chunk, max_tokens - p0)
        spans.append(Span(int(slot), p0, int(rng.integers(1, min(room, 40) + 1)) if rng.random() < 0.8 else min(room, 40)))
    total = sum(s.num_query_tokens for s in spans)
    # padding rows belong to decode steps only, so the step is compared without them
    _check(pool, _device_plan(pool, rows, total + 13 * (seed % 2)), spans, 0)


def test_bad_rows_run_on_scratch_and_are_reported():
    from lastkv_b200.contract import RMarinBackendContractError

    pool = _pool(4, 200, 32, 2)
    cases = [([5, 30, 7], [1, 4, 1], [0, 1, 2]),       # a span over a chunk boundary
             ([5, 200, 7], [1, 1, 1], [0, 1, 2]),      # past the capacity
             ([5, 2 ** 31 - 1, 7], [1, 1, 1], [0, 1, 2]),
             ([5, -3, 7], [1, 1, 1], [0, 1, 2]),
             ([5, 6, 7], [1, 1, 1], [0, 4, 2]),        # no such slot
             ([5, 6, 7], [1, 0, 1], [0, 1, 2]),        # no new token
             ([5, 6, 7], [1, -9, 1], [0, 1, 2])]
    for computed, new, slots in cases:
        plan = _device_plan(pool, 3, 8)
        plan.run(_i32(computed), _i32(new), _i32(slots))
        assert plan.error_word.tolist()[0] == 4 and plan.error_word.tolist()[3] == 1
        with pytest.raises(RMarinBackendContractError):
            plan.check_errors()
        n = max(0, new[1])
        assert plan.cu_q.tolist() == [0, 1, 1 + n, 2 + n]
        assert plan.ring_slots[1:1 + n].tolist() == [pool.scratch_ring_page * 16] * n
        assert plan.positions[0] == 5 and plan.positions[1 + n] == 7
        assert int(plan.block_tables[1, 1, 0]) == pool.ring_base(1) + pool.scratch_ring_page
        assert int(plan.seq_k[1]) == max(1, n) and int(plan.seq_k[2]) == 8
    plan = _device_plan(pool, 3, 4)  # more tokens than the buffers hold: the last row does not fit
    plan.run(_i32([0, 0, 0]), _i32([2, 2, 2]), _i32([0, 1, 2]))
    assert plan.cu_q.tolist() == [0, 2, 4, 4] and plan.error_word.tolist()[3] == 2


def test_graph_replay_follows_the_lengths():
    pool = _pool(3, 300, 32, 2)
    plan = _device_plan(pool, 3, 3)
    computed, new, slots = _i32([0, 31, 290]), _i32([1, 1, 1]), _i32([2, 0, 1])
    plan.run(computed, new, slots)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.run(computed, new, slots)
        computed.add_(1)
    for step in range(9):
        g.replay()
        assert plan.positions.tolist() == [step, 31 + step, 290 + step]
        assert plan.commit_count.tolist() == [1 if step == 1 else 0]
    assert computed.tolist() == [9, 40, 299]


def test_refusals():
    from lastkv_b200 import ops
    from lastkv_b200.contract import RMarinBackendContractError

    pool = _pool(2, 100, 32, 2)
    table = torch.from_numpy(pool.src_table).cuda()
    kw = dict(chunk_size=32, max_sequence_tokens=100, scratch_src_page=1, scratch_ring_page=1)
    for call in (lambda: ops.StepPlan(0, 1, table, pool.ring_base_dev, **kw),
                 lambda: ops.StepPlan(1, 0, table, pool.ring_base_dev, **kw),
                 lambda: ops.StepPlan(1, 1, table.cpu(), pool.ring_base_dev, **kw),
                 lambda: ops.StepPlan(1, 1, table.long(), pool.ring_base_dev, **kw),
                 lambda: ops.StepPlan(1, 1, table[:, :3], pool.ring_base_dev, **kw),
                 lambda: ops.StepPlan(1, 1, table, pool.ring_base_dev, width=6, **kw),
                 lambda: ops.StepPlan(1, 1, table, pool.ring_base_dev, **{**kw, "chunk_size": 24}),
                 lambda: ops.StepPlan(2, 2, table, pool.ring_base_dev, **kw).run(_i32([1]), _i32([1]), _i32([0])),
                 lambda: ops.StepPlan(1, 1, table, pool.ring_base_dev, **kw).run(_i32([1]).long(), _i32([1]), _i32([0]))):
        with pytest.raises(RMarinBackendContractError):
            call()
