"""Rows of a device step plan that break its rules: they run on the scratch pages alone and commit nothing."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def make_pool(slots, max_tokens, chunk, layers):
    from lastkv_b200.vllm_backend import SharedKVPool

    pages = -(-max_tokens // 16)
    return SharedKVPool(num_layers=layers, num_slots=slots, max_sequence_tokens=max_tokens, chunk_size=chunk,
                        num_kv_heads=1, head_dim=64, page_order=np.random.default_rng(3).permutation(slots * pages))


def make_plan(pool, batch, tokens, **kw):
    from lastkv_b200 import ops

    return ops.StepPlan(batch, tokens, torch.from_numpy(pool.src_table).cuda(), pool.ring_base_dev,
                        chunk_size=pool.chunk_size, max_sequence_tokens=pool.max_sequence_tokens,
                        scratch_src_page=pool.scratch_src_page, scratch_ring_page=pool.scratch_ring_page, **kw)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("rows,most", [(4, 5), (4, 3), (700, 900)])
def test_rows_past_the_buffers_commit_nothing(rows, most):
    """Every row starts at a chunk's start; those that do not fit come again, so their commits must not run now."""
    chunk, pool = 32, make_pool(rows, 200, 32, 2)
    plan = make_plan(pool, rows, most)
    computed, new, slots = [chunk * (1 + i % 5) for i in range(rows)], [2] * rows, list(range(rows))
    plan.run(i32(computed), i32(new), i32(slots))
    fits = most // 2
    assert plan.error_word.tolist()[0] == 4
    assert plan.commit_count.tolist() == [fits]
    ring = 2 * chunk // 16
    for i in range(fits):
        page = (computed[i] - chunk) // 16
        assert plan.commit_raw[i].tolist() == pool.src_table[slots[i], page:page + 2].tolist()
        assert plan.commit_ring[i].tolist() == [pool.ring_base(0) + slots[i] * ring + page % ring + j for j in (0, 1)]
    assert not bool(plan.commit_raw[fits:].any()) and not bool(plan.commit_ring[fits:].any())
    if fits < rows:  # the same rows in a step of their own: each commit is there, once
        rest = make_plan(pool, rows - fits, 2 * (rows - fits))
        rest.run(i32(computed[fits:]), i32(new[fits:]), i32(slots[fits:]))
        rest.check_errors()
        assert rest.commit_count.tolist() == [rows - fits]


@pytest.mark.parametrize("computed,new", [([0, 64], [9, 1]), ([3, 64], [2 ** 31 - 1, 1]), ([64, 3], [9, 1]), ([64], [9])])
def test_a_row_longer_than_the_buffers(computed, new):
    """The first row alone has more tokens than the buffers: it is reported, and so are the rows behind it."""
    pool = make_pool(2, 200, 32, 2)
    plan = make_plan(pool, len(new), 8)
    plan.run(i32(computed), i32(new), i32(list(range(len(new)))))
    assert plan.error_word.tolist()[0] == 4
    assert plan.commit_count.tolist() == [0]
    assert plan.cu_q.tolist() == [0, 8, 8][:len(new) + 1]
    assert plan.positions.tolist() == [0] * 8
    assert plan.ring_slots.tolist() == [pool.scratch_ring_page * 16] * 8
    assert plan.src_slots.tolist() == [pool.scratch_src_page * 16] * 8
    assert plan.seq_k.tolist() == [8, 1][:len(new)]


@pytest.mark.parametrize("new", [1, 15, 16, 17, 40, 130])
@pytest.mark.parametrize("why", ["slot", "boundary", "over"])
def test_bad_rows_read_no_sessions_pages(new, why):
    """Every page that the row's length reaches is the layer's scratch page, also past its first 16 tokens."""
    pool = make_pool(3, 300, 64, 3)
    plan = make_plan(pool, 3, 132 if why != "over" else new + 1)
    row = {"slot": (0, 3), "boundary": (63, 1), "over": (0, 1)}[why]
    n = new if why != "boundary" else max(new, 2)
    plan.run(i32([5, row[0], 7]), i32([1 if why != "over" else 2, n, 1]), i32([0, row[1], 2]))
    assert plan.error_word.tolist()[0] == 4
    tokens = n if why != "over" else n - 1
    assert int(plan.seq_k[1]) == max(1, tokens)
    pages = (max(1, tokens) + 15) // 16
    for layer in range(3):
        base = int(pool.ring_base(layer))
        assert plan.block_tables[layer, 1, :pages].tolist()[: plan.width] == \
            [base + pool.scratch_ring_page] * min(pages, plan.width)


def test_bad_rows_leave_the_sessions_alone():
    """Appending and attending as planned: the bad row's span writes and reads the scratch page alone, so its
    output does not depend on what the sessions hold, and theirs stays."""
    from lastkv_b200 import ops

    pool = make_pool(2, 300, 64, 1)
    plan = make_plan(pool, 2, 41)
    plan.run(i32([5, 0]), i32([1, 40]), i32([0, 9]))
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn((41, 1, 64), generator=g, device="cuda").bfloat16()
    outs = []
    for fill in (1.0, 50.0):
        pool.pool_k.fill_(fill)
        pool.pool_v.fill_(fill)
        page = int(pool.ring_base(0)) + pool.scratch_ring_page
        pool.pool_k[page] = 0.5
        pool.pool_v[page] = 0.25
        outs.append(ops.prefill_paged(q, pool.pool_k, pool.pool_v, plan.block_tables[0], plan.seq_k, plan.cu_q, 40,
                                      max_pages=plan.width))
    assert torch.equal(outs[0][1:], outs[1][1:])
    assert not torch.equal(outs[0][0], outs[1][0])
