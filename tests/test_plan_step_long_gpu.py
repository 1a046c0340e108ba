"""The device step plan at the end of the longest context that int32 lengths allow."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("computed,new", [(2 ** 31 - 18, 1), (2 ** 31 - 2, 1), (2 ** 31 - 21, 20), (2 ** 31 - 1024, 1)])
def test_last_pages_of_the_longest_context(computed, new):
    from lastkv_b200 import ops

    most, chunk = 2 ** 31 - 1, 1024
    pages = 2 ** 27
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    base = torch.tensor([7], dtype=torch.int32, device="cuda")
    plan = ops.StepPlan(1, 20, table, base, chunk_size=chunk, max_sequence_tokens=most, scratch_src_page=0,
                        scratch_ring_page=128, width=pages)
    args = [torch.tensor([v], dtype=torch.int32, device="cuda") for v in (computed, new, 0)]
    plan.run(*args)
    plan.check_errors()
    last = computed + new - 1
    first = last // chunk * chunk - chunk  # the previous chunk's start: from here on pages lie in the ring
    ns, used = first // 16, last // 16 + 1
    got = plan.block_tables[0, 0]
    assert torch.equal(got[ns - 64:ns], table[0, ns - 64:ns])
    want = [7 + (ns % 128 + j) % 128 for j in range(used - ns)]
    assert got[ns:used].tolist() == want
    assert bool((got[used:] == 7).all())
    assert int(plan.seq_k[0]) == last + 1 and plan.positions[:new].tolist() == list(range(computed, last + 1))
    assert plan.commit_count.tolist() == [1 if computed % chunk == 0 else 0]
    if computed % chunk == 0:
        assert plan.commit_raw[0].tolist() == list(range((computed - chunk) // 16, computed // 16))
