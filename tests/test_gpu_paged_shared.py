"""Pages that a batch shares, read once for all: what each query sees of them."""

from __future__ import annotations

import pytest
import torch

from _attention_reference import check
from _paged_checks import normal, paged_case, table_for

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def past_the_table(capacity):
    """Starts of a batch some of which have outgrown a table of so many places, one by so much
    that it sees nothing of it."""
    starts = [capacity - 90 + 3 * b for b in range(64)]
    starts[3], starts[4], starts[5] = -1, 2 * capacity + 40, 2 * capacity - 30
    return starts


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,sinks,beyond", [(1, 0, 0), (1, 3, 0), (3, 0, 0), (3, 40, 0), (1, 0, 50)])
@pytest.mark.parametrize("shared", [0, 140, 146])
def test_a_window_of_the_table(gpu, dtype, tokens, sinks, beyond, shared):
    """Windows as wide as the table hide keys of it from queries that stand behind it."""
    capacity = 146 * 16
    paged_case(gpu, "cuda", dtype, past_the_table(capacity), tokens=tokens, window=capacity + beyond,
               sinks=sinks, shared=shared, width=146, dim=64, heads=4, kv_heads=2)



@pytest.mark.parametrize("missing", [-1, 10**6, 5])
@pytest.mark.parametrize("empty,batch,ended", [(1, 64, False), (63, 64, True), (64, 130, False), (100, 130, True),
                                               (64, 64, False)])
def test_first_slots_without_a_sequence(gpu, missing, empty, batch, ended):
    """Slots that have emptied, or have no query here, name no pages, or other ones."""
    starts = [2240 + 5 * b % 77 for b in range(batch)]
    lengths = [1] * batch
    for b in range(empty):
        if ended and b % 2 == 0:
            lengths[b] = 0
        else:
            starts[b] = -1

    def change(q, ck, cv, table):
        table[:empty] = missing

    out, want = paged_case(gpu, "cuda", torch.bfloat16, starts, lengths=lengths, shared=140, dim=64, heads=4, kv_heads=2,
                           change=change)
    assert (out[:empty] == 0).all() and (empty == batch or out[empty:].abs().max() > 0)
    check(out, want, f"{empty} of {batch}")


def test_slots_that_empty_between_replays(gpu):
    """A captured call finds the pages where they are when it is replayed."""
    gen = torch.Generator().manual_seed(4)
    total, table = table_for(gen, [2300] * 64, 16, 144, shared=140)
    ck, cv = (normal(gen, torch.bfloat16, "cuda", total, 16, 2, 64) for _ in range(2))
    q = normal(gen, torch.bfloat16, "cuda", 64, 1, 4, 64)
    pages = table.int().cuda()
    starts = (2240 + torch.arange(64) % 50).cuda()

    def attend():
        return gpu.paged_attention(q, ck, cv, pages, starts=starts, shared_pages=140)

    attend()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend()
    graph.replay()
    full = out.clone()
    for empty in (1, 2, 40):
        starts[:empty] = -1
        pages[:empty] = -1
        graph.replay()
        torch.cuda.synchronize()
        assert (out[:empty] == 0).all() and torch.equal(out, attend())
        # (the others' parts are the same; what is joined with them is cut another way)
        assert (out[empty:].float() - full[empty:].float()).abs().max() <= 2.0**-7 * full.abs().max()
