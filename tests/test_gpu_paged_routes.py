"""Paged attention at sizes from which other kernels, cuts and joins are taken."""

from __future__ import annotations

import pytest
import torch

from _attention_reference import check
from _paged_checks import normal, paged_case
from _paged_reference import attention

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
TYPES = [torch.float32, torch.float16, BF16]


def padded(batch, top, seed):
    """Starts up to ``top``, some slots without a sequence."""
    gen = torch.Generator().manual_seed(seed)
    starts = torch.randint(0, top, (batch,), generator=gen)
    starts[::7] = -1
    return starts.tolist()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [96, 128])
def test_drafts_on_many_keys(gpu, dtype, dim):
    paged_case(gpu, "cuda", dtype, padded(32, 1500, 1), tokens=5, heads=16, kv_heads=4, dim=dim,
               lengths=[5, 0, 3, 1] * 8, width=130)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [500, 620])
def test_chunk_behind_many_keys(gpu, dtype, tokens):
    """Units of like length, and more rows than are joined a workgroup each."""
    paged_case(gpu, "cuda", dtype, [5000], tokens=tokens, heads=8, kv_heads=2, dim=64)


def test_chunks_of_a_padded_batch(gpu):
    paged_case(gpu, "cuda", BF16, padded(40, 700, 2), tokens=90, heads=8, kv_heads=2, dim=64,
               lengths=[90, 3, 0, 41] * 10, width=50, window=300, sinks=5)


@pytest.mark.parametrize("dtype,dim,tokens", [(BF16, 64, 64), (torch.float16, 128, 50), (BF16, 256, 33),
                                              (torch.float32, 64, 40)])
@pytest.mark.parametrize("batch", [3, 150])
def test_short_prompts(gpu, dtype, dim, tokens, batch):
    """A workgroup a tile, all of its keys."""
    lengths = [tokens, 1, 0, tokens - 7, 20] * (batch // 5) + [tokens] * (batch % 5)
    paged_case(gpu, "cuda", dtype, padded(batch, 30, 3), tokens=tokens, heads=8, kv_heads=2, dim=dim,
               lengths=lengths, width=100 // 16 + 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,tokens", [(2, 1), (40, 2), (300, 1)])
def test_few_keys(gpu, dtype, dim, batch, tokens):
    """A workgroup a sequence and kv head, of eight waves or of four."""
    paged_case(gpu, "cuda", dtype, padded(batch, 250, 4), tokens=tokens, heads=12, kv_heads=3, dim=dim,
               width=16)


def test_wide_float32_chunk(gpu):
    paged_case(gpu, "cuda", torch.float32, [700, 90], tokens=70, heads=6, kv_heads=2, dim=256,
               lengths=[70, 33])


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_a_late_key_of_a_long_chunk(gpu, dtype):
    """What only the last queries see is theirs alone, also where their parts are joined."""
    at = 5000 + 400

    def change(q, ck, cv, table):
        ck[table[0, at // 16], at % 16] = float("nan")
        cv[table[0, at // 16], at % 16] = float("inf")

    out, (value, tol) = paged_case(gpu, "cuda", dtype, [5000], tokens=620, heads=8, kv_heads=2, dim=64,
                                   change=change)
    check(out[:, :400], (value[:, :400], tol[:, :400]), "queries before")
    assert out[:, 400:].isnan().all()


@pytest.mark.parametrize("tokens", [1, 3, 80])
def test_a_page_many_times(gpu, tokens):
    """Within a row of the table and in all of them; nothing is said to be shared."""
    gen = torch.Generator().manual_seed(6)
    ck, cv = (normal(gen, BF16, "cuda", 5, 16, 2, 64) for _ in range(2))
    q = normal(gen, BF16, "cuda", 6, tokens, 4, 64)
    table = torch.randint(0, 5, (6, 40), generator=gen)
    starts = [0, 500, 77, 31, 555, 12]
    got = gpu.paged_attention(q, ck, cv, table.cuda(), starts=torch.tensor(starts).cuda())
    check(got, attention(q, ck, cv, table, starts), f"tokens {tokens}")


def test_tables_of_one_row_for_all(gpu):
    """A table, starts of one value and queries that are expanded."""
    gen = torch.Generator().manual_seed(7)
    ck, cv = (normal(gen, BF16, "cuda", 9, 16, 2, 64) for _ in range(2))
    q = normal(gen, BF16, "cuda", 1, 1, 4, 64).expand(70, -1, -1, -1)
    table = torch.randperm(9, generator=gen)[None].expand(70, -1)
    starts = torch.full((70,), 130, device="cuda")
    for shared in (0, 8, 9):
        got = gpu.paged_attention(q, ck, cv, table[:1].cuda().expand(70, -1), starts=starts,
                                  shared_pages=shared)
        check(got, attention(q, ck, cv, table, [130] * 70), f"shared {shared}")


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 128), (BF16, 128), (BF16, 200), (BF16, 256),
                                       (torch.float32, 120), (torch.float32, 128)])
@pytest.mark.parametrize("tokens,window", [(1, None), (3, None), (1, 2**41)])
def test_tables_of_more_than_the_cache_holds(gpu, dtype, dim, tokens, window):
    """Wide tables of which little is filled: keys that are read past the caches."""
    paged_case(gpu, "cuda", dtype, [0, 40, -1, 700, 2500, 33], tokens=tokens, heads=8, kv_heads=2, dim=dim,
               width=6000, window=window, lengths=[tokens, 1, 1, tokens, tokens, 0])
