"""Paged caches and the attention over them on the GPU."""

from __future__ import annotations

import math

import pytest
import torch

from _attention_reference import check
from _paged_checks import append_case, normal, paged_case, prompt_then_steps, table_for
from _paged_reference import attention

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


# -- single tokens and a few ---------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1, 5, 16, 24, 64])
@pytest.mark.parametrize("dim", [32, 64, 80, 128, 256])
def test_single_tokens(gpu, dtype, size, dim):
    paged_case(gpu, "cuda", dtype, [0, 1, 15, -1, 16, 31, 32, 33, 300], size=size, dim=dim)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (8, 1), (12, 4), (34, 2), (17, 1)])
def test_heads(gpu, dtype, heads, kv_heads):
    paged_case(gpu, "cuda", dtype, [77, 3], heads=heads, kv_heads=kv_heads, dim=64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [2, 3, 5, 8, 16])
def test_drafts(gpu, dtype, tokens):
    paged_case(gpu, "cuda", dtype, [0, 30, -1, 201], tokens=tokens, dim=64,
               lengths=[tokens, 1, tokens, tokens - 1])


@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (7, 4), (33, 40), (100, 3), (None, 2)])
@pytest.mark.parametrize("tokens", [1, 4, 70])
@pytest.mark.parametrize("size", [5, 16])
def test_window_and_sinks(gpu, window, sinks, tokens, size):
    paged_case(gpu, "cuda", torch.bfloat16, [0, 3, 31, 180, 64], tokens=tokens, window=window,
               sinks=sinks, size=size, dim=64)


@pytest.mark.parametrize("dtype", TYPES)
def test_long(gpu, dtype):
    paged_case(gpu, "cuda", dtype, [20_011], heads=8, kv_heads=2, dim=64, size=16)
    paged_case(gpu, "cuda", dtype, [9000, 3, -1, 700], heads=4, kv_heads=2, dim=128, size=24)


def test_many_sequences(gpu):
    gen = torch.Generator().manual_seed(8)
    starts = torch.randint(-1, 90, (700,), generator=gen).tolist()
    paged_case(gpu, "cuda", torch.bfloat16, starts, heads=4, kv_heads=2, dim=32, size=16)
    paged_case(gpu, "cuda", torch.float16, starts[:300], tokens=3, heads=8, kv_heads=2, dim=32, size=7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["plain", "packed", "odd"])
@pytest.mark.parametrize("dim", [64, 20, 100])
def test_layouts(gpu, dtype, layout, dim):
    paged_case(gpu, "cuda", dtype, [90, 4], tokens=3, lengths=[3, 1], layout=layout, heads=6,
               kv_heads=3, dim=dim, size=16, index=torch.int64, table_index=torch.int64)


def test_queries_at_odd_addresses(gpu):
    """Aligned caches, a query that is not."""
    gen = torch.Generator().manual_seed(4)
    total, table = table_for(gen, [41, 12], 16, 3)
    ck, cv = (normal(gen, torch.bfloat16, "cuda", total, 16, 2, 64) for _ in range(2))
    q = normal(gen, torch.bfloat16, "cuda", 2, 1, 4, 65)[..., 1:]
    starts = torch.tensor([40, 11], device="cuda")
    got = gpu.paged_attention(q, ck, cv, table.cuda(), starts=starts)
    check(got, attention(q, ck, cv, table, [40, 11]), "odd queries")


# -- chunks of prompts -----------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 80, 96, 128, 256])
@pytest.mark.parametrize("size", [16, 5, 64])
def test_chunks(gpu, dtype, dim, size):
    paged_case(gpu, "cuda", dtype, [0, 130, -1], tokens=75, lengths=[75, 61, 75], dim=dim, size=size)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (8, 8), (10, 2), (34, 2)])
def test_chunk_heads(gpu, heads, kv_heads):
    paged_case(gpu, "cuda", torch.float16, [70, 0], tokens=129, heads=heads, kv_heads=kv_heads, dim=64)


@pytest.mark.parametrize("dtype", TYPES)
def test_long_chunk(gpu, dtype):
    paged_case(gpu, "cuda", dtype, [4001], tokens=300, heads=2, kv_heads=1, dim=64, size=64)


@pytest.mark.parametrize("window,sinks", [(1, 0), (50, 4), (200, 0), (1000, 70)])
def test_chunk_window(gpu, window, sinks):
    paged_case(gpu, "cuda", torch.bfloat16, [500, 33, 0], tokens=200, window=window, sinks=sinks, dim=128,
               size=32)


# -- a prefix that the batch shares ------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 4])
@pytest.mark.parametrize("size,shared", [(16, 1), (16, 9), (5, 3), (24, 11), (64, 4)])
def test_shared_pages(gpu, dtype, tokens, size, shared):
    s = size * shared
    paged_case(gpu, "cuda", dtype, [s + 40, s + 3, -1, s, s + 100, max(s - 7, 0), 0] * 3, tokens=tokens,
               shared=shared, size=size, dim=64, heads=8, kv_heads=2)


@pytest.mark.parametrize("dim", [32, 80, 96, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (16, 2), (40, 2)])
def test_shared_heads(gpu, dim, heads, kv_heads):
    paged_case(gpu, "cuda", torch.bfloat16, [150, 131, 190, 400, 130, 129], shared=8, dim=dim, heads=heads,
               kv_heads=kv_heads)


@pytest.mark.parametrize("window,sinks", [(60, 0), (60, 20), (400, 4), (None, 3)])
@pytest.mark.parametrize("tokens", [1, 3])
def test_shared_window(gpu, window, sinks, tokens):
    paged_case(gpu, "cuda", torch.float16, [250, 131, 190, 400, 100, 129, 600], tokens=tokens, shared=8,
               window=window, sinks=sinks, dim=64, heads=8, kv_heads=2)


def test_shared_batch(gpu):
    gen = torch.Generator().manual_seed(3)
    starts = (2048 + torch.randint(0, 300, (70,), generator=gen)).tolist()
    starts[5] = -1
    paged_case(gpu, "cuda", torch.bfloat16, starts, shared=128, dim=128, heads=8, kv_heads=2)
    paged_case(gpu, "cuda", torch.bfloat16, starts[:20], shared=128, dim=64, heads=8, kv_heads=2, tokens=4,
               lengths=[4, 3, 2, 1, 0] * 4)


def test_shared_with_a_first_row_without_a_sequence(gpu):
    paged_case(gpu, "cuda", torch.bfloat16, [-1, 80, 90, 70], shared=4, dim=64, heads=4, kv_heads=2)


def test_all_pages_shared(gpu):
    paged_case(gpu, "cuda", torch.float32, [63, 40, 50, 60], shared=4, width=4, dim=64)


def behind(size, pages, batch=64, low=-9, high=90):
    """Starts of a batch behind a prefix that is long enough to be read once for all."""
    gen = torch.Generator().manual_seed(size + pages)
    starts = (pages * size + torch.randint(low, high, (batch,), generator=gen)).tolist()
    starts[0] = starts[17] = -1
    return starts


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size,pages,dim,tokens", [(16, 140, 128, 1), (24, 130, 96, 2), (5, 841, 64, 1),
                                                   (64, 65, 32, 4), (16, 200, 80, 1)])
def test_read_once(gpu, dtype, size, pages, dim, tokens):
    paged_case(gpu, "cuda", dtype, behind(size, pages), shared=pages, size=size, dim=dim, tokens=tokens,
               heads=4, kv_heads=2)


@pytest.mark.parametrize("heads,kv_heads", [(5, 5), (24, 1)])
def test_read_once_heads(gpu, heads, kv_heads):
    paged_case(gpu, "cuda", torch.bfloat16, behind(16, 260), shared=260, dim=64, heads=heads,
               kv_heads=kv_heads, layout="packed")


def test_read_once_with_what_is_not_there(gpu):
    starts = behind(16, 140)
    paged_case(gpu, "cuda", torch.float16, starts, shared=140, dim=128, heads=4, kv_heads=2, sinks=3,
               tokens=3, lengths=[3, 0, 1, 2] * 16, holes=[(b, 7) for b in range(64)] + [(5, 141)])
    # no sequence goes on behind the prefix, some end within it
    paged_case(gpu, "cuda", torch.float16, behind(16, 140, low=-900, high=-1), shared=140, dim=128,
               heads=4, kv_heads=2)


def test_read_once_values(gpu):
    """Infinite values that all see; and of two drafts' own one that the first does not."""
    def change(q, ck, cv, table):
        cv[table[1, 3], 2, :, 5] = float("inf")
        j = starts[1] + 1
        ck[table[1, j // 16], j % 16], cv[table[1, j // 16], j % 16] = float("nan"), float("-inf")

    starts = behind(16, 140, low=0)
    out, (value, tol) = paged_case(gpu, "cuda", torch.bfloat16, starts, shared=140, dim=128, heads=4,
                                   kv_heads=2, tokens=2, change=change)
    live = [b for b, s in enumerate(starts) if s >= 0]
    rest = [d for d in range(128) if d != 5]
    assert (out[live, 0, :, 5] == math.inf).all() and out[1, 1].isnan().all()
    live.remove(1)
    got, want = (t[live][..., rest] for t in (out, value))
    check(got, (want, tol[live][..., rest]), "values beside")
    check(out[1, :1][..., rest], (value[1, :1][..., rest], tol[1, :1][..., rest].nan_to_num(posinf=0)),
          "the first draft")


# -- what is not there ---------------------------------------------------------
@pytest.mark.parametrize("tokens", [1, 3, 80])
@pytest.mark.parametrize("shared", [0, 2])
def test_pages_that_are_not_there(gpu, tokens, shared):
    paged_case(gpu, "cuda", torch.float32, [130, 9, 60], tokens=tokens, dim=64, size=8, shared=shared,
               holes=[(0, 3), (0, 10), (1, 2), (2, 4)])


@pytest.mark.parametrize("tokens", [1, 3, 80])
def test_beyond_the_table(gpu, tokens):
    paged_case(gpu, "cuda", torch.float32, [30, 100, 7], tokens=tokens, width=2, size=8, dim=64)
    paged_case(gpu, "cuda", torch.float32, [2**62, 2**63 - 1, 2**40], tokens=tokens, width=2, size=8,
               dim=64, window=5, sinks=3, index=torch.int64, poison=False)
    paged_case(gpu, "cuda", torch.float32, [0, 0, 3], tokens=tokens, width=0, size=8, dim=64)


def test_nothing_to_attend(gpu):
    empty = torch.zeros(0, 4, 2, 8, device="cuda")
    pages = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    one = torch.ones(2, 1, 4, 8, device="cuda")
    assert torch.equal(gpu.paged_attention(one, empty, empty, pages), torch.zeros_like(one))
    assert gpu.paged_attention(one[:0], empty, empty, pages[:0]).shape == (0, 1, 4, 8)
    assert gpu.paged_attention(one[:, :0], empty, empty, pages).shape == (2, 0, 4, 8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,shared", [(4, 0), (4, 2), (70, 0)])
def test_a_token_that_earlier_ones_do_not_see(gpu, dtype, tokens, shared):
    """The last token's value is infinite, its key NaN: those before it do not
    see it."""
    where = {}

    def change(q, ck, cv, table):
        page, slot = table[0, (40 + tokens - 1) // 16], (40 + tokens - 1) % 16
        ck[page, slot], cv[page, slot] = float("nan"), float("inf")
        where["last"] = True

    out, (value, tol) = paged_case(gpu, "cuda", dtype, [40, 35], tokens=tokens, dim=64, shared=shared,
                                   change=change)
    assert where
    check(out[0:1, :-1], (value[0:1, :-1], tol[0:1, :-1].nan_to_num(posinf=0)), "before it")
    check(out[1:], (value[1:], tol[1:]), "the other sequence")
    assert out[0, -1].isnan().all()


@pytest.mark.parametrize("tokens,shared", [(1, 0), (1, 2), (70, 0)])
def test_infinite_values_that_are_seen(gpu, tokens, shared):
    def change(q, ck, cv, table):
        cv[table[0, 0], 3, :, 5] = float("inf")
        cv[table[0, 0], 3, :, 6] = float("-inf")

    out, _ = paged_case(gpu, "cuda", torch.bfloat16, [40, 35], tokens=tokens, dim=64, shared=shared,
                        change=change)
    n = 2 if shared else 1
    assert (out[:n, :, :, 5] == math.inf).all() and (out[:n, :, :, 6] == -math.inf).all()
    assert out[:, :, :, 7:].isfinite().all() and out[:, :, :, :5].isfinite().all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("tokens", [1, 70])
def test_scales(gpu, scale, tokens):
    paged_case(gpu, "cuda", torch.float32, [50, 7], tokens=tokens, dim=64, scale=scale, size=8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 70])
def test_large_scores(gpu, dtype, tokens):
    paged_case(gpu, "cuda", dtype, [90, 7], tokens=tokens, dim=64, spread=3.0)


# -- appending -----------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("size,layout", [(16, "plain"), (5, "packed"), (1, "odd"), (64, "packed")])
@pytest.mark.parametrize("dim,rotated", [(64, 64), (128, 32), (80, 48), (36, 30)])
def test_append(gpu, dtype, interleaved, size, layout, dim, rotated):
    append_case(gpu, "cuda", dtype, [0, 7, -1, 130], tokens=6, lengths=[6, 1, 3, 0], size=size,
                layout=layout, interleaved=interleaved, dim=dim, rotated=rotated)


def test_append_without_rotation_or_place(gpu):
    append_case(gpu, "cuda", torch.float32, [3, 9], tokens=4, rotate=False)
    append_case(gpu, "cuda", torch.bfloat16, [3, 9], tokens=4, with_q=False)
    append_case(gpu, "cuda", torch.float32, [3, 9], tokens=9, size=4, holes=[(0, 1), (1, 4)])
    append_case(gpu, "cuda", torch.float32, [3, 9], tokens=9, size=4, width=3)
    append_case(gpu, "cuda", torch.float32, [2**62, 1], tokens=2, size=4, width=3, index=torch.int64,
                with_q=False)


def test_append_shapes(gpu):
    append_case(gpu, "cuda", torch.bfloat16, list(range(0, 900, 9)), heads=32, kv_heads=8, dim=64)
    append_case(gpu, "cuda", torch.bfloat16, [100], tokens=777, heads=5, kv_heads=5, dim=64, size=24)
    append_case(gpu, "cuda", torch.float16, [100_000], width=6_300, dim=64)


# -- together ------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (9, 2)])
@pytest.mark.parametrize("chunk,size", [(8, 8), (40, 16)])
def test_prompt_then_steps(gpu, dtype, window, sinks, chunk, size):
    prompt_then_steps(gpu, "cuda", dtype, window=window, sinks=sinks, chunk=chunk, size=size, dim=64,
                      prompt=(70, 7, 41))


def serving(gpu, dtype=torch.bfloat16, batch=5, shared=2, size=16, heads=8, kv_heads=2, dim=64):
    gen = torch.Generator().manual_seed(6)
    starts = [shared * size + n for n in (3, 40, 0, 200, 17)] * (batch // 5 + 1)
    starts = starts[:batch]
    width = shared + 18
    total, table = table_for(gen, [width * size] * batch, size, width, shared=shared)
    state = {n: normal(gen, dtype, "cuda", batch, 1, h, dim)
             for n, h in (("q", heads), ("k", kv_heads), ("v", kv_heads))}
    state |= {n: normal(gen, dtype, "cuda", total, size, kv_heads, dim) for n in ("ck", "cv")}
    return state | {"pages": table.int().cuda(), "starts": torch.tensor(starts, device="cuda"),
                    "rotation": gpu.Rotary(dim)}


def one_step(gpu, s, shared):
    q = gpu.paged_cache_append(s["k"], s["v"], s["ck"], s["cv"], s["pages"], starts=s["starts"],
                               rotation=s["rotation"], q=s["q"])
    return gpu.paged_attention(q, s["ck"], s["cv"], s["pages"], starts=s["starts"], shared_pages=shared)


@pytest.mark.parametrize("shared", [0, 2, 140])
def test_captured_and_replayed(gpu, shared):
    """Two graphs of the same steps, replayed in turn with eager work between."""
    s = serving(gpu, batch=64, shared=140) if shared > 2 else serving(gpu)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        one_step(gpu, s, shared)
    torch.cuda.current_stream().wait_stream(stream)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(one_step(gpu, s, shared))
        graphs.append(graph)
    for turn in range(6):
        s["starts"].add_(1 + 7 * (turn % 2))
        s["k"].mul_(-1)
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        got = outs[turn % 2].clone()
        assert torch.equal(got, one_step(gpu, s, shared))
        torch.cuda.synchronize()


@pytest.mark.parametrize("shared", [2, 140])
def test_on_two_streams_at_once(gpu, shared):
    states = [serving(gpu, batch=64 if shared > 2 else 5, shared=shared) for _ in range(2)]
    states[1]["q"].mul_(-2)
    want = [one_step(gpu, s, shared) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [[], []]
    for _ in range(5):
        for stream, s, g in zip(streams, states, got):
            with torch.cuda.stream(stream):
                g.append(one_step(gpu, s, shared))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


@pytest.mark.parametrize("shared", [0, 2])
@pytest.mark.parametrize("tokens", [1, 4, 70])
def test_same_bits_each_time(gpu, tokens, shared):
    first, _ = paged_case(gpu, "cuda", torch.bfloat16, [3000, 40, 35, 600], tokens=tokens, dim=64, shared=shared)
    for _ in range(3):
        again, _ = paged_case(gpu, "cuda", torch.bfloat16, [3000, 40, 35, 600], tokens=tokens, dim=64,
                              shared=shared)
        assert torch.equal(first, again)


def test_offsets_past_32_bits(gpu):
    """A cache of more values than 32 bits count, pages at its end."""
    size, kv_heads, dim = 64, 8, 128
    total = 2**31 // (size * kv_heads * dim) + 40
    ck = torch.zeros(total, size, kv_heads, dim, dtype=torch.float16, device="cuda")
    cv = torch.zeros_like(ck)
    gen = torch.Generator().manual_seed(2)
    n = 300
    pages = torch.tensor([[total - 1, total - 30, 5, total - 7, total - 2]])
    for t in (ck, cv):
        t[pages[0].cuda()] = normal(gen, torch.float16, "cuda", 5, size, kv_heads, dim)
    for tokens in (1, 70):
        q = normal(gen, torch.float16, "cuda", 1, tokens, 16, dim)
        k, v = (normal(gen, torch.float16, "cuda", 1, tokens, kv_heads, dim) for _ in range(2))
        start = torch.tensor([n - tokens], device="cuda")
        gpu.paged_cache_append(k, v, ck, cv, pages.cuda(), starts=start)
        got = gpu.paged_attention(q, ck, cv, pages.cuda(), starts=start)
        held = [t[pages[0].cuda()] for t in (ck, cv)]
        assert torch.equal(held[0].flatten(0, 1)[n - tokens:n], k[0])
        check(got, attention(q, *held, torch.arange(5)[None], [n - tokens]), f"tokens {tokens}")


def test_host_operands_move_but_caches_do_not(gpu):
    s = serving(gpu)
    out = gpu.paged_attention(s["q"].cpu(), s["ck"], s["cv"], s["pages"].cpu(), starts=s["starts"].cpu())
    assert torch.equal(out, gpu.paged_attention(s["q"], s["ck"], s["cv"], s["pages"], starts=s["starts"]))
    with pytest.raises(ValueError, match="caches must be on"):
        gpu.paged_attention(s["q"], s["ck"].cpu(), s["cv"], s["pages"])
