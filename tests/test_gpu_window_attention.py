"""Window attention's kernels against the definition in 64 bits, at the sizes,
layouts and masks where they could go wrong."""

from __future__ import annotations

import pytest
import torch

from _attention_checks import forward_and_gradients, operands, prompt_then_steps, step
from _attention_reference import check, reference

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAN = float("nan")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lq,lk,window,sinks", [
    (1, 1, 1, 0), (5, 5, 1, 2), (63, 63, 9, 0), (64, 64, 64, 4), (65, 65, 400, 0),
    (129, 129, 64, 4), (200, 200, 33, 70), (31, 300, 64, 5), (1, 257, 40, 3), (300, 31, 7, 2),
    (150, 150, 3, 500), (260, 260, 128, 1)])
def test_outputs_and_gradients(gpu, dtype, lq, lk, window, sinks):
    q, k, v, g = operands(lq + lk, 2, lq, lk, 4, 2, 64, dtype, "cuda")
    forward_and_gradients(gpu, q, k, v, g, f"{lq} {lk} {window} {sinks}", window=window,
                          sinks=sinks)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [1, 7, 8, 32, 40, 72, 80, 96, 120, 128, 136, 256])
def test_head_dimensions(gpu, dtype, dim):
    q, k, v, g = operands(dim, 1, 140, 140, 3, 1, dim, dtype, "cuda")
    forward_and_gradients(gpu, q, k, v, g, f"dim {dim}", window=50, sinks=4)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 1), (6, 3), (5, 5), (16, 2), (40, 2)])
def test_shared_heads(gpu, heads, kv_heads):
    q, k, v, g = operands(heads, 2, 97, 97, heads, kv_heads, 64, BF16, "cuda")
    forward_and_gradients(gpu, q, k, v, g, f"{heads}/{kv_heads}", window=30, sinks=2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_lengths_with_nan_in_the_padding(gpu, dtype, index):
    q, k, v, g = operands(3, 5, 150, 150, 4, 2, 64, dtype, "cuda")
    lengths = torch.tensor([150, 65, 0, 1, 64], dtype=index, device="cuda")
    for b, n in enumerate(lengths.tolist()):
        for t in (q, k, v, g):
            t[b, n:] = NAN
    got = forward_and_gradients(gpu, q, k, v, g, "padded", window=40, sinks=3, lengths=lengths)
    assert got["out"][2].abs().max() == 0 and got["dk"][4, 64:].abs().max() == 0


def test_lengths_of_a_chunk(gpu):
    """Chunk queries beyond a sequence's end see nothing."""
    q, k, v, g = operands(4, 3, 70, 210, 4, 2, 32, F16, "cuda")
    lengths = torch.tensor([140, 141, 205], dtype=torch.int32, device="cuda")
    got = forward_and_gradients(gpu, q, k, v, g, "chunk", window=33, sinks=5, lengths=lengths)
    assert got["out"][0].abs().max() == 0 and got["dv"][0].abs().max() == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_layouts(gpu, dtype):
    gen = torch.Generator().manual_seed(5)

    def normal(*shape):
        return torch.randn(shape, generator=gen).to(dtype).cuda()

    pattern = {"window": 45, "sinks": 2}
    q, k, v = normal(2, 133, 8, 64).split([4, 2, 2], dim=2)  # views of one projection
    forward_and_gradients(gpu, q, k, v, normal(2, 133, 4, 64), "packed", **pattern)
    q, k, v, g = (normal(2, n, 133, 64).transpose(1, 2) for n in (4, 2, 2, 4))  # head-major
    forward_and_gradients(gpu, q, k, v, g, "head-major", **pattern)
    q, k, v, g = (normal(133, 2, n, 64).transpose(0, 1) for n in (4, 2, 2, 4))  # token-major
    forward_and_gradients(gpu, q, k, v, g, "token-major", **pattern)
    q, k, v, g = (normal(2, 133, n, 67)[..., 1:65] for n in (4, 2, 2, 4))  # unaligned rows
    forward_and_gradients(gpu, q, k, v, g, "unaligned", **pattern)
    q, k, v, g = (normal(2, 133, n, 64)[..., ::2] for n in (4, 2, 2, 4))  # values apart
    forward_and_gradients(gpu, q, k, v, g, "apart", **pattern)
    k = normal(1, 133, 2, 64).expand(2, -1, -1, -1)  # one sequence of keys for the batch
    q, v, g = normal(2, 133, 4, 64), normal(2, 133, 1, 64).expand(-1, -1, 2, -1), normal(2, 133, 4, 64)
    forward_and_gradients(gpu, q, k, v, g.expand(2, 133, 4, 64), "broadcast", **pattern)


def test_broadcast_upstream(gpu):
    """The gradient of a sum: one value, expanded with stride zero."""
    q, k, v, _ = operands(6, 2, 90, 90, 4, 2, 64, BF16, "cuda")
    forward_and_gradients(gpu, q, k, v, torch.ones((), dtype=BF16, device="cuda").expand(q.shape),
                          "sum", window=20, sinks=1)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_wide_scores(gpu, dtype):
    """Scores of both signs in the hundreds: the running maximum moves, and
    probabilities vanish."""
    q, k, v, g = operands(7, 1, 200, 200, 2, 1, 64, dtype, "cuda", spread=4.0)
    forward_and_gradients(gpu, q, k, v, g * 0.25, "wide", window=70, sinks=4)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [NAN, float("inf")])
def test_tokens_out_of_sight(gpu, dtype, bad):
    """A token that is not finite reaches the queries that see it alone."""
    q, k, v, _ = operands(8, 1, 180, 180, 2, 2, 64, dtype, "cuda")
    pattern = {"window": 20, "sinks": 2}
    want = reference(q, k, v, **pattern)["out"]
    for at in (0, 1, 5, 70, 100, 179):
        for t in range(2):
            kk, vv = k.clone(), v.clone()
            (kk, vv)[t][0, at, 1] = bad
            out = gpu.window_attention(q, kk, vv, **pattern).cpu()
            p = torch.arange(180)
            sees = (p >= at) & ((p - at < 20) | (at < 2))
            keep = ~sees[:, None].expand(-1, 2).clone()
            keep[:, 0] = True  # the other head does not read it
            value, tol = (w[0][keep] for w in want)
            check(out[0][keep], (value, tol), f"{'kv'[t]} at {at}")
            if t == 1:
                assert not torch.isfinite(out[0, sees, 1]).any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lq,window,sinks,heads,kv_heads,dim", [
    (1, 5000, 0, 4, 2, 64), (5, 4096, 20, 3, 1, 128), (40, 3000, 2, 2, 2, 32), (3, 2048, 0, 8, 1, 96)])
def test_few_queries_over_long_windows(gpu, dtype, lq, window, sinks, heads, kv_heads, dim):
    """Too few rows for the chip: the keys are cut, and the parts joined."""
    q, k, v, g = operands(lq, 1, lq, 6001, heads, kv_heads, dim, dtype, "cuda")
    forward_and_gradients(gpu, q, k, v, g, f"{lq} over {window}", window=window, sinks=sinks)
    lengths = torch.tensor([6000], device="cuda")
    forward_and_gradients(gpu, q, k, v, g, f"{lq} over {window}, cut", window=window, sinks=sinks,
                          lengths=lengths)
    if lq > 1:  # the newest key is the last query's alone
        v[0, 6000] = NAN
        out = gpu.window_attention(q, k, v, window=window, sinks=sinks)
        assert torch.isfinite(out[0, :-1]).all() and torch.isnan(out[0, -1]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,lq,heads,kv_heads,dim,window,sinks", [
    (5, 1000, 8, 8, 32, 300, 40), (1, 2111, 4, 2, 64, 900, 3), (9, 300, 16, 16, 128, 250, 0)])
def test_uneven_rounds(gpu, dtype, batch, lq, heads, kv_heads, dim, window, sinks):
    """Blocks beyond whole rounds of the chip: those are cut, with sinks in
    them and in whole blocks, and lengths that leave parts empty."""
    q, k, v, g = operands(lq, batch, lq, lq, heads, kv_heads, dim, dtype, "cuda")
    lengths = torch.tensor([(lq - 100 * b) % (lq + 1) for b in range(batch)], device="cuda")
    forward_and_gradients(gpu, q, k, v, g, f"{batch} x {lq}", window=window, sinks=sinks,
                          lengths=lengths)


def test_rows_repeat(gpu):
    """The same inputs give the same bits, gradients among them."""
    q, k, v, g = operands(9, 2, 700, 700, 8, 2, 128, BF16, "cuda")
    first = None
    for _ in range(3):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = gpu.window_attention(*leaves, window=100, sinks=4)
        got = (out.detach(), *torch.autograd.grad(out, leaves, g))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_another_stream(gpu):
    q, k, v, g = operands(10, 1, 300, 300, 4, 2, 64, BF16, "cuda")
    want = forward_and_gradients(gpu, q, k, v, g, "default stream", window=64, sinks=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = forward_and_gradients(gpu, q, k, v, g, "side stream", window=64, sinks=4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_offsets_beyond_32_bits(gpu):
    """Keys and values whose last token lies past 2^32 values."""
    q, k, v, _ = operands(11, 1, 40, 100, 2, 1, 64, BF16, "cuda")
    stride = 2**26 + 8
    room = torch.empty(99 * stride + 64, dtype=BF16, device="cuda")
    far = room.as_strided((1, 100, 1, 64), (0, stride, 64, 1))
    for name in ("k", "v"):
        far.copy_(k if name == "k" else v)
        kk, vv = (far, v) if name == "k" else (k, far)
        out = gpu.window_attention(q, kk, vv, window=30, sinks=2)
        check(out, reference(q, k, v, window=30, sinks=2)["out"], name)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (8, 1), (64, 4), (300, 0), (1000, 70)])
def test_steps(gpu, dtype, window, sinks):
    held = window + sinks
    lengths = [0, 1, sinks, max(held - 1, 0), held, 3 * held + 5, -1, 63, 64]
    step(gpu, window, lengths, 8, 2, 64, dtype, "cuda", window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [1, 24, 80, 96, 100, 128, 200, 256])
def test_step_head_dimensions(gpu, dtype, dim):
    step(gpu, dim, [5, 400], 6, 2, dim, dtype, "cuda", window=90, sinks=3, index=torch.int64)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 7), (16, 1), (40, 2), (24, 8)])
def test_step_shared_heads(gpu, heads, kv_heads):
    step(gpu, heads, [200, 17, 0], heads, kv_heads, 64, BF16, "cuda", window=130, sinks=4)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_step_unseen_slots(gpu, dtype):
    """Slots that hold nothing yet, or what the query no longer sees."""
    for unseen in (NAN, float("inf")):
        step(gpu, 1, [0, 3, 70, 500, -1], 4, 2, 64, dtype, "cuda", window=100, sinks=4,
             unseen=unseen)
        step(gpu, 2, [0, 3, 70, 500, 130], 4, 2, 64, dtype, "cuda", window=50, sinks=4, slots=777,
             unseen=unseen)


def test_step_of_one_long_sequence(gpu):
    step(gpu, 3, [50_000], 8, 2, 128, BF16, "cuda", window=20_000, sinks=4)
    step(gpu, 4, [30_000, 12], 4, 4, 64, F32, "cuda", window=9000, sinks=1, slots=30_001)


def test_step_wide_scores(gpu):
    step(gpu, 5, [700, 900], 8, 2, 64, BF16, "cuda", window=600, sinks=4, spread=4.0)


def test_step_cache_views(gpu):
    """Caches as views of one allocation, slots apart by more than a row."""
    gen = torch.Generator().manual_seed(6)
    room = torch.randn(3, 70, 2, 2, 64, generator=gen).to(BF16).cuda()
    ck, cv = room[:, :, 0], room[:, :, 1]
    q = torch.randn(3, 8, 64, generator=gen).to(BF16).cuda()
    kv = torch.randn(3, 4, 64, generator=gen).to(BF16).cuda()
    n = torch.tensor([69, 10, 200], device="cuda")
    want = gpu.window_attention_step(q, kv[:, :2], kv[:, 2:], ck.clone(), cv.clone(), n, window=60,
                                     sinks=4)
    got = gpu.window_attention_step(q, kv[:, :2], kv[:, 2:], ck, cv, n, window=60, sinks=4)
    assert torch.equal(got, want)


def test_step_in_a_graph(gpu):
    """Captured steps: a replay reads lengths and queries as they are then."""
    gen = torch.Generator(device="cuda").manual_seed(7)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=F32).to(BF16)

    q, k, v = normal(4, 8, 64), normal(4, 2, 64), normal(4, 2, 64)
    caches = [normal(4, 516, 2, 64) for _ in range(2)]
    mirror = [c.clone() for c in caches]
    n = torch.tensor([0, 100, 515, 5000], device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gpu.window_attention_step(q, k, v, *caches, n, window=512, sinks=4)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gpu.window_attention_step(q, k, v, *caches, n, window=512, sinks=4)
        n += 1
    n.copy_(torch.tensor([0, 100, 515, 5000]))
    caches[0].copy_(mirror[0])
    caches[1].copy_(mirror[1])
    eager_n = n.clone()
    for _ in range(4):
        for t in (q, k, v):
            t.copy_(normal(*t.shape))
        graph.replay()
        want = gpu.window_attention_step(q, k, v, *mirror, eager_n, window=512, sinks=4)
        eager_n += 1
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(n, eager_n)
        assert all(torch.equal(a, b) for a, b in zip(caches, mirror))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_prompt_then_steps(gpu, dtype):
    prompt_then_steps(gpu, "cuda", dtype, window=70, sinks=5, prompt=[3, 250, 74], more=9, dim=64)


def test_caches_elsewhere_are_refused(gpu):
    q, k = torch.zeros(1, 2, 8), torch.zeros(1, 1, 8)
    cache = torch.zeros(1, 9, 1, 8)
    with pytest.raises(ValueError, match="caches must be on"):
        gpu.window_attention_step(q, k, k, cache, cache.clone(), torch.tensor([0]), window=4)


def test_training_in_a_graph(gpu):
    """Forward and gradients captured once, in parts and with sinks' far pass;
    every replay against the eager call on the same inputs."""
    q, k, v, g = operands(13, 3, 700, 700, 4, 2, 64, BF16, "cuda")
    pattern = {"window": 128, "sinks": 4}
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def call():
        out = gpu.window_attention(*leaves, **pattern)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(3):
        with torch.no_grad():
            q.copy_(operands(20 + i, 3, 700, 700, 4, 2, 64, BF16, "cuda")[0])
        want = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
