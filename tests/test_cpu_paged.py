"""Paged caches and the attention over them on the host; refusals."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from _paged_checks import append_case, paged_case, prompt_then_steps

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1, 5, 16])
def test_single_tokens(cpu, dtype, size):
    paged_case(cpu, "cpu", dtype, [0, 1, 15, -1, 16, 40], size=size)


@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (7, 4), (100, 3), (None, 2)])
@pytest.mark.parametrize("tokens", [1, 4])
def test_window_and_sinks(cpu, window, sinks, tokens):
    paged_case(cpu, "cpu", torch.float32, [0, 3, 31, 18], tokens=tokens, window=window, sinks=sinks,
               size=4)


@pytest.mark.parametrize("layout", ["plain", "packed", "odd"])
@pytest.mark.parametrize("index,table_index", [(torch.int32, torch.int64), (torch.int64, torch.int32)])
def test_layouts_and_indices(cpu, layout, index, table_index):
    paged_case(cpu, "cpu", torch.float32, [9, 4], tokens=3, lengths=[3, 1], layout=layout, index=index,
               table_index=table_index, heads=6, kv_heads=3, dim=20, size=6)


def test_shared_pages(cpu):
    paged_case(cpu, "cpu", torch.float32, [40, 33, -1, 20], tokens=2, shared=2, size=8)


def test_pages_that_are_not_there(cpu):
    paged_case(cpu, "cpu", torch.float32, [30, 9], holes=[(0, 1), (1, 0), (1, 1)], size=8)
    paged_case(cpu, "cpu", torch.float32, [30], width=2, size=8)  # queries beyond the table
    paged_case(cpu, "cpu", torch.float32, [2**62, 2**63 - 1], width=2, size=8, window=5, sinks=3,
               index=torch.int64, poison=False)
    paged_case(cpu, "cpu", torch.float32, [0, 0], width=0, size=8)


def test_nothing_to_attend(cpu):
    empty = torch.zeros(0, 4, 2, 8)
    pages = torch.zeros(2, 0, dtype=torch.int32)
    assert torch.equal(cpu.paged_attention(torch.ones(2, 1, 4, 8), empty, empty, pages),
                       torch.zeros(2, 1, 4, 8))
    assert cpu.paged_attention(torch.ones(0, 1, 4, 8), empty, empty, pages[:0]).shape == (0, 1, 4, 8)
    assert cpu.paged_attention(torch.ones(2, 0, 4, 8), empty, empty, pages).shape == (2, 0, 4, 8)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("size,layout", [(16, "plain"), (5, "packed"), (1, "odd")])
def test_append(cpu, dtype, interleaved, size, layout):
    append_case(cpu, "cpu", dtype, [0, 7, -1, 30], tokens=6, lengths=[6, 1, 3, 0], size=size,
                layout=layout, interleaved=interleaved, rotated=20)


def test_append_without_rotation_or_place(cpu):
    append_case(cpu, "cpu", torch.float32, [3, 9], tokens=4, rotate=False)
    append_case(cpu, "cpu", torch.float32, [3, 9], tokens=4, with_q=False)
    append_case(cpu, "cpu", torch.float32, [3, 9], tokens=9, size=4, holes=[(0, 1), (1, 4)])
    append_case(cpu, "cpu", torch.float32, [3, 9], tokens=9, size=4, width=3)  # beyond the table
    append_case(cpu, "cpu", torch.float32, [2**62, 1], tokens=2, size=4, width=3, index=torch.int64,
                with_q=False)


@pytest.mark.parametrize("window,sinks", [(None, 0), (9, 2)])
def test_prompt_then_steps(cpu, window, sinks):
    prompt_then_steps(cpu, "cpu", torch.float32, window=window, sinks=sinks)


def caches(dtype=torch.float32, dim=8):
    return [torch.zeros(4, 4, 2, dim, dtype=dtype) for _ in range(2)]


def test_versions(cpu):
    ck, cv = caches()
    k = torch.ones(1, 2, 2, 8)
    cpu.paged_cache_append(k, k, ck, cv, torch.tensor([[1]]))
    assert ck._version == 1 and cv._version == 1 and (ck[1, :2] == 1).all() and ck.sum() == 32
    cpu.paged_attention(torch.ones(1, 2, 4, 8), ck, cv, torch.tensor([[1]]))
    assert ck._version == 1


def test_mixed_index_types(cpu):
    ck, cv = caches()
    k = torch.ones(2, 2, 2, 8)
    pages = torch.tensor([[0], [1]])
    starts, lengths = torch.tensor([1, 0]), torch.tensor([2, 1], dtype=torch.int32)
    cpu.paged_cache_append(k, k, ck, cv, pages, starts=starts, lengths=lengths)
    assert ck[:, :, 0, 0].tolist() == [[0, 1, 1, 0], [1, 0, 0, 0], [0] * 4, [0] * 4]
    out = cpu.paged_attention(torch.ones(2, 2, 4, 8), ck, cv, pages, starts=starts, lengths=lengths)
    assert (out[1, 1] == 0).all() and (out[0] != 0).all()


def test_refused_appends(cpu):
    ck, cv = caches()
    k, pages, r = torch.ones(1, 2, 2, 8), torch.tensor([[1, 0]]), cpu.Rotary(8)
    call = cpu.paged_cache_append
    with pytest.raises(TypeError, match="Rotary"):
        call(k, k, ck, cv, pages, rotation=8)
    with pytest.raises(TypeError, match="one dtype"):
        call(k, k.half(), ck, cv, pages)
    with pytest.raises(TypeError, match="pages"):
        call(k, k, ck, cv, pages.float())
    with pytest.raises(ValueError, match="pages"):
        call(k, k, ck, cv, pages[0])
    with pytest.raises(ValueError, match="pages"):
        call(k, k, ck, cv, pages.expand(2, -1))
    with pytest.raises(ValueError, match="has no rotation"):
        call(k, k, ck, cv, pages, q=k)
    with pytest.raises(ValueError, match="rotates 8"):
        call(k[..., :6], k[..., :6], ck[..., :6], cv[..., :6], pages, rotation=r)
    with pytest.raises(ValueError, match="cache"):
        call(k, k, ck, cv[:2], pages)
    with pytest.raises(ValueError, match="k must have shape"):
        call(k[:, :, :1], k[:, :, :1], ck, cv, pages)
    with pytest.raises(ValueError, match="q must have shape"):
        call(k, k, ck, cv, pages, rotation=r, q=torch.ones(1, 3, 2, 8))
    with pytest.raises(ValueError, match="expanded"):
        call(k, k, ck[:1].expand(4, -1, -1, -1), cv, pages)
    with pytest.raises(ValueError, match="require grad"):
        call(k, k, ck.clone().requires_grad_(), cv, pages)
    with pytest.raises(TypeError, match="torch tensors"):
        call(k, k, ck.numpy(), cv, pages)
    with pytest.raises(ValueError, match="starts"):
        call(k, k, ck, cv, pages, starts=torch.zeros(2, dtype=torch.int32))
    assert ck.abs().max() == 0 and cv.abs().max() == 0 and ck._version == 0


def test_refused_attention(cpu):
    ck, cv = caches()
    q, pages = torch.ones(1, 2, 4, 8), torch.tensor([[1, 0]])
    call = cpu.paged_attention
    for bad, error, text in [
        (dict(window=0), ValueError, "window"), (dict(sinks=-1), ValueError, "sinks"),
        (dict(shared_pages=3), ValueError, "shared_pages"),
        (dict(shared_pages=-1), ValueError, "shared_pages"),
        (dict(scale=float("inf")), ValueError, "scale"),
        (dict(starts=torch.zeros(1)), (TypeError, ValueError), "int32 or int64"),
        (dict(lengths=torch.zeros(2, dtype=torch.int32)), ValueError, "lengths"),
    ]:
        with pytest.raises(error, match=text):
            call(q, ck, cv, pages, **bad)
    with pytest.raises(ValueError, match="multiple"):
        call(q[:, :, :3], ck, cv, pages)
    with pytest.raises(ValueError, match="256"):
        call(torch.ones(1, 1, 2, 300), *caches(dim=300), pages)
    with pytest.raises(TypeError, match="float64"):
        call(q.double(), ck.double(), cv.double(), pages)
    with pytest.raises(TypeError, match="one dtype"):
        call(q.half(), ck, cv, pages)
    with pytest.raises(ValueError, match="expects q of shape"):
        call(q[0], ck, cv, pages)
    with pytest.raises(ValueError, match="shape"):
        call(q[..., :4], ck, cv, pages)


def test_transforms_refused(cpu):
    ck, cv = caches()
    q, pages = torch.ones(3, 1, 2, 4, 8), torch.tensor([[1, 0]])
    with pytest.raises(NotImplementedError, match="paged_attention"):
        torch.func.vmap(lambda q: cpu.paged_attention(q, ck, cv, pages))(q)
    k = torch.ones(1, 2, 2, 8)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="paged_cache_append"):
            cpu.paged_cache_append(fwd.make_dual(k, k), k, ck, cv, pages)
    assert ck.abs().max() == 0
