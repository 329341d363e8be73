"""How paged attention is planned, as far as its scratch shows it: none where a
workgroup takes all keys of a sequence and kv head, some where they are cut."""

from __future__ import annotations

import pytest

from test_cpu_paged_capi import AttentionDesc, Cache, SOME, scratch_of

F32, F16, BF16 = 0, 1, 2  # MSX_F32, MSX_F16, MSX_BF16


def scratch(vtype, batch, keys, *, heads=32, kv_heads=8, dim=256, tokens=1, size=16):
    row = kv_heads * dim
    cache = Cache(n_pages=4, page_size=size, kv_heads=kv_heads, dim=dim, k=SOME, v=SOME,
                  k_strides=(size * row, row, dim), v_strides=(size * row, row, dim), pages=SOME,
                  pages_stride=keys // size, width=keys // size)
    return scratch_of(AttentionDesc(vtype=vtype, batch=batch, tokens=tokens, heads=heads, window=2**40,
                                    scale=0.125, q=SOME, q_strides=(heads * dim, heads * dim, dim),
                                    cache=cache))


@pytest.mark.parametrize("vtype", [F16, BF16])
@pytest.mark.parametrize("batch,keys,whole", [
    # 64 workgroups, and 2,400, are cut; as many as fill the chip up to four times are not
    (8, 256, True), (8, 304, False), (8, 512, False), (30, 304, True), (30, 512, True),
    (60, 512, True), (128, 512, True), (30, 528, False), (300, 256, True), (300, 512, False)])
def test_wide_heads_of_few_keys(vtype, batch, keys, whole):
    assert (scratch(vtype, batch, keys) == 0) == whole


@pytest.mark.parametrize("vtype,batch,keys,whole", [
    (BF16, 1, 1536, True), (BF16, 1, 1552, False), (BF16, 30, 1792, True), (BF16, 30, 1808, False),
    (F32, 1, 512, True), (F32, 1, 528, False), (F32, 30, 896, True), (F32, 30, 912, False)])
def test_narrow_heads_of_few_keys(vtype, batch, keys, whole):
    assert (scratch(vtype, batch, keys, dim=64) == 0) == whole
