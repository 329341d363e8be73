"""Refusals of the C entry points of rotary positions and paged caches, before any
HIP call."""

from __future__ import annotations

import ctypes

import pytest

import _capi

I32, I64, P, F64 = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_double


class Rotation(ctypes.Structure):
    _fields_ = [("dim", I64), ("interleaved", I32), ("inverse", I32), ("magnitude", F64), ("turns", P)]


class RotaryDesc(ctypes.Structure):
    _fields_ = [("vtype", I32), ("itype", I32), ("batch", I64), ("tokens", I64), ("heads", I64),
                ("dim", I64), ("x", P), ("x_strides", I64 * 3), ("starts", P), ("positions", P),
                ("position_strides", I64 * 2), ("rotation", Rotation)]


class Cache(ctypes.Structure):
    _fields_ = [("n_pages", I64), ("page_size", I64), ("kv_heads", I64), ("dim", I64), ("k", P),
                ("v", P), ("k_strides", I64 * 3), ("v_strides", I64 * 3), ("pages", P),
                ("pages_stride", I64), ("width", I64), ("pages_itype", I32), ("reserved", I32)]


class AppendDesc(ctypes.Structure):
    _fields_ = [("vtype", I32), ("itype", I32), ("batch", I64), ("tokens", I64), ("heads", I64),
                ("q", P), ("k", P), ("v", P), ("q_strides", I64 * 3), ("k_strides", I64 * 3),
                ("v_strides", I64 * 3), ("starts", P), ("lengths", P), ("cache", Cache),
                ("rotation", Rotation)]


class AttentionDesc(ctypes.Structure):
    _fields_ = [("vtype", I32), ("itype", I32), ("batch", I64), ("tokens", I64), ("heads", I64),
                ("window", I64), ("sinks", I64), ("shared_pages", I64), ("scale", F64), ("q", P),
                ("q_strides", I64 * 3), ("starts", P), ("lengths", P), ("cache", Cache)]


SOME = 4096  # an address that no refused call reads


def cache():
    return Cache(n_pages=4, page_size=16, kv_heads=2, dim=64, k=SOME, v=SOME,
                 k_strides=(2048, 128, 64), v_strides=(2048, 128, 64), pages=SOME, pages_stride=3,
                 width=3)


def descriptors():
    rotation = Rotation(dim=64, magnitude=1.0, turns=SOME)
    return {
        "rotary": RotaryDesc(batch=2, tokens=1, heads=4, dim=64, x=SOME, x_strides=(256, 256, 64),
                             rotation=rotation),
        "append": AppendDesc(batch=2, tokens=1, heads=4, q=SOME, k=SOME, v=SOME,
                             q_strides=(256, 256, 64), k_strides=(128, 128, 64),
                             v_strides=(128, 128, 64), cache=cache(), rotation=rotation),
        "attention": AttentionDesc(batch=2, tokens=1, heads=4, window=2**40, scale=0.125, q=SOME,
                                   q_strides=(256, 256, 64), cache=cache()),
    }


def call(name, desc, host, out=None, scratch=None, size=0):
    L = _capi.lib()
    ref = None if desc is None else ctypes.byref(desc)
    if name == "rotary":
        return L.msx_rotary_cpu(ref, P(out), 1) if host else L.msx_rotary(ref, P(out), None)
    if name == "append":
        return (L.msx_paged_cache_append_cpu(ref, P(out), 1) if host
                else L.msx_paged_cache_append(ref, P(out), None))
    return (L.msx_paged_attention_cpu(ref, P(out), 1) if host
            else L.msx_paged_attention(ref, P(out), P(scratch), ctypes.c_size_t(size), None))


def scratch_of(desc):
    f = _capi.lib().msx_paged_attention_scratch
    f.restype = ctypes.c_size_t
    return f(None if desc is None else ctypes.byref(desc))


@pytest.mark.parametrize("host", [False, True])
@pytest.mark.parametrize("name", ["rotary", "append", "attention"])
def test_refused_descriptors(name, host):
    assert call(name, None, host) == _capi.EINVAL and "NULL" in _capi.last_error()

    def refused(status, text, **changes):
        d = descriptors()[name]
        for key, value in changes.items():
            at = d
            *path, last = key.split("__")
            for part in path:
                at = getattr(at, part)
            setattr(at, last, value)
        assert call(name, d, host, out=SOME) == status, changes
        assert text in _capi.last_error(), (_capi.last_error(), changes)
        if name == "attention":
            assert scratch_of(d) == 0

    refused(_capi.ETYPE, "values", vtype=3)
    refused(_capi.ETYPE, "positions", itype=9)
    refused(_capi.EINVAL, "batch", batch=-1)
    refused(_capi.EINVAL, "batch", batch=2**31)
    refused(_capi.EINVAL, "token count", tokens=2**30)
    refused(_capi.EINVAL, "heads", heads=70000)
    if name == "rotary":
        refused(_capi.EINVAL, "x is NULL", x=None)
    if name != "attention":
        refused(_capi.EINVAL, "even number", rotation__dim=66)
        refused(_capi.EINVAL, "even number", rotation__dim=3)
        refused(_capi.EINVAL, "magnitude", rotation__magnitude=1e300)
        refused(_capi.EINVAL, "turns", rotation__turns=None)
    if name == "rotary":
        refused(_capi.EINVAL, "dimension", dim=257)
        return
    refused(_capi.EINVAL, "dimension", cache__dim=0)
    refused(_capi.ETYPE, "pages", cache__pages_itype=4)
    refused(_capi.EINVAL, "heads", cache__kv_heads=0)
    refused(_capi.EINVAL, "page count", cache__n_pages=2**31)
    refused(_capi.EINVAL, "hold", cache__page_size=0)
    refused(_capi.EINVAL, "less than 2^30", cache__width=2**26)
    refused(_capi.EINVAL, "pages is NULL", cache__pages=None)
    refused(_capi.EINVAL, "caches", cache__v=None)
    refused(_capi.EINVAL, "NULL", q=None)
    if name == "append":
        return
    refused(_capi.EINVAL, "multiple", heads=5)
    refused(_capi.EINVAL, "window", window=0)
    refused(_capi.EINVAL, "sinks", sinks=-1)
    refused(_capi.EINVAL, "scale", scale=float("nan"))
    refused(_capi.EINVAL, "shared_pages", shared_pages=4)


@pytest.mark.parametrize("name", ["rotary", "append", "attention"])
def test_missing_outputs(name):
    assert call(name, descriptors()[name], False) == _capi.EINVAL
    assert "out is NULL" in _capi.last_error()


def test_scratch_is_asked_for():
    d = descriptors()["attention"]
    d.cache.width = 1000  # of more keys than a workgroup takes
    n = scratch_of(d)
    assert n > 0
    for scratch, size in ((None, n), (SOME, n - 1), (SOME + 8, n)):
        assert call("attention", d, False, out=SOME, scratch=scratch, size=size) == _capi.EINVAL
        assert "scratch" in _capi.last_error()
    assert scratch_of(None) == 0


def test_more_rows_than_are_counted():
    d = descriptors()["attention"]
    d.batch, d.tokens = 2**31 - 1, 2**29
    assert scratch_of(d) == 0
    assert call("attention", d, False, out=SOME, scratch=SOME, size=2**60) == _capi.EINVAL
    assert "rows" in _capi.last_error()


def test_nothing_to_do():
    for name, d in descriptors().items():
        for host in (False, True):
            d.tokens = 0
            assert call(name, d, host) == _capi.OK
