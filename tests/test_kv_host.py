"""The int8 key/value cache and its attention without a device: sizes, refusals, and calls with nothing to do."""
import ctypes as C

import numpy as np
import pytest

from vtl_amd import HipKVCache, capi

E, OK = capi.ERR_INVALID_ARG, capi.OK
ONE = 16     # an address that no accepted call of this file reads


def cache(**changes):
    c = capi.KVCache(ONE, 4, 32, 2, 64)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


def batch(**changes):
    b = capi.KVBatch(3, 5, ONE, ONE, None, 3, 0, 0)
    for name, value in changes.items():
        setattr(b, name, value)
    return b


def calls(c, b, k=ONE, v=ONE, stride=128, heads=4, q=1 << 20, out=1 << 24, q_stride=256, out_stride=256, ws=None, ws_bytes=0):
    c, b = (None if x is None else C.byref(x) for x in (c, b))
    return [capi.status("vtl_hip_kv_write_f32", c, b, k, stride, v, stride),
            capi.status("vtl_hip_kv_read_f32", c, b, k, stride, v, stride),
            capi.status("vtl_hip_attention_i8_f32", c, b, q, q_stride, heads, 1.0, 1, out, out_stride, ws, ws_bytes)]


@pytest.mark.parametrize("pages,page,heads,dim", [(1, 16, 1, 1), (4, 32, 2, 64), (7, 48, 3, 72), (1000, 128, 8, 128), (2, 4096, 1, 256)])
def test_bytes(pages, page, heads, dim):
    d = -(-dim // 16) * 16
    assert capi.lib().vtl_hip_kv_cache_bytes(pages, page, heads, dim) == pages * heads * page * (2 * d + 8)


@pytest.mark.parametrize("sizes", [(0, 16, 1, 64), (-1, 16, 1, 64), (1, 0, 1, 64), (1, 8, 1, 64), (1, 24, 1, 64), (1, 4112, 1, 64), (1, 16, 0, 64),
                                   (1, 16, -2, 64), (1, 16, 1, 0), (1, 16, 1, 257), (1, 16, 1, -3), (0x7fffffff, 4096, 0x7fffffff, 256)])
def test_sizes_that_no_cache_has(sizes):
    assert capi.lib().vtl_hip_kv_cache_bytes(*sizes) == 0
    with pytest.raises(ValueError):
        HipKVCache(*sizes)
    assert calls(capi.KVCache(ONE, *sizes), batch()) == [E] * 3


@pytest.mark.parametrize("c,b", [
    (None, batch()), (cache(), None), (cache(pages=None), batch()), (cache(pages=24), batch()),
    (cache(), batch(batch=-1)), (cache(), batch(rows=-1)), (cache(), batch(max_pages=0)), (cache(), batch(page_table=None)),
    (cache(), batch(lengths=None)), (cache(), batch(rows=4)), (cache(), batch(most_rows=-1)), (cache(), batch(most_length=-1))])
def test_refused(c, b):
    assert calls(c, b) == [E] * 3


def test_refused_tensors():
    assert calls(cache(), batch(), k=None)[0] == E and calls(cache(), batch(), v=None)[0] == E
    assert calls(cache(), batch(), stride=127)[:2] == [E, E]
    for more in ({"q": None}, {"out": None}, {"heads": 0}, {"heads": 3}, {"heads": -2}, {"q_stride": 255}, {"out_stride": 255},
                 {"out": (1 << 20) + 512},                                        # results over the queries
                 {"ws": 20, "ws_bytes": 1 << 30}, {"ws": 16, "ws_bytes": 8}):    # not aligned, too small
        assert calls(cache(), batch(max_pages=4000, most_length=100000), **more)[2] == E, more


def test_more_than_is_counted():
    u = capi.ERR_UNSUPPORTED
    assert calls(cache(), batch(rows=(1 << 30) + 1, starts=ONE), q_stride=256, out=1 << 60) == [u] * 3
    assert calls(cache(), batch(batch=(1 << 30) + 1, rows=(1 << 30) + 1), out=1 << 60) == [u] * 3
    assert calls(cache(kv_heads=1000), batch(batch=1 << 24, rows=1 << 24), stride=64000, heads=1000, q_stride=64000, out_stride=64000, out=1 << 60) == [u] * 3


def test_rows_of_more_than_32_bits():
    wide = {"q_stride": 1 << 32, "out_stride": 1 << 32, "out": 1 << 60}
    assert calls(cache(kv_heads=1, head_dim=256), batch(batch=1, rows=1), stride=256, heads=1 << 23, **wide)[2] == capi.ERR_UNSUPPORTED
    assert calls(cache(kv_heads=1), batch(), stride=64, heads=1 << 30, q_stride=1 << 40, out_stride=1 << 40, out=1 << 60)[2] == capi.ERR_UNSUPPORTED


def test_nothing_to_do():
    assert calls(cache(), batch(batch=0, rows=0, page_table=None, lengths=None), k=None, v=None, q=None, out=None) == [OK] * 3
    assert calls(cache(), batch(rows=0, starts=ONE)) == [OK] * 3
    assert calls(cache(), batch(batch=0, rows=3)) == [OK] * 3       # rows of no sequence
    assert calls(cache(), batch(), k=None, v=None)[1] == OK


def test_workspace_of_refused_arguments_is_none():
    w = capi.lib().vtl_hip_attention_i8_workspace
    assert w(None, C.byref(batch()), 4) == 0 and w(C.byref(cache()), None, 4) == 0
    assert w(C.byref(cache(page_size=24)), C.byref(batch()), 4) == 0 and w(C.byref(cache()), C.byref(batch()), 3) == 0
    assert w(C.byref(cache()), C.byref(batch(rows=0, batch=0)), 4) == 0


@pytest.mark.parametrize("per_page", range(1, 257))
def test_division_by_the_groups_of_a_page(per_page):
    """What the kernels do to find a page: (group * ceil(2^32 / per_page)) >> 32, exact for groups below 2^24."""
    if per_page == 1:
        return
    magic = (2 ** 32 + per_page - 1) // per_page
    q = np.arange(0, 2 ** 24 // per_page + 1, dtype=np.uint64)
    for g in (q * per_page, q * per_page + np.uint64(per_page - 1)):
        g = g[g < 2 ** 24]
        assert magic < 2 ** 32 and np.array_equal((g * np.uint64(magic)) >> np.uint64(32), g // np.uint64(per_page))
