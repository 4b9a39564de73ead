"""Attention over the int8 cache where workgroups share sequences: their parts meet within the launch, or are added up by a launch of their own (calls
recorded into a graph, streams without counters).  The same bits either way."""
import ctypes as C

import numpy as np
import pytest

from kv_cases import SHARED
from kv_reference import Cache
from vtl_amd import capi
from vtl_amd.storage import HipStorage
from vtl_amd.tensor import HipTensor

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


def normal(seed, *shape, std=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * std).astype(np.float32)


def random_cache(lengths, page, kv_heads, dim, seed):
    c = Cache(lengths, page, kv_heads, dim, seed=seed, fill=False)
    _, _, ks, vs = c.parts()
    rng = np.random.default_rng(seed)
    ks[:], vs[:] = rng.uniform(0.01, 0.03, ks.shape), rng.uniform(0.01, 0.03, vs.shape)      # codes are any
    return c.to_device()


class Call:
    """One call with its own workspace, which is overwritten before each."""

    def __init__(self, c, counts, heads, dim, seed):
        self.b, self.c, self.heads, self.dim = c.batch(counts), c, heads, dim
        self.q = HipTensor.from_host(normal(seed, self.b.rows, heads * dim))
        self.out = HipTensor.empty([self.b.rows, heads * dim], np.float32)
        self.need = capi.lib().vtl_hip_attention_i8_workspace(C.byref(c.cache.handle), C.byref(self.b.handle), heads)
        self.ws = HipStorage.empty(max(self.need, 16), np.uint8)
        self.noise = np.full(self.ws.size, 0xff, np.uint8)      # NaN

    def enqueue(self):
        width = self.heads * self.dim
        capi.call("vtl_hip_attention_i8_f32", C.byref(self.c.cache.handle), C.byref(self.b.handle), self.q.ptr, width, self.heads, self.dim ** -0.5, 1,
                  self.out.ptr, width, self.ws.ptr, self.ws.size)

    def spoil(self):
        capi.call("vtl_hip_sync")
        capi.call("vtl_hip_memcpy_h2d", self.ws.ptr, self.noise.ctypes.data, self.noise.nbytes)
        x = np.full(self.out.size, np.nan, np.float32)
        capi.call("vtl_hip_memcpy_h2d", self.out.ptr, x.ctypes.data, x.nbytes)

    def result(self):
        return self.out.cpu().view(np.uint32)


@pytest.fixture
def hiprt():
    rt = C.CDLL("libamdhip64.so")
    yield rt
    capi.call("vtl_hip_sync")
    capi.call("vtl_hip_set_stream", None)


def new_stream(rt):
    st = C.c_void_p()
    assert rt.hipStreamCreate(C.byref(st)) == 0
    return st


CASES = {f"{'_'.join(map(str, variant))}": case for variant, case in SHARED.items()}
CASES["many"] = ([900, 1100], [130, 40], 16, 4, 96)
CASES["many_256"] = ([600, 500], [40, 30], 4, 4, 256)


@pytest.mark.parametrize("case", CASES.values(), ids=CASES.keys())
def test_recorded_calls_give_the_same_bits(hiprt, case):
    lengths, counts, heads, kv_heads, dim = case
    c = random_cache(lengths, 32, kv_heads, dim, seed=len(lengths))
    call = Call(c, counts, heads, dim, seed=3)
    assert call.need > 0
    call.spoil()
    call.enqueue()
    want = call.result()
    assert np.isfinite(want.view(np.float32)).all()
    st, graph, run = new_stream(hiprt), C.c_void_p(), C.c_void_p()
    capi.call("vtl_hip_set_stream", st)
    assert hiprt.hipStreamBeginCapture(st, 0) == 0
    call.enqueue()
    assert hiprt.hipStreamEndCapture(st, C.byref(graph)) == 0
    assert hiprt.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    try:
        for _ in range(3):
            capi.call("vtl_hip_set_stream", st)
            call.spoil()
            assert hiprt.hipGraphLaunch(run, st) == 0
            capi.call("vtl_hip_sync")
            assert np.array_equal(call.result(), want)
            capi.call("vtl_hip_set_stream", None)
            call.spoil()
            call.enqueue()
            assert np.array_equal(call.result(), want)
    finally:
        capi.call("vtl_hip_sync")
        hiprt.hipGraphExecDestroy(run)
        hiprt.hipGraphDestroy(graph)
        capi.call("vtl_hip_set_stream", None)
        hiprt.hipStreamDestroy(st)
