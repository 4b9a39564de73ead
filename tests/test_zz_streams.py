"""Calls on more streams than the library keeps counters for.  The last file of all: the streams that have them keep them, and what other tests run on
streams of their own would take other paths behind this one."""
import numpy as np
import pytest

from kv_cases import SHARED
from test_gpu_kv_meeting import Call, hiprt, new_stream, random_cache  # noqa: F401
from vtl_amd import capi

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


def test_attention_on_more_streams_than_have_counters(hiprt):
    """Calls on 20 streams at once, each with a workspace of its own: the first 16 streams of a process meet within the launch."""
    lengths, counts, heads, kv_heads, dim = SHARED[128, 1, 8]
    c = random_cache(lengths, 64, kv_heads, dim, seed=5)
    calls = [Call(c, counts, heads, dim, seed=i % 3) for i in range(20)]
    want = []
    for call in calls[:3]:
        call.enqueue()
        want.append(call.result())
    streams = [new_stream(hiprt) for _ in calls]
    try:
        for _ in range(3):
            for call in calls:
                call.spoil()
            for st, call in zip(streams, calls):
                capi.call("vtl_hip_set_stream", st)
                call.enqueue()
            for st in streams:
                capi.call("vtl_hip_set_stream", st)
                capi.call("vtl_hip_sync")
            for i, call in enumerate(calls):
                assert np.array_equal(call.result(), want[i % 3]), i
    finally:
        capi.call("vtl_hip_set_stream", None)
        for st in streams:
            hiprt.hipStreamDestroy(st)
