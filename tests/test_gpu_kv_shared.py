"""The int8 key/value cache where sequences share pages, and where two threads use one cache."""
import threading

import numpy as np
import pytest

from kv_reference import Cache
from test_gpu_kv_meeting import Call, hiprt, new_stream, normal, random_cache  # noqa: F401
from vtl_amd import attention_i8_hip, capi, kv_read_hip, kv_write_hip
from vtl_amd.tensor import HipTensor

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


@pytest.mark.parametrize("counts", [None, [4, 9, 1], [70, 40, 100]])
def test_sequences_that_share_their_first_pages(guard_bands, counts):
    """Three sequences that begin with the same 256 tokens, which lie in the cache once: each writes its own rows behind them."""
    c = Cache([300, 420, 390], 64, 2, 128, seed=31)
    c.table[1:, :4] = c.table[0, :4]
    c.to_device()
    rows = [1, 1, 1] if counts is None else counts
    c.lengths[:] = [256 + max(n, 44) for n in rows]
    c.table = np.pad(c.table, ((0, 0), (0, 1)), constant_values=-1)
    b = c.batch(counts)
    k, v, q = normal(1, b.rows, 2, 128), normal(2, b.rows, 2, 128), normal(3, b.rows, 8, 128)
    kv_write_hip(c.cache, b, HipTensor.from_host(k), HipTensor.from_host(v))
    assert np.array_equal(c.fetch(), c.written(k, v))
    want_k, want_v = c.read(b.rows)
    got_k, got_v = kv_read_hip(c.cache, b)
    assert np.array_equal(got_k.cpu(), want_k) and np.array_equal(got_v.cpu(), want_v)
    for causal in (True, False):
        want, far = c.attend(q, 8, np.float32(128 ** -0.5), causal)
        assert (np.abs(attention_i8_hip(c.cache, b, HipTensor.from_host(q), 8, causal=causal).cpu() - want) <= far).all()


def test_two_threads_on_streams_of_their_own(hiprt):
    """One cache, read by both; each thread has a stream, calls and workspaces."""
    c = random_cache([3000, 700, 1500], 64, 4, 128, seed=32)
    mixes = [(None, 8), ([5, 9, 30], 8), ([70, 130, 20], 8), ([2, 1, 4], 16)]
    want = []
    for i, (counts, heads) in enumerate(mixes):
        call = Call(c, counts, heads, 128, seed=i)
        call.enqueue()
        want.append(call.result())
    wrong, streams, one_at_a_time = [], [new_stream(hiprt) for _ in range(2)], threading.Lock()

    def work(stream):
        try:
            capi.call("vtl_hip_set_device", 0)
            capi.call("vtl_hip_set_stream", stream)
            with one_at_a_time:       # Cache.batch writes down the starts
                calls = [Call(c, counts, heads, 128, seed=i) for i, (counts, heads) in enumerate(mixes)]
            for _ in range(20):
                for call in calls:
                    call.enqueue()
                capi.call("vtl_hip_sync")
                wrong.extend(i for i, call in enumerate(calls) if not np.array_equal(call.result(), want[i]))
        except Exception as e:      # told to the test
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in streams]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for s in streams:
        hiprt.hipStreamDestroy(s)
    assert not wrong, wrong
