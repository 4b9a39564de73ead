"""The int8 key/value cache and the attention over it on the device, against their definitions in 64 bits (kv_reference.py)."""
import ctypes as C

import numpy as np
import pytest

from kv_reference import Cache, quantize
from vtl_amd import (HipKVBatch, QuantLinearLayer, attention_i8_hip, capi, kv_read_hip, kv_write_hip)
from vtl_amd.storage import HipStorage
from vtl_amd.tensor import HipTensor

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


def normal(seed, *shape, std=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * std).astype(np.float32)


# -- cache: bytes of the pages, and values read back ---------------------------------------------

WRITES = [  # lengths, rows of each, page, heads, dim
    ([1], None, 16, 1, 1), ([5, 0, 17, 64], None, 16, 2, 64), ([300] * 9, None, 64, 8, 128), ([33, 7], [33, 7], 32, 3, 72),
    ([100, 260, 16, 31], [37, 130, 16, 1], 48, 2, 80), ([70, 12, 5], [3, 0, 9], 16, 2, 96), ([1000], [1000], 128, 1, 256),
    ([40, 41, 42], [17, 18, 19], 16, 5, 33), ([513, 129], [500, 128], 64, 4, 128), ([96], [64], 16, 2, 17)]


@pytest.mark.parametrize("lengths,counts,page,heads,dim", WRITES)
@pytest.mark.parametrize("fused", [False, True], ids=["dense", "fused"])
def test_write_and_read(guard_bands, lengths, counts, page, heads, dim, fused):
    c = Cache(lengths, page, heads, dim, seed=len(lengths)).to_device()
    b = c.batch(counts)
    k, v = normal(1, b.rows, heads, dim), normal(2, b.rows, heads, dim, std=30.0)
    k[..., ::7] *= 20.0
    if b.rows:
        k[0, 0], v[-1, -1] = 0.0, 0.0             # scale 0
        v[0, 0, 0] = np.nan
    if fused:
        both = np.concatenate([normal(3, b.rows, 5), k.reshape(b.rows, -1), v.reshape(b.rows, -1)], 1)
        t = HipTensor.from_host(both)
        kv_write_hip(c.cache, b, t, t, k_first=5, v_first=5 + heads * dim)
    else:
        kv_write_hip(c.cache, b, HipTensor.from_host(k), HipTensor.from_host(v))
    want = c.written(k, v)
    assert np.array_equal(c.fetch(), want)
    got_k, got_v = kv_read_hip(c.cache, b)
    want_k, want_v = c.read(b.rows)
    assert np.array_equal(got_k.cpu(), want_k) and np.array_equal(got_v.cpu(), want_v)
    for t in (got_k, got_v):
        t.release()
    c.cache.release()


def test_codes_are_those_of_the_row_quantizer():
    c = Cache([200], 64, 4, 128, fill=False).to_device()
    b = c.batch([200])
    rng = np.random.default_rng(5)
    k = (rng.standard_normal((200, 4, 128)) * np.exp2(rng.integers(-140, 100, (200, 4, 1)))).astype(np.float32)
    k[:, :, ::5] = np.rint(k[:, :, ::5])
    k[3, 1, 7], k[4, 2, 9], k[5, 3, 11] = np.inf, -np.inf, np.nan
    t = HipTensor.from_host(k.reshape(800, 128))
    q, s = t.quantize_i8(0)
    back = q.dequantize(s, 0).cpu().reshape(200, 4, 128)
    kk = HipTensor.from_host(k)
    kv_write_hip(c.cache, b, kk, kk)
    for got in kv_read_hip(c.cache, b):
        assert np.array_equal(got.cpu().view(np.uint32), back.view(np.uint32))


def test_bad_pages_and_starts_touch_nothing_else(guard_bands):
    c = Cache([60, 60, 60, 60], 16, 2, 64, seed=4).to_device()
    c.table[0, 1], c.table[1, 0], c.table[2, 3] = c.num_pages, -5, 0x7fffffff
    c.lengths[3] = 1 << 30                        # counts as the 64 tokens that the table has room for
    b = c.batch([50, 60, 20, 9])
    k, v = normal(1, b.rows, 2, 64), normal(2, b.rows, 2, 64)
    kv_write_hip(c.cache, b, HipTensor.from_host(k), HipTensor.from_host(v))
    assert np.array_equal(c.fetch(), c.written(k, v))
    got = [t.cpu() for t in kv_read_hip(c.cache, b)]
    assert all(np.array_equal(g, w) for g, w in zip(got, c.read(b.rows)))
    q = normal(3, b.rows, 4, 64)
    for causal in (True, False):
        out = attention_i8_hip(c.cache, b, HipTensor.from_host(q), 4, causal=causal).cpu()
        want, far = c.attend(q, 4, 0.125, causal)
        assert (np.abs(out - want) <= far).all()


@pytest.mark.parametrize("starts", [[3, 10, 10, 25], [-5, 8, 12, 400], [0, 0, 0, 0], [40, 40, 40, 40]])
def test_rows_of_no_sequence_are_left_alone(guard_bands, starts):
    c = Cache([50, 20, 33], 32, 2, 64, seed=8).to_device()
    rows = 40
    clamped = np.clip(starts, 0, rows)
    b = c.batch([0, 0, 0], rows=rows, starts=starts)
    c.starts = clamped
    mine = np.zeros(rows, bool)
    mine[clamped[0]:clamped[-1]] = True
    q, k, v = normal(1, rows, 4, 64), normal(2, rows, 2, 64), normal(3, rows, 2, 64)
    kv_write_hip(c.cache, b, HipTensor.from_host(k), HipTensor.from_host(v))
    assert np.array_equal(c.fetch(), c.written(k, v))
    kept = HipTensor.from_host(normal(9, rows, 4 * 64))
    before = kept.cpu()
    hq = HipTensor.from_host(q)
    capi.call("vtl_hip_attention_i8_f32", C.byref(c.cache.handle), C.byref(b.handle), hq.ptr, 256, 4, 0.125, 1, kept.ptr, 256, None, 0)
    got = kept.cpu()
    want, far = c.attend(q, 4, 0.125, True)
    assert np.array_equal(got[~mine], before[~mine])
    assert (np.abs(got.reshape(rows, 4, 64) - want)[mine] <= far[mine]).all()
    capi.call("vtl_hip_memcpy_h2d", kept.ptr, before.ctypes.data, before.nbytes)
    capi.call("vtl_hip_kv_read_f32", C.byref(c.cache.handle), C.byref(b.handle), kept.ptr, 256, None, 0)
    got = kept.cpu()
    want = before.copy()
    want[mine, :128] = c.read(rows)[0].reshape(rows, 128)[mine]
    assert np.array_equal(got, want)


# -- attention --------------------------------------------------------------------------------------

ATTENDS = [  # lengths, rows of each (None: one, without starts), page, heads, kv_heads, dim
    ([1], None, 16, 1, 1, 64), ([300], None, 16, 32, 8, 128), ([64], None, 64, 4, 4, 64), ([65, 63, 0, 1, 128, 2], None, 32, 8, 2, 128),
    ([1000, 17, 0, 333, 4000], None, 64, 10, 2, 80), ([777, 5], None, 128, 16, 1, 256), ([50, 1200], None, 16, 40, 1, 64),
    ([2500], None, 48, 7, 7, 33), ([129], None, 16, 3, 1, 1), ([700, 701], None, 16, 128, 2, 96),
    ([5, 200, 90], [5, 5, 5], 16, 16, 16, 64), ([900, 33], [8, 3], 32, 8, 2, 128), ([400, 64, 64], [2, 1, 4], 64, 16, 4, 72),
    ([64], [64], 64, 4, 2, 64), ([300], [300], 16, 8, 2, 128), ([1777, 1000, 201], [201, 90, 201], 32, 20, 4, 80),
    ([700], [130], 128, 6, 1, 256), ([257, 31], [257, 31], 16, 3, 3, 96), ([129, 500, 0, 64], [40, 33, 17, 65], 16, 4, 2, 128),
    ([1500, 1500], [77, 77], 64, 12, 12, 64), ([5000], [35], 64, 1, 1, 64), ([4000, 70], [33, 1], 128, 2, 2, 100), ([2600], [20], 64, 1, 1, 256),
    ([3000, 2500], [20, 17], 64, 16, 16, 64), ([3000, 2500], [20, 17], 64, 16, 16, 128), ([8300, 8200], [20, 17], 64, 16, 16, 128),
    (list(range(190, 230)), [18] * 40, 16, 8, 8, 64),
    ([9000], [64], 64, 32, 8, 64), ([3000, 2999, 40], [64, 63, 40], 64, 32, 8, 80), ([4100, 4000], [64, 64], 32, 32, 8, 128),
    ([700] * 5, [512] * 5, 64, 16, 16, 100), ([700, 1, 699, 0, 720], [512, 1, 511, 0, 512], 32, 16, 16, 64), ([1500], [1100], 64, 16, 16, 96),
    ([333], [333], 48, 5, 1, 100), ([20], [65], 16, 2, 2, 16), ([2100], [65], 64, 8, 8, 128)]


@pytest.mark.parametrize("lengths,counts,page,heads,kv_heads,dim", ATTENDS)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
def test_attention(guard_bands, lengths, counts, page, heads, kv_heads, dim, causal):
    c = Cache(lengths, page, kv_heads, dim, seed=heads).to_device()
    scale = dim ** -0.5
    want = None
    for hints in (True, False):
        b = c.batch(counts, hints=hints)
        q = normal(b.rows, b.rows, heads, dim, std=2.0)
        if want is None:
            want, far = c.attend(q, heads, np.float32(scale), causal)
        t = HipTensor.from_host(q)
        out = attention_i8_hip(c.cache, b, t, heads, causal=causal)
        off = np.abs(out.cpu() - want)
        assert (off <= far).all(), (hints, float((off / far).max()), np.argwhere(~(off <= far))[:5])
        out.release()
    c.cache.release()


@pytest.mark.parametrize("scale", [0.0, -0.3, 5.0])
@pytest.mark.parametrize("counts", [None, [40, 40]])
def test_scale(scale, counts):
    c = Cache([200, 90], 16, 2, 64, seed=1).to_device()
    b = c.batch(counts)
    q = normal(4, b.rows, 4, 64)
    want, far = c.attend(q, 4, np.float32(scale), True)
    out = attention_i8_hip(c.cache, b, HipTensor.from_host(q), 4, scale=scale).cpu()
    assert (np.abs(out - want) <= far).all()


@pytest.mark.parametrize("counts", [None, [70, 70]])
def test_queries_and_scales_of_every_size(counts):
    """Rows of queries from 2^-120 to 2^40, keys' scales against them, and values' scales over forty powers of two."""
    c = Cache([300, 150], 32, 2, 128, seed=2)
    _, _, ks, vs = c.parts()
    rng = np.random.default_rng(3)
    b_rows = 2 if counts is None else 140
    q = normal(6, b_rows, 4, 128) * np.exp2(rng.integers(-30, -2, (b_rows, 4, 1))).astype(np.float32)
    tiny = slice(0, b_rows, 2)
    q[tiny] *= np.float32(2.0 ** -90)
    for page in c.table[0]:
        vs[page] *= np.exp2(rng.integers(-20, 20, vs[page].shape)).astype(np.float32)
    c.to_device()
    b = c.batch(counts)
    want, far = c.attend(q, 4, np.float32(1.0), True)
    out = attention_i8_hip(c.cache, b, HipTensor.from_host(q), 4, scale=1.0).cpu()
    assert np.isfinite(out).all() and (np.abs(out - want) <= far).all()


@pytest.mark.parametrize("counts", [None, [60]])
def test_far_maxima(counts):
    """Scores in the hundreds, rising and falling along the sequence: the running maximum moves, weights underflow."""
    c = Cache([500], 16, 1, 64, seed=5)
    kc, _, ks, _ = c.parts()
    for j in range(500):
        page, slot = c.place(0, j)
        ks[page, :, slot] *= np.float32(abs(j - 250) / 40 + 0.1)
    c.to_device()
    b = c.batch(counts)
    q = normal(7, b.rows, 8, 64, std=6.0)
    want, far = c.attend(q, 8, np.float32(1.0), True)
    out = attention_i8_hip(c.cache, b, HipTensor.from_host(q), 8, scale=1.0).cpu()
    assert (np.abs(out - want) <= far).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("counts", [None, [90]])
def test_bad_numbers_stay_where_they_are_seen(bad, counts):
    """A token that is no number spoils the rows that see it and no other; a query that is none spoils its own row."""
    c = Cache([200], 16, 2, 64, seed=6)
    _, _, ks, vs = c.parts()
    for token, scales in ((150, ks), (170, vs)):
        page, slot = c.place(0, token)
        scales[page, 0 if scales is ks else 1, slot] = bad
    kc, vc, _, _ = c.parts()
    page, slot = c.place(0, 150)
    kc[page, 0, :, slot] = 0                # as the cache has such a token: codes 0 and an infinite scale
    page, slot = c.place(0, 170)
    vc[page, 1, slot // 16, :, slot % 16] = 0
    c.to_device()
    b = c.batch(counts)
    first = 200 - b.rows if counts else 199
    q = normal(8, b.rows, 4, 64)
    if counts:
        q[5, 3, 7] = bad
    out = attention_i8_hip(c.cache, b, HipTensor.from_host(q), 4).cpu()
    position = first + np.arange(b.rows)
    spoiled = np.zeros((b.rows, 4), bool)
    spoiled[position >= 150, :2] = True
    spoiled[position >= 170, 2:] = True
    if counts:
        spoiled[5, 3] = True
    want, far = c.attend(q, 4, np.float32(0.125), True)
    assert np.isnan(out[spoiled]).all()
    fine = ~spoiled
    assert np.isfinite(out[fine]).all() and (np.abs(out - want)[fine] <= far[fine]).all()


def test_many_pages_past_32_bits():
    """Pages whose bytes lie past 2^32."""
    pages, page, heads, dim = 9000, 128, 16, 128       # 4.9 GB
    from vtl_amd import HipKVCache
    cache = HipKVCache(pages, page, heads, dim)
    assert cache.pages.size > 1 << 32
    table = np.array([[pages - 1, 0, pages - 3], [4, pages - 2, 8990]], np.int32)
    dev = HipTensor.from_host
    lengths, starts = np.array([300, 384], np.int32), np.array([0, 300, 684], np.int32)
    b = HipKVBatch(dev(table), dev(lengths), dev(starts), 684, 384, 384)
    k, v = normal(1, 684, heads, dim), normal(2, 684, heads, dim)
    kv_write_hip(cache, b, dev(k), dev(v))
    got_k, got_v = (t.cpu() for t in kv_read_hip(cache, b))
    for got, x in ((got_k, k), (got_v, v)):
        codes, scale = quantize(x)
        assert np.array_equal(got, codes.astype(np.float32) * scale[..., None])
    one = HipKVBatch(dev(table), dev(lengths), None, None, 1, 384)
    q = normal(3, 2, heads, dim)
    out = attention_i8_hip(cache, one, dev(q), heads).cpu()
    for i, (lo, hi) in enumerate(((0, 300), (300, 684))):
        s = np.einsum("hd,jhd->hj", q[i].astype(np.float64), got_k[lo:hi].astype(np.float64)) * dim ** -0.5
        w = np.exp(s - s.max(1, keepdims=True))
        want = np.einsum("hj,jhd->hd", w / w.sum(1, keepdims=True), got_v[lo:hi].astype(np.float64))
        # as Cache.attend has it, with sums of |q k| below 128 and scores below 8
        assert np.abs(out[i] - want).max() <= 4 * (2 * 128 * dim ** -0.5 * (2.0 ** -21 + dim * 2.0 ** -24) + 2.0 ** -19)
    cache.release()


@pytest.fixture
def stream():
    hiprt = C.CDLL("libamdhip64.so")
    st = C.c_void_p()
    assert hiprt.hipStreamCreate(C.byref(st)) == 0
    capi.call("vtl_hip_set_stream", st)
    yield st, hiprt
    capi.call("vtl_hip_sync")
    capi.call("vtl_hip_set_stream", None)
    hiprt.hipStreamDestroy(st)


def test_same_results_twice_and_on_a_stream(stream):
    c = Cache([900, 40, 0, 2000], 32, 4, 128, seed=11).to_device()
    for counts in (None, [30, 40, 3, 200]):
        b = c.batch(counts)
        t = HipTensor.from_host(normal(12, b.rows, 16, 128))
        got = []
        for st in (None, None, stream[0], stream[0]):
            capi.call("vtl_hip_sync")
            capi.call("vtl_hip_set_stream", st)
            got.append(attention_i8_hip(c.cache, b, t, 16).cpu().view(np.uint32))
        assert all(np.array_equal(got[0], g) for g in got[1:])


@pytest.mark.parametrize("counts", [None, [4, 4, 4], [20, 20, 20]])
def test_recorded_into_a_graph(stream, counts):
    """Write and attention recorded once; between the replays the lengths and the new tokens change on the device, and the program
    makes calls of its own."""
    st, hiprt = stream
    heads, kv_heads, dim, n = 8, 2, 128, 3
    most = [1400, 900, 200]
    c = Cache(most, 32, kv_heads, dim, seed=14)
    rows = 1 if counts is None else counts[0]
    c.to_device()
    b = c.batch(counts)
    first = [1000, 500, 10]
    c.lengths[:] = first
    qkv = HipTensor.empty([n * rows, (heads + 2 * kv_heads) * dim], np.float32)
    out = HipTensor.empty([n * rows, heads * dim], np.float32)
    need = capi.lib().vtl_hip_attention_i8_workspace(C.byref(c.cache.handle), C.byref(b.handle), heads)
    ws = HipStorage.empty(max(need, 16), np.uint8)

    def enqueue():
        kv_write_hip(c.cache, b, qkv, qkv, k_first=heads * dim, v_first=(heads + kv_heads) * dim)
        capi.call("vtl_hip_attention_i8_f32", C.byref(c.cache.handle), C.byref(b.handle), qkv.ptr, qkv.shape[1], heads, dim ** -0.5, 1,
                  out.ptr, heads * dim, ws.ptr, ws.size)

    def upload():
        x = normal(int(c.lengths[0]), n * rows, (heads + 2 * kv_heads) * dim)
        capi.call("vtl_hip_memcpy_h2d", qkv.ptr, x.ctypes.data, x.nbytes)
        capi.call("vtl_hip_memcpy_h2d", b.lengths.ptr, c.lengths.ctypes.data, c.lengths.nbytes)
        x = x.reshape(n * rows, heads + 2 * kv_heads, dim)
        return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]

    def check(q):
        want, far = c.attend(q, heads, np.float32(dim ** -0.5), True)
        assert (np.abs(out.cpu().reshape(want.shape) - want) <= far).all()

    q, k, v = upload()
    enqueue()
    c.written(k, v)
    check(q)
    graph, run = C.c_void_p(), C.c_void_p()
    assert hiprt.hipStreamBeginCapture(st, 0) == 0
    enqueue()
    assert hiprt.hipStreamEndCapture(st, C.byref(graph)) == 0
    assert hiprt.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    try:
        for i in range(4):
            c.lengths += rows
            q, k, v = upload()
            assert hiprt.hipGraphLaunch(run, st) == 0
            capi.call("vtl_hip_sync")
            assert np.array_equal(c.fetch(), c.written(k, v))
            check(q)
            replayed = out.cpu()
            enqueue()                                  # the program's own, and without the caller's workspace
            assert np.array_equal(out.cpu(), replayed)
            t = HipTensor.from_host(np.ascontiguousarray(q))
            check_own = attention_i8_hip(c.cache, b, t, heads).cpu()
            assert np.array_equal(check_own.reshape(replayed.shape), replayed)
    finally:
        hiprt.hipGraphExecDestroy(run)
        hiprt.hipGraphDestroy(graph)


def test_workspace_of_the_callers():
    c = Cache([3000, 50], 64, 2, 128, seed=13).to_device()
    b = c.batch(None)
    need = capi.lib().vtl_hip_attention_i8_workspace(C.byref(c.cache.handle), C.byref(b.handle), 8)
    t = HipTensor.from_host(normal(1, 2, 8, 128))
    want = attention_i8_hip(c.cache, b, t, 8).cpu()
    ws = HipStorage.empty(max(need, 256), np.uint8)
    assert np.array_equal(attention_i8_hip(c.cache, b, t, 8, workspace=ws).cpu(), want)
    if need > 16:
        with pytest.raises(capi.VtlHipError):
            attention_i8_hip(c.cache, b, t, 8, workspace=HipStorage.empty(need - 16, np.uint8))


@pytest.mark.parametrize("lengths,counts,heads,kv_heads,dim", [([40, 900], None, 200, 1, 32), ([90], [2], 200, 1, 64), ([65], [3], 1000, 2, 16),
                                                              ([400], None, 129, 1, 256)])
def test_heads_that_share_keys(lengths, counts, heads, kv_heads, dim):
    """More query heads on one key/value head than a tile has rows: a token's rows are in several tiles."""
    test_attention(None, lengths, counts, 16, heads, kv_heads, dim, True)


@pytest.mark.parametrize("counts", [1, 3, 9])
def test_many_sequences(counts):
    """More sequences than a wave has lanes, among them empty ones and ones with no rows."""
    rng = np.random.default_rng(counts)
    lengths = np.where(rng.random(150) < 0.2, 0, rng.integers(1, 150, 150))
    each = None if counts == 1 else rng.integers(0, counts + 1, 150)
    c = Cache(lengths, 16, 2, 64, seed=17, fill=False)
    _, _, ks, vs = c.parts()
    ks[:], vs[:] = rng.uniform(0.01, 0.05, ks.shape), rng.uniform(0.01, 0.05, vs.shape)      # codes are any
    c.to_device()
    b = c.batch(each)
    q = normal(18, b.rows, 8, 64)
    want, far = c.attend(q, 8, np.float32(0.125), True)
    out = attention_i8_hip(c.cache, b, HipTensor.from_host(q), 8).cpu()
    assert (np.abs(out - want) <= far).all()


@pytest.mark.parametrize("counts,most_rows,most_length", [([50, 7, 300], 1, 10), ([50, 7, 300], 40, 64), ([3, 1, 2], 1, 1), ([600, 0, 1], 33, 100)])
@pytest.mark.parametrize("dim", [64, 200])
def test_more_than_the_host_knows(counts, most_rows, most_length, dim):
    c = Cache([700, 90, 300], 32, 2, dim, seed=19).to_device()
    b = c.batch(counts)
    b.handle.most_rows, b.handle.most_length = most_rows, most_length
    q = normal(20, b.rows, 4, dim)
    want, far = c.attend(q, 4, np.float32(dim ** -0.5), True)
    out = attention_i8_hip(c.cache, b, HipTensor.from_host(q), 4).cpu()
    assert (np.abs(out - want) <= far).all()


@pytest.mark.parametrize("counts", [[3, 2], [70, 40]])
@pytest.mark.parametrize("dim", [64, 80, 33])
@pytest.mark.parametrize("first", [0, 1, 4])
def test_columns_of_wider_rows(counts, dim, first):
    """q and the result in rows that are wider than they, from any column on."""
    c = Cache([300, 90], 16, 2, dim, seed=22).to_device()
    b = c.batch(counts)
    q = normal(23, b.rows, 4, dim)
    columns = 4 * dim + 7
    wide = normal(24, b.rows, columns)
    wide[:, first:first + 4 * dim] = q.reshape(b.rows, -1)
    kept = normal(25, b.rows, columns + 2)
    want, far = c.attend(q, 4, np.float32(0.125), True)
    hq, ho = HipTensor.from_host(wide), HipTensor.from_host(kept)
    capi.call("vtl_hip_attention_i8_f32", C.byref(c.cache.handle), C.byref(b.handle), hq.ptr + 4 * first, columns, 4, 0.125, 1, ho.ptr + 4 * first,
              columns + 2, None, 0)
    got = ho.cpu()
    mine = np.zeros(columns + 2, bool)
    mine[first:first + 4 * dim] = True
    assert np.array_equal(got[:, ~mine], kept[:, ~mine])
    assert (np.abs(got[:, mine].reshape(want.shape) - want) <= far).all()


@pytest.mark.parametrize("counts", [[5, 4, 3], [90, 70, 40]])
def test_starts_that_descend(guard_bands, counts):
    """What such rows get is undefined, but nothing else is touched, and the next call finds everything as it was."""
    c = Cache([900, 300, 500], 16, 2, 64, seed=26).to_device()
    good = c.batch(counts)
    rows = good.rows
    q = HipTensor.from_host(normal(27, rows, 8, 64))
    want = attention_i8_hip(c.cache, good, q, 8).cpu()
    for starts in ([rows, 0, rows, 2], [2, rows, 1, rows], [rows, rows - 1, 1, 0], [0, -3, rows + 9, 0]):
        bad = HipKVBatch(good.page_table, good.lengths, HipTensor.from_host(np.array(starts, np.int32)), rows)
        for causal in (True, False):
            attention_i8_hip(c.cache, bad, q, 8, causal=causal).release()
        k, v = kv_read_hip(c.cache, bad)
        k.release()
        v.release()
        assert np.array_equal(c.fetch(), c.host)
        assert np.array_equal(attention_i8_hip(c.cache, good, q, 8).cpu(), want)


@pytest.mark.parametrize("counts", [None, [33, 40, 2]])
def test_two_streams_at_once(stream, counts):
    """Calls on two streams, none waited for, each with a workspace of its own."""
    st, hiprt = stream
    c = Cache([3000, 700, 150], 64, 2, 128, seed=28).to_device()
    b = c.batch(counts)
    need = capi.lib().vtl_hip_attention_i8_workspace(C.byref(c.cache.handle), C.byref(b.handle), 16)
    q = [HipTensor.from_host(normal(29 + i, b.rows, 16, 128)) for i in range(2)]
    want = [attention_i8_hip(c.cache, b, t, 16).cpu() for t in q]
    ws = [HipStorage.empty(max(need, 16), np.uint8) for _ in q]
    other = C.c_void_p()
    assert hiprt.hipStreamCreate(C.byref(other)) == 0
    out = [[HipTensor.empty([b.rows, 16, 128], np.float32) for _ in range(8)] for _ in q]
    try:
        capi.call("vtl_hip_set_stream", other)
        capi.call("vtl_hip_sync")
        for turn in range(8):
            for i, s in enumerate((st, other)):
                capi.call("vtl_hip_set_stream", s)
                capi.call("vtl_hip_attention_i8_f32", C.byref(c.cache.handle), C.byref(b.handle), q[i].ptr, 16 * 128, 16, 128 ** -0.5, 1,
                          out[i][turn].ptr, 16 * 128, ws[i].ptr, ws[i].size)
        for s in (other, st):
            capi.call("vtl_hip_set_stream", s)
            capi.call("vtl_hip_sync")
        for i in range(2):
            assert all(np.array_equal(t.cpu(), want[i]) for t in out[i])
    finally:
        capi.call("vtl_hip_set_stream", st)
        hiprt.hipStreamDestroy(other)


# -- as a decoder uses them ------------------------------------------------------------------------------

def test_prompt_in_chunks_then_tokens():
    """Projection, write, attention, output projection: a prompt at once, the same in chunks, and token by token, of two sequences.
    Every way leaves the same cache; what comes out differs only by the order of f32 sums."""
    heads, kv_heads, dim, page, width = 8, 2, 64, 16, 256
    rng = np.random.default_rng(21)
    qkv = QuantLinearLayer((rng.standard_normal(((heads + 2 * kv_heads) * dim, width)) * 0.05).astype(np.float32), requires_grad=False)
    last = QuantLinearLayer((rng.standard_normal((width, heads * dim)) * 0.05).astype(np.float32), requires_grad=False)
    lengths = [70, 45]
    x = [normal(30 + i, n, width) for i, n in enumerate(lengths)]

    def step(c, at, counts):
        c.lengths = np.asarray(at, np.int32)
        b = c.batch(counts)
        rows = HipTensor.from_host(np.concatenate([x[i][at[i] - n:at[i]] for i, n in enumerate(counts)]))
        p = qkv.forward_device(rows)
        kv_write_hip(c.cache, b, p, p, k_first=heads * dim, v_first=(heads + kv_heads) * dim)
        a = attention_i8_hip(c.cache, b, p, heads)
        a.shape = [b.rows, heads * dim]
        y = last.forward_device(a)
        return a.cpu(), y.cpu(), p.cpu()

    def new():
        c = Cache(lengths, page, kv_heads, dim, seed=2, fill=False)
        return c.to_device()

    whole = new()
    a, y, p = step(whole, lengths, lengths)
    pages = whole.fetch()
    assert np.array_equal(pages, whole.written(p[:, heads * dim:(heads + kv_heads) * dim].reshape(-1, kv_heads, dim),
                                               p[:, (heads + kv_heads) * dim:].reshape(-1, kv_heads, dim)))
    want, far = whole.attend(p[:, :heads * dim].reshape(-1, heads, dim), heads, np.float32(dim ** -0.5), True)
    assert (np.abs(a.reshape(want.shape) - want) <= far).all()
    parted = new()
    done, got = [0, 0], [[], []]
    for n in ([33, 20], [20, 0], [1, 1], [1, 1], [5, 7], [10, 16]):
        done = [d + k for d, k in zip(done, n)]
        part, _, _ = step(parted, done, n)
        got[0].append(part[:n[0]])
        got[1].append(part[n[0]:])
    assert done == lengths
    assert np.array_equal(parted.fetch(), pages)
    assert (np.abs(np.concatenate(got[0] + got[1]).reshape(want.shape) - want) <= far).all()
    assert y.shape == (115, width) and np.isfinite(y).all()
    qkv.release()
    last.release()
