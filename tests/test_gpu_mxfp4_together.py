"""The calls on microscaled 4-bit rows behind each other as a model makes them: a projection, a layer of experts, an output layer and codes of it, eagerly, on
several streams, and recorded into graphs, with memory at any float's address."""
import ctypes as C

import numpy as np
import pytest

import mx_reference as mx
from vtl_amd import HipMoE, HipMxfp4, capi, linear_f32_mxfp4_hip, moe_mxfp4_hip
from vtl_amd.storage import HipStorage
from vtl_amd.tensor import HipTensor

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]
dev = HipTensor.from_host


def normal(seed, *shape, std=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * std).astype(np.float32)


class Model:
    """x -> a = projection(x) -> b = experts(a) -> y = relu(output(b)) -> codes of y."""

    def __init__(self, dim, experts, hidden, top, out, seed=0):
        self.dim, self.out, self.top = dim, out, top
        weights = [normal(seed + i, rows, cols, std=cols ** -0.5) for i, (rows, cols) in
                   enumerate(((dim, dim), (experts * 2 * hidden, dim), (experts * dim, hidden), (out, dim)))]
        self.values = [mx.decode(*mx.encode(w), w.shape[1]) for w in weights]
        self.q = [dev(w).quantize_mxfp4() for w in weights]
        self.router, self.bias = normal(seed + 5, experts, dim, std=dim ** -0.5), normal(seed + 6, out)
        self.layer = HipMoE(dev(self.router), self.q[1], self.q[2], top)
        self.device_bias = dev(self.bias)
        self.shapes = (experts, 2 * hidden, dim), (experts, dim, hidden)


class Run:
    """Buffers for so many tokens, with workspaces of their own."""

    def __init__(self, m, tokens, own=True):
        self.m, self.tokens = m, tokens
        self.x, self.a, self.b = (HipTensor.empty([tokens, m.dim], np.float32) for _ in range(3))
        self.y = HipTensor.empty([tokens, m.out], np.float32)
        self.codes = HipMxfp4.empty(tokens, m.out)
        L = capi.lib()
        sizes = (L.vtl_hip_linear_f32_mxfp4_workspace(tokens, m.dim, m.dim), m.layer.workspace(tokens), L.vtl_hip_linear_f32_mxfp4_workspace(tokens, m.out, m.dim))
        self.ws = [HipStorage.empty(max(16, n), np.uint8) if own else None for n in sizes]

    def enqueue(self):
        m, t, ws = self.m, self.tokens, [(w.ptr, w.size) if w else (None, 0) for w in self.ws]
        proj, out = m.q[0], m.q[3]
        capi.call("vtl_hip_linear_f32_mxfp4", self.x.ptr, proj.codes.ptr, proj.scales.ptr, None, self.a.ptr, t, m.dim, m.dim, 0, *ws[0])
        capi.call("vtl_hip_moe_mxfp4_f32", C.byref(m.layer.handle), self.a.ptr, self.b.ptr, t, *ws[1])
        capi.call("vtl_hip_linear_f32_mxfp4", self.b.ptr, out.codes.ptr, out.scales.ptr, m.device_bias.ptr, self.y.ptr, t, m.out, m.dim, 1, *ws[2])
        capi.call("vtl_hip_quantize_f32_mxfp4", self.y.ptr, m.out, t, m.out, self.codes.codes.ptr, self.codes.scales.ptr)

    def set(self, x):
        """New input, and nothing of an earlier call left."""
        capi.call("vtl_hip_sync")
        for t in [self.a, self.b, self.y, self.codes.codes, self.codes.scales] + [w for w in self.ws if w]:
            n = t.size * 4 if isinstance(t, HipTensor) else t.size
            noise = np.full(n, 0xff, np.uint8)
            capi.call("vtl_hip_memcpy_h2d", t.ptr, noise.ctypes.data, n)
        capi.call("vtl_hip_memcpy_h2d", self.x.ptr, x.ctypes.data, x.nbytes)
        self.input = x

    def bits(self):
        return [t.cpu().view(np.uint32) for t in (self.a, self.b, self.y)] + [self.codes.codes.cpu(), self.codes.scales.cpu()]

    def check(self):
        m, (a, b, y) = self.m, (t.cpu() for t in (self.a, self.b, self.y))
        def near(got, want, far):
            assert (np.abs(got - want) <= far).all(), float((np.abs(got - want) / far).max())
        near(a, *mx.linear(mx.decode(*mx.encode(self.input), m.dim), m.values[0], None, False))
        near(b, *mx.experts(a, m.router, m.values[1].reshape(m.shapes[0]), m.values[2].reshape(m.shapes[1]), m.top, True))
        near(y, *mx.linear(mx.decode(*mx.encode(b), m.dim), m.values[3], m.bias, True))
        codes, scales = mx.encode(y)
        assert np.array_equal(self.codes.codes.cpu().reshape(codes.shape), codes) and np.array_equal(self.codes.scales.cpu().reshape(scales.shape), scales)


MODELS = {"small": (320, 12, 96, 3, 700), "many": (96, 64, 1030, 6, 520)}
_models = {}


def model(name):
    if name not in _models:
        _models[name] = Model(*MODELS[name])
    return _models[name]


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


@pytest.mark.parametrize("name", MODELS)
@pytest.mark.parametrize("tokens", [1, 3, 8, 20, 64])
def test_behind_each_other(guard_bands, name, tokens):
    m = Model(*MODELS[name])
    run = Run(m, tokens)
    run.set(normal(tokens, tokens, m.dim))
    run.enqueue()
    run.check()
    first = run.bits()
    library = Run(m, tokens, own=False)
    library.set(run.input)
    library.enqueue()
    assert all(np.array_equal(p, q) for p, q in zip(first, library.bits()))


@pytest.mark.parametrize("name,tokens", [("small", 1), ("small", 12), ("small", 64), ("many", 2), ("many", 30)])
def test_two_graphs_and_calls_between_them(hiprt, name, tokens):
    """Two recordings of different sizes with workspaces of their own, replayed on two streams at once, with the program's own calls between the replays."""
    m = model(name)
    runs = [Run(m, tokens), Run(m, tokens + 5 if tokens + 5 <= 64 else tokens - 3)]
    own = [Run(m, r.tokens, own=False) for r in runs]
    streams = [new_stream(hiprt) for _ in runs]
    execs, graphs = [], []
    for r, st in zip(runs, streams):
        r.set(normal(1, r.tokens, m.dim))
        capi.call("vtl_hip_set_stream", st)
        r.enqueue()                 # not the first call of a kernel while recording
        capi.call("vtl_hip_sync")
        graph, run = C.c_void_p(), C.c_void_p()
        assert hiprt.hipStreamBeginCapture(st, 0) == 0
        r.enqueue()
        assert hiprt.hipStreamEndCapture(st, C.byref(graph)) == 0
        assert hiprt.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
        graphs.append(graph)
        execs.append(run)
    try:
        for i in range(4):
            want = []
            for r, o in zip(runs, own):
                x = normal(10 + i, r.tokens, m.dim, std=float(i + 1))
                r.set(x)
                o.set(x)
                capi.call("vtl_hip_set_stream", None)
                o.enqueue()
                capi.call("vtl_hip_sync")
                want.append(o.bits())
            for run, st in zip(execs, streams):
                assert hiprt.hipGraphLaunch(run, st) == 0
            for st in streams:
                assert hiprt.hipStreamSynchronize(st) == 0
            for r, w in zip(runs, want):
                assert all(np.array_equal(p, q) for p, q in zip(r.bits(), w)), (i, r.tokens)
            runs[i % 2].check()
    finally:
        capi.call("vtl_hip_sync")
        for run, graph in zip(execs, graphs):
            hiprt.hipGraphExecDestroy(run)
            hiprt.hipGraphDestroy(graph)


def test_two_streams_at_once(hiprt):
    m = model("many")
    runs, streams = [Run(m, t) for t in (7, 40)], [new_stream(hiprt) for _ in range(2)]
    want = []
    for r in runs:
        r.set(normal(r.tokens, r.tokens, m.dim))
        r.enqueue()
        capi.call("vtl_hip_sync")
        want.append(r.bits())
        r.set(r.input)
    for _ in range(3):
        for r, st in zip(runs, streams):
            capi.call("vtl_hip_set_stream", st)
            r.enqueue()
    for st in streams:
        assert hiprt.hipStreamSynchronize(st) == 0
    capi.call("vtl_hip_set_stream", None)
    for r, w in zip(runs, want):
        assert all(np.array_equal(p, q) for p, q in zip(r.bits(), w))


def shifted(values, by=1):
    """A device buffer in which `values` begin `by` floats behind an aligned address."""
    held = dev(np.concatenate([np.full(by, np.nan, np.float32), values.ravel(), np.full(8, np.nan, np.float32)]))
    return held, held.ptr + 4 * by


@pytest.mark.parametrize("by", [1, 2])
@pytest.mark.parametrize("tokens", [1, 4, 7, 13, 40])
def test_rows_at_any_float(tokens, by):
    m = model("small")
    x = normal(tokens, tokens, m.dim)
    held_x, at_x = shifted(x, by)
    for w, n in ((m.q[0], m.dim), (m.q[3], m.out)):
        want = linear_f32_mxfp4_hip(dev(x), w).cpu()
        held_y, at_y = shifted(np.zeros((tokens, n), np.float32), by)
        capi.call("vtl_hip_linear_f32_mxfp4", at_x, w.codes.ptr, w.scales.ptr, None, at_y, tokens, n, m.dim, 0, None, 0)
        got = held_y.cpu()
        assert np.array_equal(got[by:by + want.size], want.ravel()) and np.isnan(got[:by]).all() and np.isnan(got[by + want.size:]).all()
    want = moe_mxfp4_hip(m.layer, dev(x)).cpu()
    held_y, at_y = shifted(np.zeros_like(x), by)
    capi.call("vtl_hip_moe_mxfp4_f32", C.byref(m.layer.handle), at_x, at_y, tokens, None, 0)
    got = held_y.cpu()
    assert np.array_equal(got[by:by + want.size], want.ravel()) and np.isnan(got[:by]).all() and np.isnan(got[by + want.size:]).all()
    codes = HipMxfp4.empty(tokens, m.dim)
    capi.call("vtl_hip_quantize_f32_mxfp4", at_x, m.dim, tokens, m.dim, codes.codes.ptr, codes.scales.ptr)
    held_y, at_y = shifted(np.zeros_like(x), by)
    capi.call("vtl_hip_dequantize_mxfp4_f32", codes.codes.ptr, codes.scales.ptr, tokens, m.dim, at_y, m.dim)
    got, want = held_y.cpu(), mx.decode(*mx.encode(x), m.dim).astype(np.float32)
    assert np.array_equal(got[by:by + want.size], want.ravel()) and np.isnan(got[:by]).all() and np.isnan(got[by + want.size:]).all()


@pytest.mark.parametrize("M,N", [(1, 5), (6, 300), (12, 70), (16, 4200), (40, 64), (256, 512)])
def test_rows_without_values(M, N):
    """K = 0: the bias."""
    b = normal(1, N)
    for relu in (0, 1):
        y, db = HipTensor.empty([M, N], np.float32), dev(b)
        want = np.broadcast_to(np.where(b < 0, 0, b) if relu else b, (M, N))
        capi.call("vtl_hip_linear_mxfp4_f32", None, None, None, None, db.ptr, y.ptr, M, N, 0, relu, None, 0)
        assert np.array_equal(y.cpu(), want)
        capi.call("vtl_hip_linear_f32_mxfp4", None, None, None, db.ptr, y.ptr, M, N, 0, relu, None, 0)
        assert np.array_equal(y.cpu(), want)


def test_tokens_without_a_finite_score():
    experts, dim, hidden = 6, 64, 32
    gu, dn = dev(normal(1, experts * 2 * hidden, dim)).quantize_mxfp4(), dev(normal(2, experts * dim, hidden)).quantize_mxfp4()
    bias = np.full(experts, -np.inf, np.float32)
    layer = HipMoE(dev(normal(3, experts, dim)), gu, dn, 2, True, dev(bias))
    assert np.isnan(moe_mxfp4_hip(layer, dev(normal(4, 5, dim))).cpu()).all()
    bias[4] = 0.0       # one has a score: the other one that is chosen has no weight
    layer = HipMoE(dev(normal(3, experts, dim)), gu, dn, 2, True, dev(bias))
    one = HipMoE(dev(normal(3, experts, dim)), gu, dn, 1, True, dev(bias))
    x = dev(normal(4, 5, dim))
    assert np.array_equal(moe_mxfp4_hip(layer, x).cpu(), moe_mxfp4_hip(one, x).cpu())
