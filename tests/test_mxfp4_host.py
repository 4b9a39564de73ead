"""Microscaled 4-bit rows, their products and layers of experts without a device: sizes, refusals, calls with nothing to do, and what
calls enqueue."""
import ctypes as C
import os
import subprocess
import sys

import pytest

from vtl_amd import capi, linear_mxfp4_workspace

E, U, OK = capi.ERR_INVALID_ARG, capi.ERR_UNSUPPORTED, capi.OK
X, CODES, SCALES, W, WS, Y = (n << 50 for n in range(1, 7))     # addresses that no accepted call of this file reads
HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def quantize(rows=3, cols=40, stride=None, x=X, codes=CODES, scales=SCALES):
    s = cols if stride is None else stride
    return [capi.status("vtl_hip_quantize_f32_mxfp4", x, s, rows, cols, codes, scales),
            capi.status("vtl_hip_dequantize_mxfp4_f32", codes, scales, rows, cols, x, s)]


def linear(M=3, N=5, K=64, x=X, codes=CODES, scales=SCALES, w=W, w_scales=WS, bias=None, y=Y, ws=None, ws_bytes=0):
    return [capi.status("vtl_hip_linear_mxfp4_f32", codes, scales, w, w_scales, bias, y, M, N, K, 0, ws, ws_bytes),
            capi.status("vtl_hip_linear_f32_mxfp4", x, w, w_scales, bias, y, M, N, K, 0, ws, ws_bytes)]


def layer(**changes):
    m = capi.MoE(8, 2, 64, 32, 1, 16, None, CODES, SCALES, None, W, WS, None)
    for name, value in changes.items():
        setattr(m, name, value)
    return m


def experts(m, tokens=3, x=X, y=Y, ws=None, ws_bytes=0):
    return capi.status("vtl_hip_moe_mxfp4_f32", None if m is None else C.byref(m), x, y, tokens, ws, ws_bytes)


@pytest.mark.parametrize("cols,padded", [(1, 256), (256, 256), (257, 512), (1000, 1024), (1 << 24, 1 << 24), ((1 << 24) + 1, 0), (0, 0), (-5, 0), (2 ** 31 - 1, 0)])
def test_padded_rows(cols, padded):
    assert capi.lib().vtl_hip_mxfp4_padded_row(cols) == padded


def test_refused_rows():
    for args in ({"rows": -1}, {"cols": -1}, {"stride": 39}, {"x": None}, {"codes": None}, {"scales": None}, {"codes": CODES + 8}, {"scales": SCALES + 4},
                 {"codes": X}, {"codes": X + 464}, {"scales": X + 472}, {"codes": X - 128}, {"x": SCALES + 16}):
        assert quantize(**args) == [E, E], args
    assert quantize(codes=X + 128 * 1000, rows=1001, stride=1000) == [E, E]      # between rows of x
    for args in ({"cols": (1 << 24) + 1}, {"rows": 1 << 31}, {"rows": 1 << 30, "cols": 600}, {"rows": 1 << 62, "cols": 1}):
        assert quantize(**args) == [U, U], args


def test_no_rows():
    assert quantize(rows=0, x=None, codes=None, scales=None) == [OK, OK]
    assert quantize(cols=0, x=None, codes=None, scales=None) == [OK, OK]


def test_refused_products():
    for args in ({"M": -1}, {"N": -1}, {"K": -1}, {"w": None}, {"w_scales": None}, {"y": None}, {"w": W + 8}, {"w_scales": WS + 4},
                 {"ws": None, "ws_bytes": 8}, {"y": W + 128 * 5 - 4}, {"y": WS}, {"bias": Y + 56}):
        assert linear(**args) == [E, E], args
    for args in ({"codes": None}, {"scales": None}, {"codes": CODES + 8}, {"scales": SCALES + 4}, {"y": CODES + 380}, {"y": SCALES + 16}):
        assert linear(**args)[0] == E, args
    for args in ({"x": None}, {"y": X + 64}, {"x": Y + 56}):
        assert linear(**args)[1] == E, args
    for args in ({"K": (1 << 24) + 1}, {"M": 1 << 30}, {"N": (1 << 27) - 15}, {"M": 1 << 20, "K": 1 << 20}, {"N": 1 << 20, "K": 1 << 20}):
        assert linear(**args) == [U, U], args
    for M, N, K in ((20, 64, 4096), (64, 4096, 14336), (16, 100, 300)):
        for codes in (True, False):
            need = linear_mxfp4_workspace(M, N, K, codes)
            if need:
                assert linear(M, N, K, ws=1 << 48, ws_bytes=need - 1)[0 if codes else 1] == E
                assert linear(M, N, K, ws=(1 << 48) + 8, ws_bytes=need)[0 if codes else 1] == E
    assert linear_mxfp4_workspace(16, 100, 300) > 0


def test_no_products():
    assert linear(M=0, x=None, codes=None, w=None, y=None) == [OK, OK] and linear(N=0, x=None, codes=None, w=None, y=None) == [OK, OK]
    for sizes in ((0, 5, 64), (5, 0, 64), (5, 5, 0), (-1, 5, 64), (5, 5, (1 << 24) + 1)):
        assert linear_mxfp4_workspace(*sizes) == 0 and linear_mxfp4_workspace(*sizes, True) == 0


def test_refused_layers():
    assert experts(None) == E and experts(layer(), tokens=-1) == E and experts(layer(), x=None) == E and experts(layer(), y=None) == E
    for name in ("router", "gate_up", "gate_up_scales", "down", "down_scales"):
        assert experts(layer(**{name: None})) == E, name
    for changes in ({"experts": 0}, {"top_k": 0}, {"top_k": 9}, {"dim": 0}, {"hidden": 0}, {"hidden": -4}, {"gate_up": CODES + 8}, {"gate_up_scales": SCALES + 4},
                    {"down": W + 8}, {"down_scales": WS + 4}):
        assert experts(layer(**changes)) == E, changes
    for changes in ({"experts": 513}, {"experts": 17, "top_k": 17}, {"dim": 65537}, {"hidden": 65537}):
        assert experts(layer(**changes)) == U, changes
    assert experts(layer(), tokens=65) == U
    for y in (X, X + 3 * 256 - 4, 16 + 8 * 256 - 4, CODES, SCALES + 8 * 64 * 8 - 4, W + 8 * 64 * 128 - 4, WS):
        assert experts(layer(), y=y) == E, hex(y)
    for name in ("router_bias", "gate_up_bias", "down_bias"):
        assert experts(layer(**{name: Y + 3 * 256 - 4})) == E, name
    need = capi.lib().vtl_hip_moe_mxfp4_workspace(C.byref(layer()), 3)
    assert need > 0 and experts(layer(), ws=1 << 48, ws_bytes=need - 1) == E and experts(layer(), ws=(1 << 48) + 4, ws_bytes=need) == E
    assert experts(layer(), ws_bytes=4) == E


def test_no_layers():
    assert experts(layer(router=None), tokens=0, x=None, y=None) == OK
    w = capi.lib().vtl_hip_moe_mxfp4_workspace
    assert w(C.byref(layer()), 0) == 0 and w(C.byref(layer()), 65) == 0 and w(C.byref(layer(top_k=0)), 3) == 0 and w(None, 3) == 0


_PRELUDE = r"""
import ctypes as C, re, sys
fake = C.CDLL(sys.argv[2], mode=C.RTLD_GLOBAL)
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/tests"]
import test_mxfp4_host as t
from vtl_amd import capi
fake.fake_set(1, 0, 0, 0)

def launches():
    buf = C.create_string_buffer(1 << 20)
    n = fake.fake_log(buf, C.c_size_t(len(buf)))
    lines = [l.split() for l in buf.raw[:n].decode().splitlines()]
    return [(re.search(r"\d([a-z]\w*?_kernel)", l[4]).group(1), int(l[3]), [int(i) for i in re.findall(r"L[ib](\d+)E", l[4])]) for l in lines if l[0] == "launch"]

def of(status):
    assert status == capi.OK, status
    return launches()
BIG = {"ws": 1 << 48, "ws_bytes": 1 << 45}
"""


@pytest.fixture(scope="module")
def fake_runtime(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("runtime") / "libfake_runtime.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    os.path.join(HERE, "host_runtime", "fake_runtime.cpp"), "-o", out], check=True)
    return out


def _run(fake, program):
    res = subprocess.run([sys.executable, "-c", _PRELUDE + program, ROOT, fake], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert res.returncode == 0 and res.stdout.strip().endswith("done"), res.stdout[-3000:]


def test_launches_of_products(fake_runtime):
    """Up to 16 rows are one launch, f32 rows are made codes in it up to 8 (4 beside large weights); more are a launch of the same kernel or of tiles, and K in ranges is joined by a launch
    of its own."""
    _run(fake_runtime, r"""
for M in range(1, 17):
    for index, name in ((0, "vtl_hip_linear_mxfp4_f32"), (1, "vtl_hip_linear_f32_mxfp4")):
        args = (t.X,) if index else (t.CODES, t.SCALES)
        log = of(capi.status(name, *args, t.W, t.WS, None, t.Y, M, 4096, 4096, 0, BIG["ws"], BIG["ws_bytes"]))
        assert [l[0] for l in log] == ["quantize_mxfp4_kernel"] * (index and M > 8) + ["linear_few_mxfp4_kernel"], (M, log)
        if index:
            log = of(capi.status(name, t.X, t.W, t.WS, None, t.Y, M, 8192, 4096, 0, BIG["ws"], BIG["ws_bytes"]))
            assert [l[0] for l in log] == ["quantize_mxfp4_kernel"] * (M > 4) + ["linear_few_mxfp4_kernel"], (M, log)
            assert (capi.lib().vtl_hip_linear_f32_mxfp4_workspace(M, 8192, 4096) > 0) == (M > 4)
def tile(M, N, K):
    st = capi.status("vtl_hip_linear_mxfp4_f32", t.CODES, t.SCALES, t.W, t.WS, None, t.Y, M, N, K, 0, BIG["ws"], BIG["ws_bytes"])
    return of(st)
tiles = set()
for M in (17, 40, 100, 201, 256, 512, 1024, 4096):
    for N in (64, 1000, 4096, 14336):
        for K in (0, 1, 256, 4096, 11008, 14336):
            log = tile(M, N, K)
            bm, bn = log[0][2][:2]
            if log[0][0] == "linear_few_mxfp4_kernel":
                assert bn == 8 and len(log) == 1 and log[0][1] == -(-N // (16 * bm)) * -(-M // 32), (M, N, K, log)
                tiles.add((32, 16 * bm))
                continue
            tiles.add((bm, bn))
            whole = -(-M // bm) * -(-N // bn)
            assert log[0][0] == "linear_tile_mxfp4_kernel" and log[0][1] % whole == 0, (M, N, K, log)
            splits = log[0][1] // whole
            assert [l[0] for l in log[1:]] == ["linear_join_mxfp4_kernel"] * (splits > 1), (M, N, K, log)
            need = capi.lib().vtl_hip_linear_mxfp4_workspace(M, N, K)
            assert need >= (4 * splits * M * N if splits > 1 else 0) and splits * 4 <= max(4, -(-K // 256)), (M, N, K, splits)
assert tiles == {(32, 16), (32, 32), (64, 64), (128, 96), (128, 128), (256, 128), (256, 256)}, tiles
print("done")
""")


def test_grids_of_very_many_rows(fake_runtime):
    """A grid has less than 2^32 threads in a row."""
    _run(fake_runtime, r"""
most_n, most_m = (1 << 27) - 16, (1 << 30) - 1
for M, N in ((1, most_n), (8, most_n), (16, most_n), (17, most_n), (33, most_n), (300, most_n), (most_m, 1), (most_m, 64), (most_m, 65), (1 << 20, 1 << 20)):
    st = capi.status("vtl_hip_linear_mxfp4_f32", t.CODES, t.SCALES, t.W, t.WS, None, t.Y, M, N, 200, 0, 1 << 60, 1 << 59)
    log = launches()
    if (M, N) == (1 << 20, 1 << 20):
        assert st == capi.ERR_UNSUPPORTED or log
    else:
        assert st == capi.OK, (M, N, st)
    for name, blocks, sizes in log:
        assert blocks * 256 < 1 << 32, (M, N, log)
print("done")
""")


def test_launches_of_layers(fake_runtime):
    """Up to eight tokens without a launch for the plan where hidden values are few, one wave along K where there are enough of them, and a join where the output has fewer rows than compute units."""
    _run(fake_runtime, r"""
def names(tokens, **changes):
    return of(t.experts(t.layer(**changes), tokens, **BIG))
few = names(1, experts=64, top_k=6, dim=2048, hidden=512)
# (six experts of one unit each are less than two for each of 16 waves)
assert [l[0] for l in few] == ["moe_scores_kernel", "moe_gate_up_kernel", "moe_down_kernel"] and few[1][2] == [1, 2, 2, 2, 1, 0], few
assert [l[0] for l in names(1, experts=64, top_k=6, dim=2048, hidden=4096)] == [
    "moe_scores_kernel", "moe_plan_kernel", "moe_gate_up_kernel", "moe_down_kernel", "moe_join_kernel"]      # 768 workgroups of 32 hidden values
assert [l[0] for l in names(1, experts=64, top_k=6, dim=4096, hidden=512)] == ["moe_scores_kernel", "moe_gate_up_kernel", "moe_down_kernel"]
for experts, each in ((128, 2), (129, 4), (256, 4), (257, 8), (512, 8)):
    assert names(1, experts=experts, top_k=6, dim=4096, hidden=512)[1][2] == [1, 2, 2, each, 1, 0], experts
    assert names(64, experts=experts, top_k=1, dim=4096, hidden=32)[1] == ("moe_plan_kernel", 1, [each]), experts
assert names(4, experts=64, top_k=6, dim=4096, hidden=512)[1][2] == [2, 2, 2, 2, 1, 0]
assert names(8, experts=300, top_k=2, dim=4096, hidden=512)[1][2] == [2, 2, 2, 8, 1, 0]
nine = names(9, experts=64, top_k=2, dim=4096, hidden=512)
assert [l[0] for l in nine] == ["moe_scores_kernel", "moe_plan_kernel", "moe_gate_up_kernel", "moe_down_kernel"] and nine[2][2] == [2, 2, 2, 0, 1, 0], nine
many = names(24, experts=128, top_k=8, dim=2048, hidden=1024)
assert [l[0] for l in many] == ["moe_scores_kernel", "moe_plan_kernel", "moe_gate_up_kernel", "moe_down_kernel", "moe_join_kernel"] and many[2][2] == [2, 2, 1, 0, 1, 1] and many[3][2] == [2, 1, 8, 1], many
assert names(24, experts=128, top_k=8, dim=512, hidden=1024)[2][2] == [2, 2, 1, 0, 1, 0]
assert names(2, experts=128, top_k=16, dim=2048, hidden=2048)[2][2] == [2, 2, 1, 0, 1, 1]
# four pairs of an expert and more: waves with twice the weights
dense = names(16, experts=8, top_k=2, dim=4096, hidden=2816)
assert [l[0] for l in dense] == ["moe_scores_kernel", "moe_plan_kernel", "moe_gate_up_kernel", "moe_down_kernel", "moe_join_kernel"], dense
assert dense[2][2] == [4, 1, 1, 0, 2, 0] and dense[3][2] == [4, 2, 4, 0] and dense[3][1] == 2 * 128, dense
assert names(8, experts=8, top_k=4, dim=4096, hidden=64)[1][2] == [2, 2, 2, 2, 1, 0]
# few workgroups: up to eleven passes over 64 pairs beside each other
small = names(64, experts=4, top_k=2, dim=4096, hidden=64)
assert small[2][1:] == (4 * 16 * 11, [2, 2, 2, 0, 1, 0]), small
most = names(64, experts=512, top_k=16, dim=65536, hidden=65536)
assert all(blocks * 512 < 1 << 32 for _, blocks, _ in most), most
print("done")
""")


def test_refusals_of_the_python_mirror(fake_runtime):
    _run(fake_runtime, r"""
import numpy as np
from vtl_amd import *
from vtl_amd.storage import HipStorage
from vtl_amd.tensor import HipTensor
def refused(f, *args, **more):
    try:
        f(*args, **more)
    except (ValueError, TypeError):
        return True
f32 = lambda *shape: HipTensor.empty(shape, np.float32)
w, x = HipMxfp4.empty(5, 300), f32(3, 300)
assert w.codes.size == 5 * 256 and w.scales.size == 5 * 16
assert refused(HipMxfp4, w.codes, w.scales, 5, 600) and refused(HipMxfp4, w.codes, w.scales, 4, 300) and refused(HipMxfp4.empty, 4, 0)
codes, scales = np.zeros((5, 150), np.uint8), np.zeros((5, 10), np.uint8)
assert refused(HipMxfp4.from_packed, codes, scales, 302) and refused(HipMxfp4.from_packed, codes.astype(np.int8), scales, 300)
assert refused(HipMxfp4.from_packed, codes[0], scales, 300) and refused(HipMxfp4.from_packed, codes, scales[:4], 300)
assert refused(HipTensor.empty([3, 300], np.float64).quantize_mxfp4) and refused(f32(300).quantize_mxfp4)
assert linear_f32_mxfp4_hip(x, w).shape == [3, 5] and linear_mxfp4_hip(x.quantize_mxfp4(), w, f32(5)).shape == [3, 5]
assert refused(linear_f32_mxfp4_hip, f32(3, 256), w) and refused(linear_f32_mxfp4_hip, f32(300), w) and refused(linear_f32_mxfp4_hip, x, w, f32(4))
assert refused(linear_mxfp4_hip, HipMxfp4.empty(3, 256), w) and refused(linear_mxfp4_hip, x.quantize_mxfp4(), w, HipTensor.empty([5], np.float64))
parts = lambda hidden=40, dim=64, experts=6: (f32(experts, dim), HipMxfp4.empty(experts * 2 * hidden, dim), HipMxfp4.empty(experts * dim, hidden))
layer = HipMoE(*parts(), 2)
assert moe_mxfp4_hip(layer, f32(7, 64)).shape == [7, 64]
ws = HipStorage.empty(layer.workspace(7), np.uint8)
assert moe_mxfp4_hip(layer, f32(7, 64), ws).shape == [7, 64]
assert refused(moe_mxfp4_hip, layer, f32(7, 60)) and refused(moe_mxfp4_hip, layer, HipTensor.empty([7, 64], np.float64))
for bad in ((f32(6, 60), *parts()[1:]), (parts()[0], HipMxfp4.empty(480, 60), parts()[2]), (parts()[0], HipMxfp4.empty(470, 64), parts()[2]),
            (*parts()[:2], HipMxfp4.empty(6 * 64, 41)), (*parts()[:2], HipMxfp4.empty(5 * 64, 40))):
    assert refused(HipMoE, *bad, 2)
assert refused(HipMoE, *parts(), 0) and refused(HipMoE, *parts(), 7)
assert refused(HipMoE, *parts(), 2, True, f32(5)) and refused(HipMoE, *parts(), 2, True, None, f32(6 * 79)) and refused(HipMoE, *parts(), 2, True, None, None, f32(64))
for tokens, many in ((65, HipMoE(*parts(), 2)), (1, HipMoE(*parts(experts=513, hidden=8), 2))):
    try:
        moe_mxfp4_hip(many, f32(tokens, 64))
        assert False
    except capi.VtlHipError as e:
        assert e.status == capi.ERR_UNSUPPORTED, e
print("done")
""")
