"""A workspace that shares memory with what a call reads or writes is refused, without a device; memory behind the bytes that the call takes is the caller's."""
import ctypes as C

import pytest

import test_mxfp4_host as t
from test_mxfp4_host import fake_runtime  # noqa: F401
from vtl_amd import capi, linear_mxfp4_workspace

E = capi.ERR_INVALID_ARG
WS = 1 << 48        # of a caller; no accepted call of this file is made, so nothing reads it


@pytest.mark.parametrize("M,N,K", [(12, 64, 300), (100, 4096, 14336), (700, 100, 40)])
def test_products(M, N, K):
    for codes in (True, False):
        need = linear_mxfp4_workspace(M, N, K, codes)
        if not need:
            continue
        row = -(-K // 256)
        operands = {"w": N * row * 128, "w_scales": N * row * 8, "bias": 4 * N, "y": 4 * M * N}
        operands |= {"codes": M * row * 128, "scales": M * row * 8} if codes else {"x": 4 * M * K}
        for name, size in operands.items():
            for at in (WS, WS + (need - 1) // 16 * 16, WS + 16 - (size + 15) // 16 * 16):
                assert t.linear(M, N, K, ws=WS, ws_bytes=need, **{name: at})[0 if codes else 1] == E, (name, hex(at))


def test_something_needs_one():
    assert linear_mxfp4_workspace(12, 64, 300) and linear_mxfp4_workspace(100, 4096, 14336, True) and linear_mxfp4_workspace(700, 100, 40)


def test_layers():
    need = capi.lib().vtl_hip_moe_mxfp4_workspace(C.byref(t.layer()), 3)
    sizes = {"router": 8 * 64 * 4, "router_bias": 8 * 4, "gate_up": 8 * 64 * 128, "gate_up_scales": 8 * 64 * 8, "gate_up_bias": 8 * 64 * 4, "down": 8 * 64 * 128,
             "down_scales": 8 * 64 * 8, "down_bias": 8 * 64 * 4}
    for name, size in sizes.items():
        for at in (WS, WS + (need - 1) // 16 * 16, WS + 16 - size):
            assert t.experts(t.layer(**{name: at}), ws=WS, ws_bytes=need) == E, (name, hex(at))
    for at in (WS, WS + need - 4, WS - 3 * 64 * 4 + 4):
        assert t.experts(t.layer(), x=at, ws=WS, ws_bytes=need) == E and t.experts(t.layer(), y=at, ws=WS, ws_bytes=need) == E, hex(at)


def test_memory_behind_it(fake_runtime):
    t._run(fake_runtime, r"""
from vtl_amd import linear_mxfp4_workspace
WS, MUCH = 1 << 48, 1 << 40
for codes in (True, False):
    need = linear_mxfp4_workspace(100, 4096, 14336, codes)
    assert need % 16 == 0
    for name in ("y", "w", "codes" if codes else "x", "bias"):
        assert t.linear(100, 4096, 14336, ws=WS, ws_bytes=MUCH, **{name: WS + need})[0 if codes else 1] == capi.OK, name
need = capi.lib().vtl_hip_moe_mxfp4_workspace(C.byref(t.layer()), 3)
assert t.experts(t.layer(), y=WS + need, ws=WS, ws_bytes=MUCH) == capi.OK and t.experts(t.layer(down=WS + need), ws=WS, ws_bytes=MUCH) == capi.OK
print("done")
""")
