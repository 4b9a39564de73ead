"""Microscaled 4-bit floating point (MXFP4): rows of codes, linear layers on them, and a layer of experts.

A row is 4-bit codes with a scale, a power of two, for every 32 values; include/vtl_hip.h has the layout and the contract of each call.
`HipTensor.quantize_mxfp4` makes such rows of f32, `HipMxfp4.from_packed` takes those of a checkpoint.  As everywhere in this package the
work is enqueued on the library's stream.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import capi
from .storage import HipParams, HipStorage
from .tensor import HipTensor


class HipMxfp4:
    """A matrix [rows, cols] of MXFP4 values on the device."""

    def __init__(self, codes: HipStorage, scales: HipStorage, rows: int, cols: int):
        padded = padded_row(cols)
        if codes.size != rows * padded // 2 or scales.size != rows * padded // 32:
            raise ValueError(f"HipMxfp4: {codes.size} bytes of codes and {scales.size} of scales for {rows} rows of {cols} values")
        self.codes, self.scales = codes, scales
        self.shape = [rows, cols]

    @staticmethod
    def empty(rows: int, cols: int, params: HipParams | None = None) -> "HipMxfp4":
        padded = padded_row(cols)
        return HipMxfp4(HipStorage.empty(rows * padded // 2, np.uint8, params), HipStorage.empty(rows * padded // 32, np.uint8, params), rows, cols)

    @staticmethod
    def from_packed(codes: np.ndarray, scales: np.ndarray, cols: int, params: HipParams | None = None) -> "HipMxfp4":
        """Codes [rows, ceil(cols / 2)], the even value in the low four bits, and scales [rows, ceil(cols / 32)] of a host."""
        codes, scales = np.asarray(codes), np.asarray(scales)
        if codes.dtype != np.uint8 or scales.dtype != np.uint8:
            raise TypeError(f"from_packed: uint8 codes and scales expected, got {codes.dtype} and {scales.dtype}")
        padded = padded_row(cols)
        if codes.ndim != 2 or codes.shape[1] != -(-cols // 2) or scales.shape != (codes.shape[0], -(-cols // 32)):
            raise ValueError(f"from_packed: codes {codes.shape} and scales {scales.shape} for rows of {cols} values")
        rows = codes.shape[0]
        c, s = np.zeros((rows, padded // 2), np.uint8), np.zeros((rows, padded // 32), np.uint8)
        c[:, :codes.shape[1]], s[:, :scales.shape[1]] = codes, scales
        if cols % 2:
            c[:, cols // 2] &= 15
        return HipMxfp4(HipStorage.from_cpu(c, params), HipStorage.from_cpu(s, params), rows, cols)

    def packed(self):
        """Codes and scales on the host, as from_packed takes them."""
        rows, cols = self.shape
        padded = padded_row(cols)
        codes, scales = HipStorage.cpu_all([self.codes, self.scales])
        return (codes.reshape(rows, padded // 2)[:, :-(-cols // 2)].copy(), scales.reshape(rows, padded // 32)[:, :-(-cols // 32)].copy())

    def dequantize(self) -> HipTensor:
        """`(q &HipMxfp4) dequantize() !&HipTensor[f32]`."""
        rows, cols = self.shape
        x = HipTensor.empty([rows, cols], np.float32, self.codes.params)
        capi.call("vtl_hip_dequantize_mxfp4_f32", self.codes.ptr or None, self.scales.ptr or None, rows, cols, x.ptr or None, cols)
        return x

    def release(self) -> None:
        self.codes.release()
        self.scales.release()


def padded_row(cols: int) -> int:
    """Values that a row of `cols` takes up."""
    padded = capi.lib().vtl_hip_mxfp4_padded_row(cols)
    if not padded:
        raise ValueError(f"MXFP4: no rows of {cols} values")
    return padded


def quantize_mxfp4_hip(x: HipTensor) -> HipMxfp4:
    """`(x &HipTensor[f32]) quantize_mxfp4() !&HipMxfp4`."""
    x._assert(np.float32, what="quantize_mxfp4")
    rows, cols = x.shape
    q = HipMxfp4.empty(rows, cols, x.data.params)
    capi.call("vtl_hip_quantize_f32_mxfp4", x.ptr or None, cols, rows, cols, q.codes.ptr or None, q.scales.ptr or None)
    return q


def _address(t):
    return t.ptr or None if t is not None else None


def _workspace(ws: HipStorage | None):
    return (ws.ptr, ws.size) if ws is not None else (None, 0)


def _bias(bias: HipTensor | None, n: int, what: str):
    if bias is not None:
        bias._assert(np.float32, matrix=False, what=f"{what} bias")
        if bias.size != n:
            raise ValueError(f"{what}: bias has {bias.size} entries, expected {n}")
    return _address(bias)


def _sizes(x, w: HipMxfp4, what: str):
    (m, k), (n, k2) = x.shape, w.shape
    if k != k2:
        raise ValueError(f"{what}: rows of {k} values with weights of {k2}")
    return m, n, k


def linear_mxfp4_workspace(m: int, n: int, k: int, codes: bool = False) -> int:
    """Bytes of the workspace that `linear_f32_mxfp4_hip` takes, or `linear_mxfp4_hip` where codes is set (0: none is needed): for calls that
    may overlap on a device, and for calls recorded into a graph, `HipStorage.empty(bytes, np.uint8)` each."""
    return (capi.lib().vtl_hip_linear_mxfp4_workspace if codes else capi.lib().vtl_hip_linear_f32_mxfp4_workspace)(m, n, k)


def linear_mxfp4_hip(x: HipMxfp4, w: HipMxfp4, bias: HipTensor | None = None, relu: bool = False, workspace: HipStorage | None = None) -> HipTensor:
    """`linear_mxfp4_hip(x, w, bias, relu) !&HipTensor[f32]`: y = x . w^T + bias of codes."""
    m, n, k = _sizes(x, w, "linear_mxfp4_hip")
    b = _bias(bias, n, "linear_mxfp4_hip")
    y = HipTensor.empty([m, n], np.float32, x.codes.params)
    capi.call("vtl_hip_linear_mxfp4_f32", _address(x.codes), _address(x.scales), _address(w.codes), _address(w.scales), b, _address(y), m, n, k, int(relu),
              *_workspace(workspace))
    return y


def linear_f32_mxfp4_hip(x: HipTensor, w: HipMxfp4, bias: HipTensor | None = None, relu: bool = False, workspace: HipStorage | None = None) -> HipTensor:
    """`linear_f32_mxfp4_hip(x, w, bias, relu) !&HipTensor[f32]`: the same of f32 rows, which become codes on the way."""
    x._assert(np.float32, what="linear_f32_mxfp4_hip x")
    m, n, k = _sizes(x, w, "linear_f32_mxfp4_hip")
    b = _bias(bias, n, "linear_f32_mxfp4_hip")
    y = HipTensor.empty([m, n], np.float32, x.data.params)
    capi.call("vtl_hip_linear_f32_mxfp4", _address(x), _address(w.codes), _address(w.scales), b, _address(y), m, n, k, int(relu), *_workspace(workspace))
    return y


class HipMoE:
    """A layer of experts: router [experts, dim] f32, gate_up [experts * 2 * hidden, dim] (for each expert the rows of its gate and then
    those of its up) and down [experts * dim, hidden] as MXFP4 rows; router_bias [experts], gate_up_bias [experts, 2 * hidden], down_bias
    [experts, dim].  A token takes the top_k experts with the largest scores, weighted by the softmax of all scores (renormalize: of the chosen)."""

    def __init__(self, router: HipTensor, gate_up: HipMxfp4, down: HipMxfp4, top_k: int, renormalize: bool = True,
                 router_bias: HipTensor | None = None, gate_up_bias: HipTensor | None = None, down_bias: HipTensor | None = None):
        router._assert(np.float32, what="HipMoE router")
        experts, dim = router.shape
        hidden = down.shape[1]
        if experts < 1 or gate_up.shape != [experts * 2 * hidden, dim] or down.shape != [experts * dim, hidden]:
            raise ValueError(f"HipMoE: router {router.shape}, gate_up {gate_up.shape}, down {down.shape}")
        if not 1 <= top_k <= experts:
            raise ValueError(f"HipMoE: top_k {top_k} of {experts} experts")
        self.experts, self.dim, self.hidden, self.top_k = experts, dim, hidden, top_k
        self.tensors = (router, gate_up, down, router_bias, gate_up_bias, down_bias)     # the handle has their addresses
        self.handle = capi.MoE(experts, top_k, dim, hidden, int(renormalize), router.ptr, _bias(router_bias, experts, "HipMoE router"),
                               gate_up.codes.ptr, gate_up.scales.ptr, _bias(gate_up_bias, experts * 2 * hidden, "HipMoE gate_up"),
                               down.codes.ptr, down.scales.ptr, _bias(down_bias, experts * dim, "HipMoE down"))

    def workspace(self, tokens: int) -> int:
        """Bytes of the workspace of a call of so many tokens, as `linear_mxfp4_workspace`."""
        return capi.lib().vtl_hip_moe_mxfp4_workspace(C.byref(self.handle), tokens)


def moe_mxfp4_hip(layer: HipMoE, x: HipTensor, workspace: HipStorage | None = None) -> HipTensor:
    """`moe_mxfp4_hip(layer, x) !&HipTensor[f32]`: the layer's output for a few tokens [tokens, dim]."""
    x._assert(np.float32, what="moe_mxfp4_hip x")
    tokens, dim = x.shape
    if dim != layer.dim:
        raise ValueError(f"moe_mxfp4_hip: tokens of {dim} values, a layer of {layer.dim}")
    y = HipTensor.empty([tokens, dim], np.float32, x.data.params)
    capi.call("vtl_hip_moe_mxfp4_f32", C.byref(layer.handle), _address(x), _address(y), tokens, *_workspace(workspace))
    return y
