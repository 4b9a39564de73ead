"""Timed cases of microscaled 4-bit floating point: rows into codes and back, linear layers, a layer of experts.

Rows of f32 become e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) with a scale, a power of two, for 32 values each
(`codes`, which reads them back so that the values they stand for can be seen; `values` is the way back alone).
`linear` multiplies rows with such weights: rows that come as codes too, or f32 rows that become codes on the way.
`experts` is a whole mixture-of-experts layer for the tokens of a decode step: router, the chosen experts' two products with
SiLU(gate) * up between them, and the weighted sum; there the rows stay f32.

A matrix [rows, cols] lies in rows padded to a multiple of 256 values: codes uint8 [rows, padded / 2], the even value in
the low four bits, and scales uint8 [rows, padded / 32], a byte b for 2^(b - 127); zeros behind the end.
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False


def listed():
    return [
        # The activations of a few tokens: the smallest call.
        {"name": "codes_8x4096", "op": "codes", "rows": 8, "cols": 4096},
        # Weights of a large layer when a model is loaded; their way back for a layer that multiplies in f32.
        {"name": "codes_14336x4096", "op": "codes", "rows": 14336, "cols": 4096},
        {"name": "values_11008x4096", "op": "values", "rows": 11008, "cols": 4096},
        # Rows that are no whole number of blocks.
        {"name": "codes_1777x1000", "op": "codes", "rows": 1777, "cols": 1000},
        # One token and a small batch of tokens through a large layer, the weights read once.
        {"name": "linear_1x4096x14336", "op": "linear", "given": "f32", "rows": 1, "cols": 4096, "out": 14336, "bias": False, "relu": False},
        {"name": "linear_16x4096x14336", "op": "linear", "given": "f32", "rows": 16, "cols": 4096, "out": 14336, "bias": True, "relu": False},
        # The odd last chunk of a prompt.
        {"name": "linear_201x4096x11008", "op": "linear", "given": "f32", "rows": 201, "cols": 4096, "out": 11008, "bias": True, "relu": True},
        # A prompt, and a large one whose rows come as codes.
        {"name": "linear_4096x4096x4096", "op": "linear", "given": "f32", "rows": 4096, "cols": 4096, "out": 4096, "bias": True, "relu": False},
        {"name": "linear_8192x8192x8192", "op": "linear", "given": "codes", "rows": 8192, "cols": 8192, "out": 8192, "bias": False, "relu": False},
        # One token, a batch of sequences' next tokens, and odd sizes with biases.
        {"name": "experts_1_of_64", "op": "experts", "rows": 1, "dim": 4096, "hidden": 1024, "experts": 64, "top": 6, "renormalize": True, "bias": False},
        {"name": "experts_24_of_128", "op": "experts", "rows": 24, "dim": 2048, "hidden": 1024, "experts": 128, "top": 8, "renormalize": True, "bias": False},
        {"name": "experts_5_of_20_odd", "op": "experts", "rows": 5, "dim": 1000, "hidden": 720, "experts": 20, "top": 3, "renormalize": False, "bias": True},
    ]


def _log_size(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["codes", "values", "linear", "linear", "linear", "experts", "experts"])
    if op in ("codes", "values"):
        cols = _log_size(rng, 16, 16384)
        if rng.random() < 0.5:
            cols = max(64, cols // 64 * 64)
        return {"op": op, "rows": _log_size(rng, 1, min(32768, (1 << 26) // cols)), "cols": cols}
    if op == "linear":
        few = rng.random() < 0.5
        case = {"op": op, "given": rng.choice(["f32", "f32", "codes"]), "rows": _log_size(rng, 1, 40) if few else _log_size(rng, 32, 8192),
                "cols": _log_size(rng, 64, 16384), "out": _log_size(rng, 32, 16384), "bias": rng.random() < 0.5, "relu": rng.random() < 0.3}
        if rng.random() < 0.6:
            case["cols"], case["out"] = case["cols"] // 64 * 64, case["out"] // 32 * 32
        while case["rows"] * case["cols"] * case["out"] > 1 << 38:
            case["rows"] = (case["rows"] + 1) // 2
        return case
    experts = rng.choice([8, 16, 20, 32, 60, 64, 128, 256])
    dim, hidden = _log_size(rng, 256, 6144), _log_size(rng, 128, 4096)
    if rng.random() < 0.7:
        dim, hidden = dim // 32 * 32, hidden // 32 * 32
    while experts * dim * hidden > 1 << 28:
        hidden = (hidden + 1) // 2
    return {"op": op, "rows": _log_size(rng, 1, 64), "dim": dim, "hidden": hidden, "experts": experts,
            "top": rng.randrange(1, 9), "renormalize": rng.random() < 0.6, "bias": rng.random() < 0.3}


# -- the format ------------------------------------------------------------------------------

_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _padded(cols):
    return -(-cols // 256) * 256


def _encode(x):
    """Codes and scales of rows."""
    rows, cols = x.shape
    blocks = torch.nn.functional.pad(x, (0, _padded(cols) - cols)).view(rows, -1, 32)
    top = blocks.abs().amax(-1)
    finite = torch.isfinite(blocks).all(-1)
    byte = ((top.view(torch.int32) >> 23) - 2).clamp(min=0)
    # a power of two times an f32 number: exact, but where the product is far below the smallest code
    v = (blocks * ((254 - byte) << 23).view(torch.float32)[..., None]).abs()
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    v = (torch.round(v / step) * step).clamp(max=6.0)
    code = torch.where(v < 2, v * 2, torch.where(v < 4, v + 2, v * 0.5 + 4)) + 8.0 * torch.signbit(blocks)
    code = torch.where(finite[..., None], code, torch.zeros_like(code)).to(torch.uint8).view(rows, -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), torch.where(finite, byte, 255).to(torch.uint8)


def _decode(codes, scales, cols):
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=codes.device)
    v = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).view(codes.shape[0], -1, 32)
    factor = (scales.int() << 23).view(torch.float32)
    factor = torch.where(scales == 0, torch.full_like(factor, 2.0 ** -127), factor)
    factor = torch.where(scales == 255, torch.full_like(factor, float("nan")), factor)
    return (v * factor[..., None]).view(codes.shape[0], -1)[:, :cols].contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def activations(rows, cols):
        """Rows of tokens, with the few large channels that activations have."""
        x = normal(rows, cols)
        x[:, ::61] *= 8.0
        return x

    def weights(rows, cols):
        codes = torch.empty(rows, _padded(cols) // 2, dtype=torch.uint8, device="cuda")
        scales = torch.empty(rows, _padded(cols) // 32, dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 24) // cols)
        for lo in range(0, rows, step):
            n = min(step, rows - lo)
            codes[lo:lo + n], scales[lo:lo + n] = _encode(normal(n, cols) * cols ** -0.5)
        return codes, scales

    s = {"case": dict(case)}
    if case["op"] == "codes":
        s["x"] = activations(case["rows"], case["cols"])
    elif case["op"] == "values":
        s["w"] = weights(case["rows"], case["cols"])
    elif case["op"] == "linear":
        s["x"] = activations(case["rows"], case["cols"])
        if case["given"] == "codes":
            s["x"] = _encode(s["x"])
        s["w"] = weights(case["out"], case["cols"])
        s["bias"] = normal(case["out"]) * 0.1 if case["bias"] else None
    else:
        experts, dim, hidden = case["experts"], case["dim"], case["hidden"]
        s["x"] = activations(case["rows"], dim)
        s["router"] = normal(experts, dim) * dim ** -0.5
        s["gate_up"] = weights(experts * 2 * hidden, dim)
        s["down"] = weights(experts * dim, hidden)
        if case["bias"]:
            s["router_bias"], s["gate_up_bias"], s["down_bias"] = normal(experts) * 0.1, normal(experts, 2 * hidden) * 0.1, normal(experts, dim) * 0.1
        else:
            s["router_bias"] = s["gate_up_bias"] = s["down_bias"] = None
    return s


# -- the plain forms -----------------------------------------------------------------------

def _plain_linear(s):
    cols = s["case"]["cols"]
    x = _decode(*(s["x"] if s["case"]["given"] == "codes" else _encode(s["x"])), cols)
    y = torch.matmul(x, _decode(*s["w"], cols).T)
    if s["bias"] is not None:
        y = y + s["bias"]
    return torch.where(y < 0, torch.zeros_like(y), y) if s["case"]["relu"] else y


def _plain_experts(s):
    case, x = s["case"], s["x"]
    dim, hidden, top = case["dim"], case["hidden"], case["top"]
    # scores next to each other decide on experts: sums in 64 bits, rounded once
    score = torch.matmul(x.double(), s["router"].double().T).float()
    if s["router_bias"] is not None:
        score = score + s["router_bias"]
    chosen = torch.sort(score, dim=1, descending=True, stable=True)[1][:, :top]
    p = torch.exp(score - score.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    p = torch.zeros_like(p).scatter(1, chosen, torch.gather(p, 1, chosen))
    if case["renormalize"]:
        p = p / p.sum(1, keepdim=True)
    # every expert with all rows, or the experts of one row after the other where that is less
    y = torch.zeros(case["rows"], dim, device="cuda")
    if case["rows"] * top < case["experts"]:
        jobs = [(chosen[t, slot:slot + 1], slice(t, t + 1)) for t in range(case["rows"]) for slot in range(top)]
    else:
        jobs = [(torch.full((1,), e, device="cuda"), slice(None)) for e in range(case["experts"])]
    for e, rows in jobs:
        at = e * 2 * hidden + torch.arange(2 * hidden, device="cuda")
        gu = torch.matmul(x[rows], _decode(s["gate_up"][0][at], s["gate_up"][1][at], dim).T)
        if s["gate_up_bias"] is not None:
            gu = gu + s["gate_up_bias"][e]
        g, u = gu[:, :hidden], gu[:, hidden:]
        h = g / (1 + torch.exp(-g)) * u
        at = e * dim + torch.arange(dim, device="cuda")
        out = torch.matmul(h, _decode(s["down"][0][at], s["down"][1][at], hidden).T)
        if s["down_bias"] is not None:
            out = out + s["down_bias"][e]
        y[rows] += p[rows, e] * out
    return y


# -- the framework's operators ---------------------------------------------------------------

def _at(t):
    return t.data_ptr() if t is not None else None


def _own_codes(s):
    from vtl_amd import capi
    rows, cols = s["x"].shape
    codes = torch.empty(rows, _padded(cols) // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, _padded(cols) // 32, dtype=torch.uint8, device="cuda")
    capi.call("vtl_hip_quantize_f32_mxfp4", _at(s["x"]), cols, rows, cols, _at(codes), _at(scales))
    return codes, scales


def _own_values(codes, scales, cols):
    from vtl_amd import capi
    x = torch.empty(codes.shape[0], cols, device="cuda")
    capi.call("vtl_hip_dequantize_mxfp4_f32", _at(codes), _at(scales), codes.shape[0], cols, _at(x), cols)
    return x


def _own_linear(s):
    from vtl_amd import capi
    case, (w, ws) = s["case"], s["w"]
    M, N, K = case["rows"], case["out"], case["cols"]
    y = torch.empty(M, N, device="cuda")
    if case["given"] == "codes":
        capi.call("vtl_hip_linear_mxfp4_f32", _at(s["x"][0]), _at(s["x"][1]), _at(w), _at(ws), _at(s["bias"]), _at(y),
                  M, N, K, int(case["relu"]), None, 0)
    else:
        capi.call("vtl_hip_linear_f32_mxfp4", _at(s["x"]), _at(w), _at(ws), _at(s["bias"]), _at(y), M, N, K, int(case["relu"]), None, 0)
    return y


def _own_experts(s):
    from vtl_amd import capi
    case = s["case"]
    layer = capi.MoE(case["experts"], case["top"], case["dim"], case["hidden"], int(case["renormalize"]), _at(s["router"]), _at(s["router_bias"]),
                     _at(s["gate_up"][0]), _at(s["gate_up"][1]), _at(s["gate_up_bias"]),
                     _at(s["down"][0]), _at(s["down"][1]), _at(s["down_bias"]))
    y = torch.empty_like(s["x"])
    capi.call("vtl_hip_moe_mxfp4_f32", ctypes.byref(layer), _at(s["x"]), _at(y), case["rows"], None, 0)
    return y


def run(s):
    case = s["case"]
    if case["op"] == "codes":
        cols = case["cols"]
        return _own_values(*_own_codes(s), cols) if own else _decode(*_encode(s["x"]), cols)
    if case["op"] == "values":
        return _own_values(*s["w"], case["cols"]) if own else _decode(*s["w"], case["cols"])
    if case["op"] == "linear":
        return _own_linear(s) if own else _plain_linear(s)
    return _own_experts(s) if own else _plain_experts(s)


def work(case):
    def held(rows, cols):
        return rows * (-(-cols // 2) + -(-cols // 32))

    if case["op"] in ("codes", "values"):
        rows, cols = case["rows"], case["cols"]
        once = held(rows, cols) + 4 * rows * cols
        return {"bytes": 2 * once if case["op"] == "codes" else once, "flops": rows * cols * (2 if case["op"] == "codes" else 1)}
    if case["op"] == "linear":
        M, N, K = case["rows"], case["out"], case["cols"]
        x = held(M, K) if case["given"] == "codes" else 4 * M * K
        return {"bytes": x + held(N, K) + 4 * M * N + (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    T, E, D, F, k = (case[n] for n in ("rows", "experts", "dim", "hidden", "top"))
    active = E * (1.0 - (1.0 - k / E) ** T)        # experts that somebody chose, where all are as likely
    return {"bytes": int(active * (held(2 * F, D) + held(D, F))) + 4 * E * D + 8 * T * D, "flops": 2 * T * E * D + 6 * T * k * F * D}


def exact(case, seed):
    """The definition in 64 bits, from the format's description and value by value."""
    s = prepare(case, seed)
    grid = torch.tensor(_VALUES, dtype=torch.float64, device="cuda")

    def held(pair, rows, cols):
        """What rows of codes stand for."""
        codes, scales = (t[rows] for t in pair)
        at = torch.arange(cols, device="cuda")
        code = (codes[:, at // 2] >> (4 * (at % 2)).to(torch.uint8)) & 15
        v = grid[(code & 7).long()]
        return torch.where(code >= 8, -v, v) * torch.pow(2.0, scales[:, at // 32].double() - 127.0)

    def nearest(x):
        """What f32 rows stand for as codes: by distance from the eight magnitudes, the even code where two are as near."""
        rows, cols = x.shape
        out = torch.zeros(rows, cols, dtype=torch.float64, device="cuda")
        for lo in range(0, cols, 32):
            b = x[:, lo:lo + 32].double()
            top = b.abs().amax(1, keepdim=True)
            e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
            e = torch.where(torch.pow(2.0, e) > top, e - 1, torch.where(torch.pow(2.0, e + 1) <= top, e + 1, e))
            unit = torch.pow(2.0, torch.clamp(torch.where(top > 0, e, torch.zeros_like(e)) - 2, min=-127.0))
            away = ((b / unit).abs()[..., None] - grid).abs()
            near = away == away.amin(-1, keepdim=True)
            index = torch.arange(8, device="cuda").expand_as(near)
            pick = torch.where(near, index + 8 * (index % 2), torch.full_like(index, 99)).amin(-1) % 8
            out[:, lo:lo + 32] = torch.sign(b) * grid[pick] * unit
        return out

    if case["op"] == "codes":
        step = max(1, (1 << 24) // case["cols"])
        return torch.cat([nearest(s["x"][lo:lo + step]) for lo in range(0, case["rows"], step)])
    if case["op"] == "values":
        return held(s["w"], slice(None), case["cols"])
    if case["op"] == "linear":
        x = held(s["x"], slice(None), case["cols"]) if case["given"] == "codes" else nearest(s["x"])
        y = torch.matmul(x, held(s["w"], slice(None), case["cols"]).T)
        if s["bias"] is not None:
            y += s["bias"].double()
        return y.clamp(min=0.0) if case["relu"] else y
    x, dim, hidden = s["x"].double(), case["dim"], case["hidden"]
    score = torch.matmul(x, s["router"].double().T).float()     # a score is an f32 number by definition
    if s["router_bias"] is not None:
        score = score + s["router_bias"]
    p = torch.softmax(score.double(), 1)
    y = torch.zeros(case["rows"], dim, dtype=torch.float64, device="cuda")
    rows, experts = case["rows"], case["experts"]
    ranks = (score[:, None, :] > score[:, :, None]).sum(-1)
    ranks += ((score[:, None, :] == score[:, :, None]) & torch.ones(experts, experts, device="cuda", dtype=torch.bool).tril(-1)).sum(-1)
    p = torch.where(ranks < case["top"], p, torch.zeros_like(p))
    if case["renormalize"]:
        p = p / p.sum(1, keepdim=True)
    for e in range(experts):
        mine = (ranks[:, e] < case["top"]).nonzero()[:, 0]
        if not len(mine):
            continue
        gu = torch.matmul(x[mine], held(s["gate_up"], slice(e * 2 * hidden, (e + 1) * 2 * hidden), dim).T)
        if s["gate_up_bias"] is not None:
            gu += s["gate_up_bias"][e].double()
        h = gu[:, :hidden] * torch.sigmoid(gu[:, :hidden]) * gu[:, hidden:]
        out = torch.matmul(h, held(s["down"], slice(e * dim, (e + 1) * dim), hidden).T)
        if s["down_bias"] is not None:
            out += s["down_bias"][e].double()
        y[mine] += p[mine, e:e + 1] * out
    return y
