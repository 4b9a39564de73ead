"""Microscaled 4-bit rows, linear layers and a layer of experts by their definitions, in numpy and 64 bits, with how far f32 sums may be off."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
BORDERS = (GRID[1:] + GRID[:-1]) / 2
U = 2.0 ** -24      # half a step of f32


def padded(cols):
    return -(-cols // 256) * 256


def encode(x):
    """Packed codes and scales of f32 rows, padded."""
    rows, cols = x.shape
    v = np.zeros((rows, padded(cols)), np.float32)
    v[:, :cols] = x
    blocks = v.reshape(rows, -1, 32)
    good = np.isfinite(blocks).all(-1)
    clean = np.where(good[..., None], blocks, 0).astype(np.float64)
    top = np.abs(clean).max(-1)
    e = np.frexp(np.where(top > 0, top, 1))[1] - 1                  # 2^e <= top < 2^(e + 1)
    byte = np.where(top > 0, np.maximum(e + 127 - 2, 0), 0)
    q = np.abs(clean) / np.exp2(byte - 127.0)[..., None]
    # the nearest, the even one of two: how many borders between neighbours lie below, and one more on a border above an odd code
    code = np.searchsorted(BORDERS, q)
    code = code + ((code % 2 == 1) & (q == BORDERS[np.minimum(code, 6)]))
    code = np.where(np.signbit(blocks) & good[..., None], code + 8, code)
    code = code.reshape(rows, -1).astype(np.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), np.where(good, byte, 255).astype(np.uint8)


def decode(codes, scales, cols):
    """What they stand for, in f64 (NaN where a scale is none)."""
    code = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    v = np.where(code >= 8, -GRID[code & 7], GRID[code & 7])
    factor = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(codes.shape[0], -1, 32) * factor[..., None]).reshape(codes.shape[0], -1)[:, :cols]


def linear(x, w, bias, relu):
    """x . w^T + bias of f64 values that are codes', and how far f32 sums may be off: block sums are exact, and each that is added is rounded once,
    as are the waves' and ranges' sums (32 and 64 of them at most) and the bias."""
    y = x @ w.T
    far = (x.shape[1] / 32 + 100) * U * (np.abs(x) @ np.abs(w).T)
    if bias is not None:
        y = y + bias
        far = far + U * np.abs(y)
    return (np.where(y < 0, 0.0, y) if relu else y), far + 1e-44


def scores(x, router, bias):
    s = (x.astype(np.float64) @ router.astype(np.float64).T).astype(np.float32)
    return s if bias is None else (s + bias).astype(np.float32)


def choose(score, top):
    """Each token's experts: the largest scores, the lower index of equal ones, NaN last."""
    key = np.where(np.isnan(score), -np.inf, score.astype(np.float64))
    order = np.lexsort((np.broadcast_to(np.arange(score.shape[1]), score.shape), -key, np.isnan(score)), axis=-1)
    return order[:, :top]


def experts(x, router, gate_up, down, top, renormalize, router_bias=None, gate_up_bias=None, down_bias=None):
    """The layer's output, and how far it may be off.  gate_up [experts, 2 hidden, dim] and down [experts, dim, hidden] in f64."""
    tokens, dim = x.shape
    hidden = down.shape[2]
    s = scores(x, router, router_bias)
    chosen = choose(s, top)
    p = np.exp(s.astype(np.float64) - s.max(1, keepdims=True))
    taken = np.take_along_axis(p, chosen, 1)
    weight = taken / (taken.sum(1, keepdims=True) if renormalize else p.sum(1, keepdims=True))
    # an exponential of a difference d (rounded: |d| U), its own 2 steps, sums of up to 512 in a tree of at most 16 additions, a quotient
    # (the exponential of minus infinity is exactly 0)
    spread = s.max(1, keepdims=True) - s
    spread = np.where(np.isinf(spread), 0, spread)
    off_p = U * (np.abs(np.take_along_axis(spread, chosen, 1)) + spread.max() + 40)
    y, far = np.zeros((tokens, dim)), np.zeros((tokens, dim))
    x64 = x.astype(np.float64)
    block = np.zeros((tokens, padded(dim)))
    block[:, :dim] = np.abs(x64)
    top_x = np.repeat(block.reshape(tokens, -1, 32).max(-1), 32, 1)[:, :dim]
    for t in range(tokens):
        for k in range(top):
            e, w = chosen[t, k], weight[t, k]
            g = gate_up[e]
            gu = g @ x64[t]
            # five digits' columns of dim / 32 block sums each, digits that stop at 2^-24 of the block's largest, joins
            off = (dim / 32 + 100) * U * (np.abs(g) @ (np.abs(x64[t]) * 1.1)) + U * (np.abs(g) @ top_x[t])
            if gate_up_bias is not None:
                gu = gu + gate_up_bias[e]
                off = off + U * np.abs(gu)
            gate, up = gu[:hidden], gu[hidden:]
            sig = 1 / (1 + np.exp(-gate))
            silu = gate * sig
            h = w * silu * up
            # |d silu / d g| <= 1.1; the exponential is off by |g| U and 2 steps, three operations behind it, two products
            off_h = np.abs(w) * (1.1 * off[:hidden] * (np.abs(up) + off[hidden:]) + np.abs(silu) * off[hidden:]) + np.abs(h) * (U * (np.abs(gate) + 12) + off_p[t, k])
            d = down[e]
            y[t] += d @ h
            hp = np.zeros(padded(hidden))
            hp[:hidden] = np.abs(h) + off_h
            top_h = np.repeat(hp.reshape(-1, 32).max(-1), 32)[:hidden]
            far[t] += np.abs(d) @ (1.1 * off_h + U * top_h) + (top * hidden / 32 + 100) * U * (np.abs(d) @ (1.1 * np.abs(h) + off_h))
            if down_bias is not None:
                y[t] += w * down_bias[e]
                far[t] += np.abs(w * down_bias[e]) * (U * (top + 4) + off_p[t, k])
        far[t] += 2 * U * np.abs(y[t])
    return y, far + 1e-37
