"""How near attention over the int8 cache comes to its definition, as a norm over a call: near enough that losing one of the two fp16 halves of the queries or of
the weights shows.  (The bound of every single value, kv_reference.attend's, is for the worst sums; it lets such a loss pass.)

The norm: the scores of these cases are below 2^5 in powers of two, where a step of f32 is 2^-19 at most.  A score is rounded three times (the
product with the key's scale, the difference from the maximum, and what the sums of its products lose), half a step each and in the mean square
1 / sqrt(12) of one: sqrt(3) 2^-19 / sqrt(12) = 2^-20, of which a weight is off by ln 2 times, and its row's sum by no more.  Both, the exponential
(2^-23), the weights' 22 bits and the f32 sums of values come to 2 ln 2 2^-20 + 2^-21 = 1.8e-6 at most; the limit is twice that."""
import numpy as np
import pytest

from kv_reference import Cache
from test_gpu_kv import ATTENDS, normal
from vtl_amd import attention_i8_hip
from vtl_amd.tensor import HipTensor

LIMIT = 3.6e-6


def off(got, want):
    """Relative, in the norm, over the rows that see a token."""
    some = np.abs(want).max(-1) > 0
    return float(np.linalg.norm((got - want)[some]) / np.linalg.norm(want[some])) if some.any() else 0.0


@pytest.mark.gpu
@pytest.mark.usefixtures("hip")
@pytest.mark.parametrize("lengths,counts,page,heads,kv_heads,dim", ATTENDS)
def test_norm(lengths, counts, page, heads, kv_heads, dim):
    c = Cache(lengths, page, kv_heads, dim, seed=heads).to_device()
    b = c.batch(counts)
    q = normal(b.rows, b.rows, heads, dim, std=2.0)
    want, _ = c.attend(q, heads, np.float32(dim ** -0.5), True)
    t = HipTensor.from_host(q)
    for most_length in (b.handle.most_length, 64):      # the tokens of many rows in several parts, and in one
        b.handle.most_length = most_length
        assert off(attention_i8_hip(c.cache, b, t, heads).cpu(), want) <= LIMIT


def halves(x, both, to):
    """What is left of rows of x as one fp16 number or two, their largest values between 2^to and 2^(to + 1)."""
    unit = np.exp2(to - np.floor(np.log2(np.maximum(np.abs(x).max(-1, keepdims=True), 1e-300))))
    x = (x * unit).astype(np.float32)
    hi = x.astype(np.float16).astype(np.float32)
    lo = (x - hi).astype(np.float16).astype(np.float32) if both else 0
    return (hi + lo).astype(np.float64) / unit


def attend_in_halves(c, q, heads, scale, both_of_q, both_of_weights):
    """The kernels' arithmetic, but for the order of their sums."""
    out = np.zeros((q.shape[0], heads, c.dim))
    kc, vc, ks, vs = c.parts()
    for b in range(len(c.lengths)):
        lo, hi = c.rows_of(b)
        n = c.length(b)
        at = [c.place(b, j) for j in range(n)]
        for h in range(heads if n else 0):
            g = h // (heads // c.kv_heads)
            keys = np.array([kc[p, g, :, s].reshape(-1)[:c.dim] for p, s in at], np.float64)
            values = np.array([vc[p, g, s // 16, :c.dim, s % 16] for p, s in at], np.float64)
            x = q[lo:hi, h] * np.float32(scale) * np.float32(np.log2(np.e))
            s = (halves(x, both_of_q, 14) @ keys.T).astype(np.float32) * np.array([ks[p, g, s] for p, s in at])
            s[np.arange(n)[None] > (np.arange(lo, hi) - hi + n)[:, None]] = -np.inf
            w = np.exp2(s - s.max(1, keepdims=True))
            o = halves(w * np.array([vs[p, g, s] for p, s in at]), both_of_weights, 13) @ values
            out[lo:hi, h] = o.astype(np.float32) / w.sum(1, keepdims=True)
    return out


@pytest.mark.parametrize("lengths,counts,page,heads,kv_heads,dim", [
    ([300], [1], 16, 8, 4, 64), ([777, 50], [1, 1], 64, 4, 2, 80), ([300], [1], 16, 32, 8, 128), ([777, 5], [1, 1], 128, 4, 1, 256), ([400], [35], 16, 3, 3, 64),
    ([333], [40], 32, 2, 1, 80), ([210], [65], 64, 2, 2, 128), ([260], [20], 64, 1, 1, 256)])
def test_the_limit_is_above_two_halves_and_below_one(lengths, counts, page, heads, kv_heads, dim):
    c = Cache(lengths, page, kv_heads, dim, seed=heads)
    c.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    scale = np.float32(dim ** -0.5)
    q = normal(1, sum(counts), heads, dim, std=2.0)
    want, _ = c.attend(q, heads, scale, True)
    with np.errstate(invalid="ignore", divide="ignore"):
        assert off(attend_in_halves(c, q, heads, scale, True, True), want) <= LIMIT / 2
        assert off(attend_in_halves(c, q, heads, scale, False, True), want) >= 4 * LIMIT
        assert off(attend_in_halves(c, q, heads, scale, True, False), want) >= 4 * LIMIT
