"""Activations of a layer of experts whose neighbours in a block of 32 are far larger, where nothing hides what becomes of them: the large ones meet
weights of 0."""
import numpy as np
import pytest

import mx_reference as mx
from vtl_amd import HipMoE, HipMxfp4, moe_mxfp4_hip
from vtl_amd.tensor import HipTensor

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]
dev = HipTensor.from_host
LARGE = [2.0 ** 8, 2.0 ** 13, 2.0 ** 17, 2.0 ** 21]


def normal(seed, *shape, std=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * std).astype(np.float32)


def weights_without(seed, rows, cols):
    """Rows of weights with the code 0 at the first place of each block of 32, and what they stand for."""
    w = normal(seed, rows, cols, std=cols ** -0.5)
    w[:, ::32] = 0.0
    return dev(w).quantize_mxfp4(), mx.decode(*mx.encode(w), cols)


def tops(values):
    """The largest of each value's block."""
    tokens, cols = values.shape
    top = np.zeros((tokens, mx.padded(cols)))
    top[:, :cols] = np.abs(values)
    return np.repeat(top.reshape(tokens, -1, 32).max(-1), 32, 1)[:, :cols]


def check(got, values, weights, times, steps):
    """A value keeps 24 bits of its own down to 2^-6 of the largest of its block, below that all but 2^-30 of the largest.  Each output is within the worst of
    that, of sums of digits' products, of blocks and of waves, and of `steps` roundings in front and behind; and since roundings do not all go one way, a token's
    outputs together are within 64 half steps and twice the root of the squares of what every value of every output may lose."""
    want, a, top = times * (values @ weights.T), np.abs(weights).T, tops(values)
    cols = values.shape[1]
    far = times * ((cols / 32 + 100 + steps) * mx.U * (np.abs(values) @ a) + 2.0 ** -30 * (top @ a)) + steps * mx.U * np.abs(want)
    off = np.abs(got - want)
    assert (off <= far).all(), float((off / far).max())
    lost = times * 2.0 ** -30 * np.sqrt(((top ** 2) @ (a ** 2)).sum(1))
    together = np.linalg.norm(off, axis=1)
    limit = 64 * mx.U * np.linalg.norm(want, axis=1) + 2 * lost
    assert (together <= limit).all(), (float((together / limit).max()), float((together / np.linalg.norm(want, axis=1)).max() / mx.U))


@pytest.mark.parametrize("large", LARGE)
@pytest.mark.parametrize("dim,tokens", [(256, 1), (1000, 5), (520, 12), (256, 64)])
def test_tokens(dim, tokens, large):
    """Gates of 64, where the sigmoid is 1 in f32, and 0 from the second hidden value of a block on, so that outputs are 64 times one up each."""
    n = dim // 32
    hidden = 32 * n
    x = normal(tokens, tokens, dim)
    x[:, ::32] *= np.float32(large)
    up_q, up = weights_without(dim, hidden, dim)
    keep = np.arange(hidden) % 32 == 0
    codes, scales = up_q.packed()
    none = np.zeros((hidden, dim), np.float32)
    gq = dev(none).quantize_mxfp4().packed()
    gate_up = HipMxfp4.from_packed(np.concatenate([gq[0], codes * keep[:, None]]), np.concatenate([gq[1], scales]), dim)
    bias = np.concatenate([np.full(hidden, 64.0), np.zeros(hidden)]).astype(np.float32)
    down = np.zeros((dim, hidden), np.float32)
    down[np.arange(n), 32 * np.arange(n)] = 1.0
    layer = HipMoE(dev(np.zeros((1, dim), np.float32)), gate_up, dev(down).quantize_mxfp4(), 1, True, None, dev(bias))
    got = moe_mxfp4_hip(layer, dev(x)).cpu()[:, :n]
    check(got, x.astype(np.float64), up[::32][:n], 64, 8)


@pytest.mark.parametrize("large", LARGE)
@pytest.mark.parametrize("dim,hidden,tokens", [(64, 256, 1), (64, 1000, 5), (96, 520, 12), (40, 2080, 64)])
def test_hidden_values(dim, hidden, tokens, large):
    """Tokens of zeros: gates of 64 and ups are the biases."""
    down_q, down = weights_without(hidden, dim, hidden)
    up = normal(hidden + 1, hidden)
    up[::32] *= np.float32(large)
    bias = np.concatenate([np.full(hidden, 64.0), up]).astype(np.float32)
    none = np.zeros((2 * hidden, dim), np.float32)
    layer = HipMoE(dev(np.zeros((1, dim), np.float32)), dev(none).quantize_mxfp4(), down_q, 1, True, None, dev(bias))
    got = moe_mxfp4_hip(layer, dev(np.zeros((tokens, dim), np.float32))).cpu()
    check(got, np.broadcast_to(up.astype(np.float64), (tokens, hidden)), down, 64, 8)
