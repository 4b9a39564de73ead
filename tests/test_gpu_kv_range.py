"""Attention over the int8 cache where numbers are far from 1, or none: against its definition in 64 bits (kv_reference.py)."""
import numpy as np
import pytest

from kv_reference import Cache
from vtl_amd import attention_i8_hip
from vtl_amd.tensor import HipTensor

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]

# rows of each of two sequences, and whether they are few or many to the library
ROWS = [None, [3, 5], [20, 20], [70, 90]]


def normal(seed, *shape, std=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * std).astype(np.float32)


def attend(c, counts, q, heads, scale, causal=True):
    b = c.batch(counts)
    return attention_i8_hip(c.cache, b, HipTensor.from_host(q), heads, scale=scale, causal=causal).cpu(), *c.attend(q, heads, np.float32(scale), causal)


def rows_of(counts):
    return 2 if counts is None else sum(counts)


@pytest.mark.parametrize("counts", ROWS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("power", [115, 100, -115])
def test_scales_of_keys_far_from_one(counts, dim, power):
    """Keys' scales of 2^power against queries of 2^-power: scores are as ever."""
    c = Cache([700, 330], 32, 2, dim, seed=3)
    ks = c.parts()[2]
    with np.errstate(over="ignore"):        # where nothing has been written
        for page in c.table[c.table >= 0]:
            ks[page] *= np.float32(2.0 ** power)
    c.to_device()
    q = normal(5, rows_of(counts), 4, dim, std=2.0) * np.float32(2.0 ** -power)
    out, want, far = attend(c, counts, q, 4, dim ** -0.5)
    assert (np.abs(out - want) <= far).all()


@pytest.mark.parametrize("counts", ROWS)
@pytest.mark.parametrize("target", [0, 70])
def test_scores_far_below_zero(counts, target):
    """All scores are below -2^100, one token's by a factor of three less than the others': its values are what comes out."""
    c = Cache([300, 180], 16, 2, 64, seed=4)
    kc, _, ks, _ = c.parts()
    kc[:], ks[c.table[c.table >= 0]] = -127, np.float32(3 * 2.0 ** 36)
    for b in range(2):
        page, slot = c.place(b, target)
        ks[page, :, slot] = np.float32(2.0 ** 36)
    c.to_device()
    q = np.random.default_rng(6).uniform(1, 2, (rows_of(counts), 4, 64)).astype(np.float32) * np.float32(2.0 ** 58)
    b = c.batch(counts)
    out = attention_i8_hip(c.cache, b, HipTensor.from_host(q), 4, scale=1.0).cpu()
    for b in range(2):
        lo, hi = c.rows_of(b)
        _, v, _ = c.tokens(b, [target])
        want = np.repeat(v[0], 2, axis=0)
        # the weight is 1, the value's scale two halves of fp16 (22 bits), and sum and quotient are rounded once each
        assert (np.abs(out[lo:hi] - want) <= np.abs(want) * 2.0 ** -20).all()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("counts", [None, [6], [30], [90]])
@pytest.mark.parametrize("dim", [64, 128])
def test_keys_scales_that_are_no_numbers(bad, counts, dim):
    """Whatever the token's codes are, and so whatever sign a score has: the rows that see it are no numbers, and no other."""
    c = Cache([200], 16, 2, dim, seed=6)
    rows = 1 if counts is None else counts[0]
    page, slot = c.place(0, 150 if rows > 49 else 200 - (rows + 1) // 2)
    ks = c.parts()[2]
    ks[page, 0, slot] = bad
    c.to_device()
    q = normal(8, rows, 4, dim)
    out, want, far = attend(c, counts, q, 4, 0.125)
    spoiled = np.isnan(want)
    assert spoiled[-1, :2].all() and not spoiled[:, 2:].any() and (rows < 3 or not spoiled[0].any())
    assert np.isnan(out[spoiled]).all()
    assert (np.abs(out - want)[~spoiled] <= far[~spoiled]).all()
