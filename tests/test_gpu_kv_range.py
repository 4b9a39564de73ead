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
