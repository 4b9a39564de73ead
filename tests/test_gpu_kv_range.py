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


def results(c, counts, q, heads, scale, causal=True):
    """What comes out with the tokens cut into parts as the library would, and, where rows are many, in one part (the host knows of 64 tokens only)."""
    b, t = c.batch(counts), HipTensor.from_host(q)
    yield attention_i8_hip(c.cache, b, t, heads, scale=scale, causal=causal).cpu()
    b.handle.most_length = 64
    yield attention_i8_hip(c.cache, b, t, heads, scale=scale, causal=causal).cpu()


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
    for out in results(c, counts, q, 4, dim ** -0.5):
        want, far = c.attend(q, 4, np.float32(dim ** -0.5), True)
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
    for out in results(c, counts, q, 4, 1.0):
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
    for out in results(c, counts, q, 4, 0.125):
        want, far = c.attend(q, 4, np.float32(0.125), True)
        spoiled = np.isnan(want)
        assert spoiled[-1, :2].all() and not spoiled[:, 2:].any() and (rows < 3 or not spoiled[0].any())
        assert np.isnan(out[spoiled]).all()
        assert (np.abs(out - want)[~spoiled] <= far[~spoiled]).all()


def attend_alone(c, q, heads, scale, causal):
    """As Cache.attend, but with a bound that nothing enters that a row gives no weight to: a weight times its value's scale is off by 2^-25 / 2^13 of
    the largest of the row's such products, a score by half a step more below 128 (2^-18) where its row has no weights but for tokens of small scales."""
    out, far = np.zeros((q.shape[0], heads, c.dim)), np.full((q.shape[0], heads, c.dim), 1e-30)
    for b in range(len(c.lengths)):
        lo, hi = c.rows_of(b)
        n = c.length(b)
        k, v, there = (x.astype(np.float64) for x in c.tokens(b, np.arange(n)))
        last = np.arange(lo, hi) - hi + n if causal else np.full(hi - lo, n - 1)
        seen = (there[None] > 0) & (np.arange(n)[None] <= last[:, None])
        for h in range(heads):
            kg, vg, x = k[:, h // (heads // c.kv_heads)], v[:, h // (heads // c.kv_heads)], q[lo:hi, h].astype(np.float64)
            s, size = x @ kg.T * scale, np.abs(x) @ np.abs(kg).T * abs(scale)
            top = np.where(seen, s, -np.inf).max(1)[:, None]
            w = np.where(seen, np.exp(np.minimum(s - top, 0)), 0)
            total = w.sum(1)[:, None]
            score_off = np.where(seen, size * (2.0 ** -22 + 2.0 ** -23 + c.dim * 2.0 ** -24) + 2.0 ** -21 * (np.abs(s) + np.abs(top)), 0).max(1)[:, None]
            largest = (w * np.abs(vg).max(1)).max(1)[:, None] / total
            out[lo:hi, h] = w / total @ vg
            far[lo:hi, h] += (w / total @ np.abs(vg)) * (2 * (score_off + 2.0 ** -18) + 2.0 ** -20 + (n / 8 + 64) * 2.0 ** -24)
            far[lo:hi, h] += n * 2.0 ** -38 * largest * 127 / 64      # random codes come to half of 127 at least
    return out, far


@pytest.mark.parametrize("counts", [[4], [30], [90], [190]])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("power", [14, 30, 60, 100])
def test_large_values_that_a_row_does_not_see(counts, dim, power):
    """New tokens in the middle of the call's have values 2^power as large as the others': nothing to the rows in front of them."""
    c = Cache([400], 32, 2, dim, seed=7)
    first = 400 - counts[0] // 2
    vs = c.parts()[3]
    for token in range(first, first + 2):
        page, slot = c.place(0, token)
        vs[page, 0, slot] *= np.float32(2.0 ** power)
    c.to_device()
    q = normal(9, counts[0], 4, dim)
    for out in results(c, counts, q, 4, 0.125):
        want, far = attend_alone(c, q, 4, 0.125, True)
        off = np.abs(out - want)
        assert (off <= far).all(), float((off / far).max())


@pytest.mark.parametrize("counts", ROWS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("power", [20, 50, 90])
def test_large_values_without_weight(counts, dim, power):
    """Some tokens have values 2^power as large as the others' and weights that are as much smaller, or none at all."""
    c = Cache([700, 330], 32, 2, dim, seed=8)
    kc, _, ks, vs = c.parts()
    for b in range(2):
        for i, token in enumerate((1, 65, 66, 190, 230)):
            page, slot = c.place(b, token)
            kc[page, :, :, slot] = -100
            ks[page, :, slot] = np.float32((power + 10 if i % 2 else 300) / (100 * dim * 1.5))
            vs[page, :, slot] *= np.float32(2.0 ** power)
    c.to_device()
    q = np.random.default_rng(10).uniform(1, 2, (rows_of(counts), 4, dim)).astype(np.float32)
    for causal in (True, False):
        for out in results(c, counts, q, 4, 1.0, causal):
            want, far = attend_alone(c, q, 4, 1.0, causal)
            off = np.abs(out - want)
            assert (off <= far).all(), float((off / far).max())


@pytest.mark.parametrize("counts", ROWS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("mean", [-250, -500])
def test_low_scores_beside_large_values(counts, dim, mean):
    """All scores are far below zero, and values' scales 2^40 apart from the first token on."""
    c = Cache([400, 330], 32, 2, dim, seed=16)
    kc, _, ks, vs = c.parts()
    rng = np.random.default_rng(17)
    kc[:] = rng.integers(-103, -96, kc.shape)
    written = c.table[c.table >= 0]
    ks[written], vs[written] = np.float32(-mean / (100 * dim * 1.5)), np.exp2(rng.integers(-20, 20, vs[written].shape)).astype(np.float32)
    c.to_device()
    q = rng.uniform(1, 2, (rows_of(counts), 4, dim)).astype(np.float32)
    for out in results(c, counts, q, 4, 1.0):
        want, far = attend_alone(c, q, 4, 1.0, True)
        off = np.abs(out - want)
        assert (off <= far).all(), float((off / far).max())


@pytest.mark.parametrize("counts", ROWS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("power", [16, 30, 80])
def test_weight_on_tokens_without_values(counts, dim, power):
    """A few tokens have all the weight and values of zero: what comes out is the others', by 2^power smaller and as exact as ever."""
    c = Cache([400, 330], 32, 2, dim, seed=18)
    kc, _, ks, vs = c.parts()
    ks[c.table[c.table >= 0]] = np.float32(0.02 / dim ** 0.5)        # the others' scores are near 0
    for b in range(2):
        for token in (0, 70, 200):
            page, slot = c.place(b, token)
            kc[page, :, :, slot], ks[page, :, slot], vs[page, :, slot] = 100, np.float32(power * np.log(2) / (100 * dim * 1.5)), 0
    c.to_device()
    q = np.random.default_rng(19).uniform(1, 2, (rows_of(counts), 4, dim)).astype(np.float32)
    for out in results(c, counts, q, 4, 1.0):
        want, far = attend_alone(c, q, 4, 1.0, True)
        off = np.abs(out - want)
        assert (off <= far).all(), float((off / far).max())


@pytest.mark.parametrize("counts", ROWS)
def test_values_that_grow_and_shrink(counts):
    """Values' scales rise by 2^80 along a sequence and fall again, the scores against them: what counts is now here, now there."""
    c = Cache([700, 330], 32, 1, 64, seed=12)
    vs = c.parts()[3]
    for b, n in enumerate((700, 330)):
        for j in range(n):
            page, slot = c.place(b, j)
            vs[page, :, slot] *= np.float32(2.0 ** (40 - abs(j - 150) / 4))
    c.to_device()
    q = normal(13, rows_of(counts), 8, 64, std=6.0)
    for out in results(c, counts, q, 8, 1.0):
        want, far = attend_alone(c, q, 8, 1.0, True)
        off = np.abs(out - want)
        assert (off <= far).all(), float((off / far).max())


@pytest.mark.parametrize("counts", ROWS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("power", [20, 26, 40, 90])
def test_scores_far_above_one(counts, dim, power):
    """Scores so large that f32 has steps of more than 1 there: which of the largest a row takes is the rounding's choice, but its weights are
    none above their sum."""
    c = Cache([700, 330], 32, 2, dim, seed=14).to_device()
    q = normal(15, rows_of(counts), 4, dim) * np.float32(2.0 ** power)
    for out in results(c, counts, q, 4, 1.0):
        for b in range(2):
            lo, hi = c.rows_of(b)
            _, v, _ = c.tokens(b, np.arange(c.length(b)))
            most = np.repeat(np.abs(v).max(0), 2, axis=0)
            assert (np.abs(out[lo:hi]) <= most * (1 + 2.0 ** -12)).all()


@pytest.mark.parametrize("counts", [[4, 5], [30, 20], [90, 70], [250, 300]])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("power", [14, 30, 60, 90])
def test_large_queries_beside_a_row(counts, dim, power):
    """Some rows' queries are 2^power as large as the others': nothing to those."""
    c = Cache([400, 330], 32, 2, dim, seed=9).to_device()
    q = normal(11, sum(counts), 4, dim)
    large = np.zeros(q.shape[:2], bool)
    large[1::7, 1], large[counts[0] - 1, 3] = True, True
    q[large] *= np.float32(2.0 ** power)
    for out in results(c, counts, q, 4, 0.125):
        want, far = c.attend(q, 4, np.float32(0.125), True)
        assert (np.abs(out - want)[~large] <= far[~large]).all()
        assert np.isfinite(out).all()
