"""Products of 4-bit rows, row by row and column by column: what a worst case allows each output would hide a register that is read too early."""
import numpy as np
import pytest

import mx_reference as mx
from vtl_amd import linear_f32_mxfp4_hip, linear_mxfp4_hip
from vtl_amd.tensor import HipTensor

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]
dev = HipTensor.from_host

SIZES = [(1, 700, 4096), (2, 9000, 2500), (4, 300, 13742), (6, 6200, 4200), (7, 700, 3000), (16, 1000, 1024), (20, 6000, 1300), (32, 512, 4097), (64, 4100, 1100),
         (65, 6064, 10917), (66, 2886, 13742), (90, 1000, 6000), (100, 4096, 14336), (201, 9000, 2100), (300, 300, 8000), (512, 512, 1024), (768, 8192, 4096), (1000, 1100, 520),
         (1172, 10044, 261), (2560, 4096, 1024)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("spread", [1, 7])     # of blocks' sizes, in powers of two: sums that are exact in f32, most of them, and sums that are not
def test_rows_and_columns(M, N, K, spread):
    rng = np.random.default_rng(M + N + K)
    def rows(n):
        sizes = np.repeat(rng.integers(-spread, spread + 1, (n, -(-K // 32))), 32, 1)[:, :K]
        return dev(rng.standard_normal((n, K), np.float32) * np.exp2(sizes).astype(np.float32)).quantize_mxfp4()

    x, w = rows(M), rows(N)
    xd, wd = x.dequantize().cpu().astype(np.float64), w.dequantize().cpu().astype(np.float64)
    want, size = xd @ wd.T, (xd ** 2) @ (wd ** 2).T         # what sums are, and their squares as signs would have it by chance
    y = linear_mxfp4_hip(x, w).cpu()
    # Blocks' sums are exact; one is added for 32 values, in the unit, and up to 32 more where waves and ranges of K meet.  Each is off by at most a
    # step of a sum that is no larger, on average, than the last one
    limit = 2 * (K / 32 + 33) * mx.U
    for axis in (0, 1):
        off = np.linalg.norm(y - want, axis=axis) / np.sqrt(size.sum(axis))
        assert (off <= limit).all(), (axis, float(off.max() / limit), int(off.argmax()))
    # nothing but ReLU
    assert np.array_equal(linear_mxfp4_hip(x, w, None, True).cpu(), np.where(y < 0, np.float32(0), y))


@pytest.mark.parametrize("M", [1, 6, 12, 40, 200])
def test_relu_without_a_bias_behind_codes(M):
    rng = np.random.default_rng(M)
    x, w = dev(rng.standard_normal((M, 520), np.float32)), dev(rng.standard_normal((300, 520), np.float32)).quantize_mxfp4()
    y = linear_f32_mxfp4_hip(x, w).cpu()
    assert (y < 0).any() and np.array_equal(linear_f32_mxfp4_hip(x, w, None, True).cpu(), np.where(y < 0, np.float32(0), y))
