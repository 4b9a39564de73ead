"""4-bit rows whose places do not fit 32 bits, and the longest ones: of weights of several GB only the last rows are set and looked at."""
import numpy as np
import pytest

import mx_reference as mx
from vtl_amd import HipMoE, HipMxfp4, capi, linear_mxfp4_hip, moe_mxfp4_hip
from vtl_amd.storage import HipStorage
from vtl_amd.tensor import HipTensor

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]
dev = HipTensor.from_host


def normal(seed, *shape, std=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * std).astype(np.float32)


def drawn(seed, rows, cols):
    """Padded codes and scales, about 1 / sqrt(cols) in size (what is behind the end of a row is zeros)."""
    rng = np.random.default_rng(seed)
    codes, scales = rng.integers(0, 256, (rows, mx.padded(cols) // 2), np.uint8), np.zeros((rows, mx.padded(cols) // 32), np.uint8)
    scales[:] = 127 - int(np.log2(3 * cols ** 0.5)) + rng.integers(-1, 2, scales.shape)
    assert cols % 256 == 0
    return codes, scales


def rows_at_the_end(rows, cols, codes, scales):
    """A matrix of which nothing but the last rows is set."""
    q = HipMxfp4.empty(rows, cols)
    for to, part in ((q.codes, codes), (q.scales, scales)):
        capi.call("vtl_hip_memcpy_h2d", to.ptr + to.size - part.nbytes, part.ctypes.data, part.nbytes)
    return q


@pytest.mark.parametrize("M", [2, 20, 200])
def test_weights_behind_4_gib(M):
    N, K, last = 70000, 131072, 5
    codes, scales = drawn(1, last, K)
    w = rows_at_the_end(N, K, codes, scales)
    x = normal(2, M, K)
    y = linear_mxfp4_hip(dev(x).quantize_mxfp4(), w)
    got = y.cpu().reshape(M, N)[:, -last:]
    want, far = mx.linear(mx.decode(*mx.encode(x), K), mx.decode(codes, scales, K), None, False)
    assert (np.abs(got - want) <= far).all(), float((np.abs(got - want) / far).max())
    w.release()


def test_codes_behind_4_gib_and_back():
    rows, cols, last = 140000, 65536, 3
    codes, scales = drawn(3, last, cols)
    q = rows_at_the_end(rows, cols, codes, scales)
    x = HipStorage.empty(last * cols, np.float32)
    at = rows - last
    values = HipTensor(x, [last, cols])
    capi.call("vtl_hip_dequantize_mxfp4_f32", q.codes.ptr, q.scales.ptr, 0, cols, values.ptr, cols)     # no rows: nothing is written
    capi.call("vtl_hip_dequantize_mxfp4_f32", q.codes.ptr + at * (cols // 2), q.scales.ptr + at * (cols // 32), last, cols, values.ptr, cols)
    assert np.array_equal(values.cpu(), mx.decode(codes, scales, cols).astype(np.float32))
    # f32 rows so far apart that the last begins behind 4 GiB of them
    stride = 700 << 20
    wide = HipStorage.empty((last - 1) * stride + cols, np.float32)
    host = normal(4, last, cols)
    for i in range(last):
        capi.call("vtl_hip_memcpy_h2d", wide.ptr + 4 * i * stride, host[i].ctypes.data, host[i].nbytes)
    capi.call("vtl_hip_quantize_f32_mxfp4", wide.ptr, stride, last, cols, q.codes.ptr + at * (cols // 2), q.scales.ptr + at * (cols // 32))
    want = mx.encode(host)
    got = HipMxfp4.empty(last, cols)
    capi.call("vtl_hip_memcpy_d2d", got.codes.ptr, q.codes.ptr + at * (cols // 2), got.codes.size)
    capi.call("vtl_hip_memcpy_d2d", got.scales.ptr, q.scales.ptr + at * (cols // 32), got.scales.size)
    assert np.array_equal(got.codes.cpu().reshape(want[0].shape), want[0]) and np.array_equal(got.scales.cpu().reshape(want[1].shape), want[1])
    q.release()
    wide.release()


@pytest.mark.parametrize("tokens", [1, 12])
def test_experts_behind_4_gib(tokens):
    experts, dim, hidden = 512, 16384, 1024
    gu, dn = drawn(5, 2 * hidden, dim), drawn(6, dim, hidden)
    gate_up, down = rows_at_the_end(experts * 2 * hidden, dim, *gu), rows_at_the_end(experts * dim, hidden, *dn)
    bias = np.full(experts, -np.inf, np.float32)
    bias[-1] = 0.0
    router, x = normal(7, experts, dim, std=dim ** -0.5), normal(8, tokens, dim)
    layer = HipMoE(dev(router), gate_up, down, 1, True, dev(bias))
    got = moe_mxfp4_hip(layer, dev(x)).cpu()
    want, far = mx.experts(x, router[-1:], mx.decode(*gu, dim)[None], mx.decode(*dn, hidden)[None], 1, True)
    assert (np.abs(got - want) <= far).all(), float((np.abs(got - want) / far).max())
    gate_up.release()
    down.release()


@pytest.mark.parametrize("dim,hidden,tokens", [(65536, 256, 2), (256, 65536, 3), (65536, 256, 20), (256, 65536, 20)])
def test_longest_rows_of_experts(dim, hidden, tokens):
    gu, dn = drawn(9, 2 * 2 * hidden, dim), drawn(10, 2 * dim, hidden)
    router, x = normal(11, 2, dim, std=dim ** -0.5), normal(12, tokens, dim)
    layer = HipMoE(dev(router), HipMxfp4.from_packed(*gu, dim), HipMxfp4.from_packed(*dn, hidden), 2)
    got = moe_mxfp4_hip(layer, dev(x)).cpu()
    want, far = mx.experts(x, router, mx.decode(*gu, dim).reshape(2, 2 * hidden, dim), mx.decode(*dn, hidden).reshape(2, dim, hidden), 2, True)
    assert (np.abs(got - want) <= far).all(), float((np.abs(got - want) / far).max())


@pytest.mark.parametrize("M", [1, 7, 30, 300])
def test_long_rows(M):
    N, K = 40, 1 << 18
    codes, scales = drawn(13, N, K)
    x = normal(14, M, K)
    y = linear_mxfp4_hip(dev(x).quantize_mxfp4(), HipMxfp4.from_packed(codes, scales, K)).cpu()
    want, far = mx.linear(mx.decode(*mx.encode(x), K), mx.decode(codes, scales, K), None, False)
    assert (np.abs(y - want) <= far).all(), float((np.abs(y - want) / far).max())
