"""Microscaled 4-bit rows, linear layers and a layer of experts on the device, against their definitions (mx_reference.py)."""
import ctypes as C

import numpy as np
import pytest

import mx_reference as mx
from vtl_amd import HipMoE, HipMxfp4, capi, linear_f32_mxfp4_hip, linear_mxfp4_hip, linear_mxfp4_workspace, moe_mxfp4_hip
from vtl_amd.storage import HipStorage
from vtl_amd.tensor import HipTensor

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]
dev = HipTensor.from_host


def normal(seed, *shape, std=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * std).astype(np.float32)


def fetch(q):
    rows, cols = q.shape
    padded = mx.padded(cols)
    return q.codes.cpu().reshape(rows, padded // 2), q.scales.cpu().reshape(rows, padded // 32)


def wide(seed, rows, cols):
    """Values of all magnitudes, zeros, ties between codes, values at the border of a binade."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-149, 127, (rows, 1)))
    at = rng.random((rows, cols))
    x = np.where(at < 0.1, 0.0, x)
    ties = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9999], (rows, cols)) * np.exp2(rng.integers(-130, 120, (rows, 1)))
    x = np.where(rng.random((rows, 1)) < 0.5, ties * np.sign(x), x)
    return x.astype(np.float32)


# -- codes ----------------------------------------------------------------------------------------

SIZES = [(1, 1), (1, 32), (3, 31), (2, 33), (5, 256), (4, 257), (7, 1000), (65, 96), (1, 20000), (300, 64), (33, 4096)]


@pytest.mark.parametrize("rows,cols", SIZES)
def test_codes_and_values(guard_bands, rows, cols):
    x = wide(rows * cols, rows, cols)
    q = dev(x).quantize_mxfp4()
    codes, scales = fetch(q)
    want_codes, want_scales = mx.encode(x)
    assert np.array_equal(scales, want_scales) and np.array_equal(codes, want_codes)
    with np.errstate(over="ignore"):
        want = mx.decode(want_codes, want_scales, cols).astype(np.float32)
    assert np.array_equal(q.dequantize().cpu().view(np.uint32), want.view(np.uint32))
    back = HipMxfp4.from_packed(*q.packed(), cols)
    assert all(np.array_equal(a, b) for a, b in zip(fetch(back), (codes, scales)))
    q.release()


def test_every_code_and_scale():
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))[:, :128]
    codes[:, :16] = np.arange(240, 256)
    scales = np.tile(np.arange(256, dtype=np.uint8)[:, None], (1, 8))
    got = HipMxfp4.from_packed(codes, scales, 256).dequantize().cpu()
    with np.errstate(over="ignore"):
        want = mx.decode(codes, scales, 256).astype(np.float32)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(want[255]).all()
    assert np.array_equal(got[:255].view(np.uint32), want[:255].view(np.uint32))


def test_no_numbers_take_their_block_with_them():
    x = normal(1, 4, 200)
    x[0, 40], x[1, 199], x[2, 0] = np.nan, np.inf, -np.inf
    q = dev(x).quantize_mxfp4()
    assert all(np.array_equal(a, b) for a, b in zip(fetch(q), mx.encode(x)))
    bad = np.isnan(q.dequantize().cpu())
    want = np.zeros_like(bad)
    want[0, 32:64] = want[1, 192:200] = want[2, :32] = True
    assert np.array_equal(bad, want)


@pytest.mark.parametrize("first,cols,stride", [(0, 64, 64), (4, 64, 100), (1, 64, 100), (3, 61, 97), (32, 300, 1000)])
def test_rows_in_wider_rows(guard_bands, first, cols, stride):
    rows = 19
    both = normal(first, rows, stride)
    t, kept = dev(both), dev(normal(7, rows, stride))
    x = np.ascontiguousarray(both[:, first:first + cols])
    q = HipMxfp4.empty(rows, cols)
    capi.call("vtl_hip_quantize_f32_mxfp4", t.ptr + 4 * first, stride, rows, cols, q.codes.ptr, q.scales.ptr)
    want = mx.encode(x)
    assert all(np.array_equal(a, b) for a, b in zip(fetch(q), want))
    expected = kept.cpu().copy()
    capi.call("vtl_hip_dequantize_mxfp4_f32", q.codes.ptr, q.scales.ptr, rows, cols, kept.ptr + 4 * first, stride)
    expected[:, first:first + cols] = mx.decode(*want, cols)
    assert np.array_equal(kept.cpu(), expected)


# -- linear layers ----------------------------------------------------------------------------------

LINEARS = [(1, 1, 1), (1, 33, 31), (2, 64, 256), (3, 100, 1000), (5, 31, 4096), (8, 256, 700), (9, 40, 513), (16, 1000, 1024), (17, 48, 300), (31, 129, 2048), (32, 512, 4097),
           (33, 64, 256), (64, 130, 520), (65, 65, 65), (100, 1024, 96), (128, 128, 2048), (129, 257, 777), (200, 640, 1300), (256, 256, 256),
           (300, 300, 8000), (513, 770, 256), (1000, 1100, 520), (40, 5000, 512), (2048, 70, 300), (1500, 1536, 512),
           (512, 512, 1024), (256, 768, 3584), (256, 256, 2048), (2560, 4096, 1024),
           (256, 10752, 1024), (201, 9000, 2100), (66, 2886, 13742), (4096, 8192, 1024),
           (20, 6000, 1300), (64, 4100, 1100), (2, 9000, 2500), (3, 17000, 2500), (6, 6200, 4200), (7, 700, 3000), (90, 1000, 6000),
           (1280, 256, 1024), (33, 4666, 64), (33, 4200, 4591), (65, 6064, 10917), (768, 4096, 1024), (263, 8702, 64), (66, 8581, 8726), (566, 10095, 2594),
           (768, 11008, 1024), (1172, 10044, 261), (768, 8192, 4096)]


def check_linear(got, want, far):
    off = np.abs(got - want)
    assert (off <= far).all(), (float((off / far).max()), np.argwhere(~(off <= far))[:5])


@pytest.mark.parametrize("M,N,K", LINEARS)
@pytest.mark.parametrize("bias,relu", [(False, False), (True, True)])
def test_linear(guard_bands, M, N, K, bias, relu):
    x, w = normal(M, M, K), normal(N + 1, N, K, std=K ** -0.5)
    x[:, ::29] *= 9.0
    x *= np.exp2(np.random.default_rng(K).integers(-9, 9, (M, 1))).astype(np.float32)
    b = normal(3, N) if bias else None
    wq = dev(w).quantize_mxfp4()
    xd, wd = mx.decode(*mx.encode(x), K), mx.decode(*mx.encode(w), K)
    want, far = mx.linear(xd, wd, b, relu)
    db = dev(b) if bias else None
    xt = dev(x)
    y = linear_f32_mxfp4_hip(xt, wq, db, relu)
    check_linear(y.cpu(), want, far)
    z = linear_mxfp4_hip(xt.quantize_mxfp4(), wq, db, relu)
    check_linear(z.cpu(), want, far)
    for _ in range(2):      # the same call gives the same bits, with a workspace of its own too
        ws = HipStorage.empty(max(1, linear_mxfp4_workspace(M, N, K)), np.uint8)
        assert np.array_equal(linear_f32_mxfp4_hip(xt, wq, db, relu, workspace=ws).cpu(), y.cpu())


def test_linear_of_blocks_without_a_number():
    for M in (3, 70):
        x, w = normal(1, M, 500), normal(2, 90, 500)
        x[1, 300], w[7, 2] = np.inf, np.nan
        y = linear_f32_mxfp4_hip(dev(x), dev(w).quantize_mxfp4()).cpu()
        want = np.zeros((M, 90), bool)
        want[1], want[:, 7] = True, True
        assert np.array_equal(np.isnan(y), want)


@pytest.mark.parametrize("M", [1, 20, 140])
def test_linear_of_far_scales(M):
    """Rows and weights whose scales are far apart, up to the ends of the bytes: results are f32's."""
    N, K = 96, 512
    x, w = wide(1, M, K), normal(5, N, K)
    x = np.where(np.abs(x) > 1e30, np.float32(1), x)
    wq = dev(w).quantize_mxfp4()
    want, far = mx.linear(mx.decode(*mx.encode(x), K), mx.decode(*mx.encode(w), K), None, False)
    check_linear(linear_f32_mxfp4_hip(dev(x), wq).cpu(), want, far + 2.0 ** -149 * K)


# -- experts ------------------------------------------------------------------------------------------

class Layer:
    def __init__(self, experts, dim, hidden, top, renormalize, bias, seed=0):
        self.args = (experts, dim, hidden, top)
        self.top, self.renormalize = top, renormalize
        self.router = normal(seed, experts, dim, std=dim ** -0.5)
        gu, dn = normal(seed + 1, experts * 2 * hidden, dim, std=dim ** -0.5), normal(seed + 2, experts * dim, hidden, std=hidden ** -0.5)
        self.gate_up, self.down = dev(gu).quantize_mxfp4(), dev(dn).quantize_mxfp4()
        self.gu = mx.decode(*mx.encode(gu), dim).reshape(experts, 2 * hidden, dim)
        self.dn = mx.decode(*mx.encode(dn), hidden).reshape(experts, dim, hidden)
        self.biases = (normal(seed + 3, experts, std=0.3), normal(seed + 4, experts, 2 * hidden, std=0.3), normal(seed + 5, experts, dim, std=0.3)) if bias else (None,) * 3
        self.hip()

    def hip(self):
        self.held = [dev(b) if b is not None else None for b in self.biases]
        self.layer = HipMoE(dev(self.router), self.gate_up, self.down, self.top, self.renormalize, *self.held)

    def want(self, x):
        return mx.experts(x, self.router, self.gu, self.dn, self.top, self.renormalize, *self.biases)


def check_layer(l, x, workspace=None):
    """Each value within what a sum of so many terms may be off by at worst; and since roundings do not all go one way, a token's values together
    within 64 half steps of f32 (2^12 independent ones, as many as the largest layer here has behind each other)."""
    got = moe_mxfp4_hip(l.layer, dev(x), workspace).cpu()
    want, far = l.want(x)
    off = np.abs(got - want)
    together = np.linalg.norm(off, axis=1) / np.maximum(np.linalg.norm(want, axis=1), 1e-30)
    assert (together <= 64 * mx.U).all(), (together.max() / mx.U, int(together.argmax()))
    assert (off <= far).all(), (float(np.nanmax(off / far)), np.argwhere(~(off <= far))[:5])
    return got


MOES = [  # experts, dim, hidden, top, tokens
    (1, 1, 1, 1, 1), (2, 32, 32, 1, 3), (4, 256, 256, 2, 1), (8, 300, 100, 2, 5), (8, 256, 512, 8, 4), (20, 1000, 72, 3, 5), (64, 512, 256, 6, 1),
    (64, 520, 160, 6, 24), (128, 256, 64, 8, 64), (60, 96, 33, 4, 17), (512, 64, 32, 16, 9), (3, 2048, 40, 1, 64), (5, 64, 2000, 5, 33), (130, 40, 16, 2, 2),
    (6, 300, 100, 6, 7), (4, 1000, 530, 2, 20), (16, 264, 72, 16, 64), (200, 96, 64, 2, 6), (9, 2100, 48, 1, 50), (256, 64, 32, 8, 40), (257, 40, 32, 3, 7), (255, 40, 32, 16, 2)]


@pytest.mark.parametrize("experts,dim,hidden,top,tokens", MOES)
@pytest.mark.parametrize("renormalize,bias", [(True, False), (False, True)])
def test_experts(guard_bands, experts, dim, hidden, top, tokens, renormalize, bias):
    l = Layer(experts, dim, hidden, top, renormalize, bias, seed=tokens)
    x = normal(99, tokens, dim)
    x[:, ::31] *= 8.0
    got = check_layer(l, x)
    ws = HipStorage.empty(l.layer.workspace(tokens), np.uint8)
    assert np.array_equal(moe_mxfp4_hip(l.layer, dev(x), ws).cpu(), got)


class LargeLayer(Layer):
    """Of codes and scales drawn as such."""

    def __init__(self, experts, dim, hidden, top, bias, seed=0):
        rng = np.random.default_rng(seed)

        def rows(n, cols):
            codes = rng.integers(0, 256, (n, mx.padded(cols) // 2), np.uint8)
            scales = (127 - int(np.log2(3 * cols ** 0.5)) + rng.integers(-1, 2, (n, mx.padded(cols) // 32))).astype(np.uint8)
            return HipMxfp4.from_packed(codes[:, :-(-cols // 2)], scales[:, :-(-cols // 32)], cols), mx.decode(codes, scales, cols)

        self.top, self.renormalize = top, True
        self.router = normal(seed, experts, dim, std=dim ** -0.5)
        self.gate_up, gu = rows(experts * 2 * hidden, dim)
        self.down, dn = rows(experts * dim, hidden)
        self.gu, self.dn = gu.reshape(experts, 2 * hidden, dim), dn.reshape(experts, dim, hidden)
        self.biases = (normal(seed + 3, experts, std=0.3), normal(seed + 4, experts, 2 * hidden, std=0.3), normal(seed + 5, experts, dim, std=0.3)) if bias else (None,) * 3
        self.hip()


@pytest.mark.parametrize("experts,dim,hidden,top,tokens,bias", [
    (64, 96, 1000, 6, 40, False), (16, 550, 2100, 8, 12, True), (8, 40, 4112, 4, 9, False), (64, 64, 1030, 16, 8, True), (20, 64, 2080, 16, 1, False),
    (96, 1028, 1450, 5, 17, True),      # 128 MB of weights
    (8, 100, 2600, 4, 40, True)])       # 20 pairs of an expert
def test_hidden_values_for_every_compute_unit(guard_bands, experts, dim, hidden, top, tokens, bias):
    l = LargeLayer(experts, dim, hidden, top, bias)
    x = normal(98, tokens, dim)
    assert np.array_equal(check_layer(l, x), check_layer(l, x))


def test_equal_scores_go_to_the_lowest_experts():
    l = Layer(12, 64, 32, 3, True, False)
    l.router[:] = l.router[0]
    l.router[5] *= 2.0
    l.hip()
    check_layer(l, normal(4, 6, 64))


def test_experts_that_a_bias_rules_out():
    l = Layer(9, 64, 48, 4, True, True)
    l.biases[0][[1, 4, 8]] = -np.inf
    l.hip()
    check_layer(l, normal(5, 10, 64))


def test_all_tokens_with_one_expert_and_a_token_each():
    l = Layer(64, 128, 64, 1, False, False)
    x = normal(6, 64, 128)
    l.router[:] = 0.0
    l.router[17, 0] = 1.0
    l.hip()
    x[:, 0] = 50.0
    check_layer(l, x)
    l.router = np.ascontiguousarray(x[:64] * 3.0)
    l.hip()
    check_layer(l, x)


def test_tokens_of_all_magnitudes():
    l = Layer(8, 256, 96, 2, True, False)
    x = normal(8, 40, 256) * np.exp2(np.linspace(-60, 8, 40)).astype(np.float32)[:, None]
    x[3] = 0.0
    check_layer(l, x)


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_a_token_without_a_number_is_alone_with_it(value):
    l = Layer(16, 256, 64, 2, True, True)
    x = normal(9, 7, 256)
    clean = moe_mxfp4_hip(l.layer, dev(x)).cpu()
    x[4, 100] = value
    got = moe_mxfp4_hip(l.layer, dev(x)).cpu()
    assert np.isnan(got[4]).all()
    others = np.arange(7) != 4
    want, far = l.want(np.where(np.isfinite(x), x, 0))
    assert (np.abs(got - want) <= far)[others].all() and np.isfinite(clean).all()


def test_block_of_weights_without_a_number():
    l = Layer(4, 64, 64, 1, True, False)
    x = normal(3, 12, 64)
    scales = l.down.scales.cpu().reshape(4 * 64, 8)
    scales[2 * 64 + 5, 1] = 255
    capi.call("vtl_hip_memcpy_h2d", l.down.scales.ptr, scales.ctypes.data, scales.nbytes)
    got = moe_mxfp4_hip(l.layer, dev(x)).cpu()
    chosen = mx.choose(mx.scores(x, l.router, None), 1)[:, 0]
    want = np.zeros((12, 64), bool)
    want[chosen == 2, 5] = True
    assert (chosen == 2).any() and np.array_equal(np.isnan(got), want)
