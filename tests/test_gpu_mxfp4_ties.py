"""Scores of a layer of experts that are equal though their bits are not: -0, which a sum too small for f32 leaves where it is negative, and +0."""
import numpy as np
import pytest

import mx_reference as mx
from vtl_amd import HipMoE, moe_mxfp4_hip
from vtl_amd.tensor import HipTensor

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]
dev = HipTensor.from_host


def normal(seed, *shape, std=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * std).astype(np.float32)


@pytest.mark.parametrize("experts,top", [(6, 1), (6, 4), (130, 2), (300, 16)])
@pytest.mark.parametrize("tokens", [1, 5, 12])
def test_zeros_of_both_signs_go_to_the_lowest_expert(experts, top, tokens):
    dim, hidden = 64, 32
    # 2^-100 times 2^-60 is below half of f32's least number: a score of -0 where the router has -2^-60, of +0 where it has 0 or 2^-60
    x = np.full((tokens, dim), 2.0 ** -100, np.float32)
    router = np.zeros((experts, dim), np.float32)
    router[:, 3] = np.random.default_rng(experts).choice([-1.0, 0.0, 1.0], experts) * 2.0 ** -60
    router[:2, 3] = [-2.0 ** -60, 0.0]
    score = mx.scores(x, router, None)
    assert (score == 0).all() and np.signbit(score[:, 0]).all() and not np.signbit(score[:, 1]).any()
    gu, dn, bias = normal(1, experts * 2 * hidden, dim), normal(2, experts * dim, hidden), normal(3, experts, dim)
    layer = HipMoE(dev(router), dev(gu).quantize_mxfp4(), dev(dn).quantize_mxfp4(), top, True, None, None, dev(bias))
    got = moe_mxfp4_hip(layer, dev(x)).cpu()
    # hidden values are products of two of 2^-100, nothing beside biases: their mean over the first experts.  Each of them with a weight that is rounded
    # twice, a product and a sum
    want = bias[:top].astype(np.float64).mean(0)
    far = (top + 4) * mx.U * np.abs(bias[:top].astype(np.float64)).mean(0)
    assert (np.abs(got - want) <= far).all(), float((np.abs(got - want) / far).max())
