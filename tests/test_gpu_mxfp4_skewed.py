"""Layers of experts whose router sends all tokens to the same few experts: as many pairs of an expert as there are tokens, in every way that a layer is launched."""
import numpy as np
import pytest

import mx_reference as mx
from test_gpu_mxfp4 import LargeLayer, check_layer, normal

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


@pytest.mark.parametrize("experts,dim,hidden,top,tokens", [
    (64, 96, 1000, 6, 40), (64, 64, 1030, 16, 8),       # many hidden values: one wave along K
    (96, 1028, 1450, 5, 17), (96, 1028, 1450, 5, 64),   # 128 MB of weights: past the caches
    (8, 100, 2600, 4, 40), (8, 40, 4112, 4, 64),        # four pairs of an expert and more by chance
    (12, 264, 72, 3, 64), (12, 264, 72, 3, 7)])         # few
@pytest.mark.parametrize("one_more", [False, True])
def test_the_same_experts_for_all(guard_bands, experts, dim, hidden, top, tokens, one_more):
    l = LargeLayer(experts, dim, hidden, top, True, seed=experts)
    rng = np.random.default_rng(tokens)
    favoured = rng.permutation(experts)[:top]
    l.biases[0][favoured] += 50.0
    l.hip()
    x = normal(tokens, tokens, dim)
    if one_more:        # but for one token, which has a mind of its own
        l.biases[0][:] = 0.0
        x[:, 0] = 10.0
        l.router[favoured, 0] += 5.0
        x[tokens // 2, 0] = -10.0
        l.hip()
    chosen = mx.choose(mx.scores(x, l.router, l.biases[0]), top)
    same = (np.sort(chosen, 1) == np.sort(favoured)).all(1)
    assert same.sum() == tokens - one_more
    check_layer(l, x)
