"""SiLU(gate) * up of a layer of experts from one end of f32 to the other.  The token is zeros, so gates and ups are the biases; the down product hands
hidden values on."""
import numpy as np
import pytest

import mx_reference as mx
from vtl_amd import HipMoE, moe_mxfp4_hip
from vtl_amd.tensor import HipTensor

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]
dev = HipTensor.from_host

GATES = [-3e38, -1e30, -1e20, -1e10, -5000.0, -300.0, -180.0, -150.0, -120.0, -104.0, -103.0, -100.0, -95.0, -90.0, -88.8, -88.0, -87.5, -87.0, -86.9, -86.0, -80.0, -50.0,
         -20.0, -3.0, -1.0, -0.25, -1e-3, -1e-20, 0.0, 1e-20, 1e-3, 0.25, 1.0, 3.0, 20.0, 50.0, 87.0, 90.0, 1000.0, 1e10, 1e20, 1e30]
UPS = [1.0, -3.7, 100.0, 1e-5, 1e10, -1e18, 1e25, 3e38]


def hidden_values(gate, up, tokens, weights=None):
    """What the layer makes of these gates and ups (one block of 32 hidden values each), a row of the output for each token."""
    n = gate.size
    hidden, dim = 32 * n, 32 * n        # down: output i is the first hidden value of block i
    down = np.zeros((dim, hidden), np.float32)
    down[np.arange(n), 32 * np.arange(n)] = 1.0
    zeros = np.zeros((2 * hidden, dim), np.float32)
    bias = np.concatenate([np.repeat(gate, 32), np.repeat(up, 32)]).astype(np.float32)
    layer = HipMoE(dev(np.ones((1, dim), np.float32)), dev(zeros).quantize_mxfp4(), dev(down).quantize_mxfp4(), 1, True, None, dev(bias))
    return moe_mxfp4_hip(layer, dev(np.zeros((tokens, dim), np.float32))).cpu()[:, :n]


def silu_up(gate, up):
    with np.errstate(over="ignore"):
        return gate / (1 + np.exp(-gate)) * up


@pytest.mark.parametrize("tokens", [1, 5, 12])
@pytest.mark.parametrize("up", UPS)
def test_every_gate(tokens, up):
    gate = np.array(GATES, np.float32).astype(np.float64)
    want = silu_up(gate, np.float64(np.float32(up)))
    gate, want = gate[np.abs(want) < 3e38], want[np.abs(want) < 3e38]
    got = hidden_values(gate, np.full_like(gate, up), tokens)
    # the exponential of an argument that is rounded, as is the constant in it (5/4 |gate| half steps; what the value has of them vanishes where it is 1 + a
    # small number), its own steps and those of a dozen operations, digits that stop at 2^-24 of the value; values below 2^-103 are cut off at 2^-128
    far = np.abs(want) * mx.U * (1.25 * np.minimum(np.abs(gate), 400) + 32) + 2.0 ** -127
    off = np.abs(got - want)
    assert (off <= far).all(), [(float(gate[i]), float(got[t, i]), float(want[i])) for t, i in np.argwhere(~(off <= far))[:6]]


@pytest.mark.parametrize("low,high", [(-100.0, -80.0), (-80.0, -40.0), (-40.0, -8.0), (-8.0, 8.0)])
def test_exponentials_are_those_of_the_gate(low, high):
    """Not of a gate rounded to fewer digits.  The exponential's fourth root is off by a step of the instruction's and a rounding, 3 half steps and so 12 in the
    value; the reciprocal of its sum with 1 by 9, the products by 7, digits by 1, sums by 5."""
    gate = np.linspace(low, high, 1500).astype(np.float32).astype(np.float64)
    up = np.float64(np.float32(1.7))
    want = silu_up(gate, up)
    got = hidden_values(gate, np.full_like(gate, up), 1)[0]
    off = np.abs(got - want) / (np.abs(want) * mx.U + 2.0 ** -127)
    assert (off <= 40).all(), (float(off.max()), float(gate[off.argmax()]))
