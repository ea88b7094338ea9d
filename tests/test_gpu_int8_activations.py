"""The gated activations of a layer of experts in f32, relative to their size over the whole range.

A layer with one hidden value that is not zero: x = (v, 1), gate and up read v and 1, down passes the hidden value on. Its integer is 127
with the scale |h| / 127, so that the output is 127^2 times that scale and no quantization is in the way. In units of 2^-24, relative:
expf 4 (two units of the last place), the sum 1 + exp and what the exponential's error does to it 3, the reciprocal 2, two products 2; the
product with up 1, the scale 1, its product with the integer sum 1: 14. tanh-GELU is x times the sigmoid of t = 2 u(x), off by 7 units
(five operations, two constants), and the exponential of it by 7 |t|. Below t = -87.3 the exponential is subnormal: two steps of 2^-149,
times |x * up|; a scale below the normal range is off by half a step, 2^-150, times 127^2.
"""
import pytest
import torch

import inference_rs_b200 as pkg
from inference_rs_b200 import ops
from gpu_util import assert_device_ok

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def one_value_layer(act, up_scale, down_scale=1.0):
    gate, up, down = torch.zeros(2, 8, 16, dtype=torch.int8), torch.zeros(2, 8, 16, dtype=torch.int8), torch.zeros(2, 16, 8, dtype=torch.int8)
    gate[:, 0, 0], up[:, 0, 1], down[:, 0, 0] = 127, 127, 127
    scales = lambda n, s: torch.full((2, n), s, device="cuda")
    parts = [pkg.Int8Tensor(d.cuda(), scales(d.shape[1], s)) for d, s in ((gate, 1 / 127), (up, up_scale), (down, down_scale))]
    return pkg.Int8Experts(*parts, activation=act), parts


@pytest.mark.parametrize("tokens", [4, 600])  # the products for few tokens and those on the tensor cores
@pytest.mark.parametrize("up_scale", [1e-2, 1e20])
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_activations_are_right_relative_to_their_size(act, up_scale, tokens):
    layer, (gate, up, _) = one_value_layer(act, up_scale)
    v = torch.cat([torch.linspace(-104, 30, 500), torch.linspace(-2, 2, 100)]).cuda()
    x = torch.zeros(600, 16, device="cuda")
    x[:, 0], x[:, 1] = v, 1
    ids, weights = (torch.arange(600, device="cuda") % 2)[:, None], torch.ones(600, 1, device="cuda")
    got = torch.cat([layer(x[i:i + tokens], ids[i:i + tokens], weights[i:i + tokens]) for i in range(0, 600, tokens)])
    xq, xs = ops.int8_quantize(x)
    g, u = (ops.int8_gemm(xq, xs, w.data[0], w.scales[0], 16, torch.float32)[:, 0].double() for w in (gate, up))
    assert g.min() < -100 and g.max() > 25
    t = 2 * (2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3) if act == "gelu" else g
    factor = torch.ones_like(g) if act == "sigmoid" else g
    # 1 / (1 + exp(-t)) in 64 bits, without losing the small ones
    want = 127 * factor * u * torch.where(t < 0, torch.exp(t.clamp(max=0)), 1.0) / (1 + torch.exp(-t.abs()))
    tol = (14 + (7 * t.abs() if act == "gelu" else 0)) * U * want.abs() + 127 * (factor * u).abs() * 2.0 ** -148 + 127 ** 2 * 2.0 ** -150
    off = (got[:, 0].double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{int(bad.sum())} off, first at {g[bad][0]}: {got[:, 0][bad][0]} for {want[bad][0]}, {off[bad][0] / (U * want[bad][0].abs())} units"
    assert not got[:, 1:].any()
    assert_device_ok()


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "relu", "gelu_erf"])
def test_gates_as_large_as_f32_holds(act):
    """The activations' limits, without a NaN: 0 below and x above (sigmoid: 1). Relative 14 units as above, doubled for all of them.

    Not so the first and the last: a product is (sum * x_scale) * w_scale, and 127^2 * 3e38 / 127 = 3.8e40 passes f32's range before the
    weights' scale brings it back. Gate and up are infinite there by definition, up times 0 or infinity is a NaN or an infinity, and the
    row with it in is NaN."""
    layer, (gate, up, _) = one_value_layer(act, 1e-41, 1 / 127)
    x = torch.zeros(6, 16, device="cuda")
    x[:, 0] = torch.tensor([-3e38, -1e25, -1e12, 1e12, 1e25, 3e38], device="cuda")
    x[:, 1] = x[:, 0].abs()
    got = layer(x, torch.zeros(6, 1, dtype=torch.int64, device="cuda"), torch.ones(6, 1, device="cuda"))[:, 0].double()
    xq, xs = ops.int8_quantize(x)
    g, u = (ops.int8_gemm(xq, xs, w.data[0], w.scales[0], 16, torch.float32)[:, 0].double() for w in (gate, up))
    assert g[[0, 5]].isinf().all() and u[[0, 5]].isinf().all() and got[[0, 5]].isnan().all()
    want = u[3:5] * (1 if act == "sigmoid" else g[3:5])
    assert not got[1:3].any()
    assert ((got[3:5] - want).abs() <= 28 * U * want + 127 * 2.0 ** -150).all()
