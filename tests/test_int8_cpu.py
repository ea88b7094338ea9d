"""What the int8 and routing classes refuse, and how they lay weights out: no GPU needed."""
import pytest
import torch

import inference_rs_b200 as pkg
from inference_rs_b200 import ops


def int8_tensor(*shape):
    return pkg.Int8Tensor(torch.randint(-127, 128, shape, dtype=torch.int8), torch.rand(shape[:-1]))


def test_rows_are_padded_with_zeros():
    data = torch.randint(-127, 128, (5, 37), dtype=torch.int8)
    t = pkg.Int8Tensor(data, torch.rand(5))
    assert t.shape == (5, 37) and t.data.shape == (5, 48)
    assert torch.equal(t.data[:, :37], data) and not t.data[:, 37:].any()
    whole = torch.zeros(3, 32, dtype=torch.int8)
    assert pkg.Int8Tensor(whole, torch.rand(3)).data is whole  # used as it is
    strided = torch.zeros(3, 64, dtype=torch.int8)[:, :32]
    assert pkg.Int8Tensor(strided, torch.rand(3)).data.is_contiguous()


@pytest.mark.parametrize("ffn", [8, 13, 24])
def test_gate_and_up_alternate_in_eights(ffn):
    gate, up, down = int8_tensor(2, ffn, 32), int8_tensor(2, ffn, 32), int8_tensor(2, 32, ffn)
    layer = pkg.Int8Experts(gate, up, down)
    p = (ffn + 7) // 8 * 8
    assert layer.gate_up.shape == (2, 2 * p, 32) and layer.gate_up_scales.shape == (2, 2 * p)
    for i in range(p):
        at = 16 * (i // 8) + i % 8
        for part, row in ((gate, at), (up, at + 8)):
            want = part.data[:, i] if i < ffn else torch.zeros(2, 32, dtype=torch.int8)
            assert torch.equal(layer.gate_up[:, row], want)
            assert torch.equal(layer.gate_up_scales[:, row], part.scales[:, i] if i < ffn else torch.zeros(2))


def test_refusals():
    with pytest.raises(TypeError, match="int8 values and f32 scales"):
        pkg.Int8Tensor(torch.zeros(4, 16), torch.zeros(4))
    with pytest.raises(ValueError, match="scales"):
        pkg.Int8Tensor(torch.zeros(4, 16, dtype=torch.int8), torch.zeros(5))
    with pytest.raises(ValueError, match="matrix"):
        pkg.Int8MatMul(int8_tensor(2, 8, 16))
    with pytest.raises(ValueError, match="one shape"):
        pkg.Int8Tensor.from_qtensor()
    w = pkg.Int8MatMul(int8_tensor(8, 16))
    for x, match in ((torch.zeros(16), "one dimension"), (torch.zeros(16, 2).t(), "not contiguous"), (torch.zeros(2, 15), "incompatible"),
                     (torch.zeros(2, 16), "CUDA"), (torch.zeros(2, 16, requires_grad=True), "no gradient")):
        with pytest.raises(ValueError, match=match):
            w(x)
    with pytest.raises(TypeError, match="f32, f16 or bf16"):
        w(torch.zeros(2, 16, dtype=torch.float64))
    with pytest.raises(ValueError, match="expected"):
        pkg.Int8Experts(int8_tensor(2, 8, 16), int8_tensor(2, 8, 16), int8_tensor(2, 8, 16))
    with pytest.raises(ValueError, match="unknown activation"):
        pkg.Int8Experts(int8_tensor(2, 8, 16), int8_tensor(2, 8, 16), int8_tensor(2, 16, 8), "swish")
    layer = pkg.Int8Experts(int8_tensor(2, 8, 16), int8_tensor(2, 8, 16), int8_tensor(2, 16, 8))
    ids, weights = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, 2)
    with pytest.raises(ValueError, match="layer of width 16"):
        layer(torch.zeros(3, 15), ids, weights)
    with pytest.raises(ValueError, match="layer of width 16"):
        layer(torch.zeros(4, 16), ids, weights)
    with pytest.raises(ValueError, match="CUDA"):
        layer(torch.zeros(3, 16), ids, weights)
    with pytest.raises(ValueError, match="no gradient"):
        layer(torch.zeros(3, 16), ids, weights.requires_grad_())


def test_routing_refusals():
    with pytest.raises(ValueError, match="a dimension for the tokens"):
        pkg.TokenRouting(torch.zeros(3, dtype=torch.int32), 4)
    with pytest.raises(TypeError, match="int32 or int64"):
        pkg.TokenRouting(torch.zeros(3, 2), 4)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.TokenRouting(torch.zeros(3, 2, dtype=torch.int64), 4)
    with pytest.raises(TypeError, match="f32, f16 or bf16"):
        ops.route_dispatch(torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(5, dtype=torch.int32))


def test_the_library_refuses_what_it_cannot_take():
    lib = pkg.library()
    err = lambda: lib.b200q_last_error().decode()
    assert lib.b200q_int8_quantize(7, 1, 16, 16, 16, 16, 1, 16, None) == -1
    assert lib.b200q_int8_quantize(0, 16, 16, 16, 24, 16, 1, 16, None) == -2 and "16" in err()
    assert lib.b200q_int8_quantize(0, 16, 16, 16, 16, 16, 1, 131072, None) == -1 and "131071" in err()
    assert lib.b200q_int8_quantize(0, None, 16, None, 16, None, 0, 16, None) == 0
    assert lib.b200q_int8_matmul(0, 16, 16, 16, 16, 4, 4, 16, 16, 16, 4, 256, 8, None) == -4
    assert lib.b200q_int8_matmul(0, 16, 16, 16, 16, 4, 4, 16, 16, 16, 4, 257, 1 << 20, None) == -2
    assert lib.b200q_int8_gemm(0, 16, 16, 16, 16, 16, 4, 4, 16, 16, 16, 4, None, 2, None) == -2 and "offsets" in err()
    assert lib.b200q_route_sort(16, 2, 4, 4, 16, 16, 16, None) == -1
    assert lib.b200q_route_sort(16, 4, 4, 1025, 16, 16, 16, None) == -1 and "1024" in err()
    assert lib.b200q_int8_experts(2, 9, 16, 16, 16, 4, 16, 16, 16, 16, 16, 16, 1, 4, 2, 16, 16, 256, 1 << 20, None) == -2
    assert lib.b200q_int8_experts(2, 0, 16, 16, 16, 4, 16, 16, 16, 16, 16, 16, 1, 4, 2, 16, 16, 256, 16, None) == -4
    assert lib.b200q_int8_matmul_workspace_bytes(3, 37) >= 3 * 48 + 12
    assert lib.b200q_int8_experts_workspace_bytes(2, 0, 2, 4, 16, 16) == 0
    most = 2 ** 31 - 1  # columns: a kernel's step over them would pass 32 bits
    assert lib.b200q_route_dispatch(0, 16, most, 16, 16, 4, 16, 1, 2, most, None) == -2
    assert lib.b200q_route_combine(0, 0, 16, most, 16, 16, 16, 1, 2, most, None) == -2
    assert lib.b200q_route_combine_grad(0, 0, 16, most, 16, most, 16, 16, 4, 16, 16, 16, 1, 2, most, None) == -2


def test_scales_are_constants():
    scales = torch.rand(4, requires_grad=True)
    assert not pkg.Int8Tensor(torch.zeros(4, 16, dtype=torch.int8), scales).scales.requires_grad
