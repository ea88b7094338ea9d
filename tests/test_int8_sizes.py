"""Sizes that 32 bits do not hold are refused by name, not cut down to what they leave in 32 bits: shapes without memory, no GPU needed."""
import pytest
import torch

import inference_rs_b200 as pkg
from inference_rs_b200 import ops

BIG = 2 ** 32 + 16  # its low 32 bits are a size that would be taken


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("name,call", [
    ("int8_quantize", lambda: ops.int8_quantize(meta(1, BIG))),
    ("int8_dequantize", lambda: ops.int8_dequantize(meta(1, BIG, dtype=torch.int8), meta(1, dtype=torch.float32), BIG)),
    ("int8_gemm", lambda: ops.int8_gemm(meta(BIG, 16, dtype=torch.int8), meta(BIG), meta(4, 16, dtype=torch.int8), meta(4), 16, torch.float32)),
    ("int8_gemm", lambda: ops.int8_gemm(meta(2, 16, dtype=torch.int8), meta(2), meta(BIG, 16, dtype=torch.int8), meta(BIG), 16, torch.float32)),
    ("int8_matmul", lambda: ops.int8_matmul(meta(BIG, 1), meta(4, 16, dtype=torch.int8), meta(4))),
    ("int8_matmul", lambda: ops.int8_matmul(meta(1, 1), meta(BIG, 16, dtype=torch.int8), meta(BIG))),
    ("route_sort", lambda: pkg.TokenRouting(meta(BIG // 2, 2, dtype=torch.int32), 4)),
    ("route_sort", lambda: pkg.TokenRouting(meta(3, 2, dtype=torch.int32), BIG)),
    ("route_dispatch", lambda: ops.route_dispatch(meta(1, BIG), meta(1, 2, dtype=torch.int32), meta(5, dtype=torch.int32))),
    ("route_combine", lambda: ops.route_combine(meta(2, BIG), meta(1, 2, dtype=torch.int32), None, torch.bfloat16)),
    ("route_combine_grad", lambda: ops.route_combine_grad(meta(1, BIG), meta(2, BIG), meta(1, 2, dtype=torch.int32), meta(5, dtype=torch.int32), meta(1, 2))),
    ("int8_experts", lambda: ops.int8_experts(meta(BIG, 16), meta(BIG, 1, dtype=torch.int32), meta(BIG, 1), meta(2, 16, 16, dtype=torch.int8), meta(2, 16),
                                              meta(2, 16, 16, dtype=torch.int8), meta(2, 16), 8)),
])
def test_sizes_beyond_32_bits(name, call):
    with pytest.raises(ValueError, match=f"{name}: a size of .* does not fit 32 bits"):
        call()

