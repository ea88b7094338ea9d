"""A layer of experts out of a llama-shaped GGUF file: stacked quantized matrices become one int8 layer."""
import io

import numpy as np
import pytest
import torch

from oracle import kquants as kq

import inference_rs_b200 as pkg
from inference_rs_b200 import llama_gguf as lg
from inference_rs_b200.gguf_file import Content, GgufError, Value, write

EXPERTS, FFN, HIDDEN = 3, 96, 256
DT = {"ffn_gate_exps": (kq.Q4_K, pkg.GgmlDType.Q4K, (EXPERTS, FFN, HIDDEN)), "ffn_up_exps": (kq.Q6_K, pkg.GgmlDType.Q6K, (EXPERTS, FFN, HIDDEN)),
      "ffn_down_exps": (kq.Q8_0, pkg.GgmlDType.Q8_0, (EXPERTS, HIDDEN, FFN))}


def expert_file(**changed):
    """A file with one layer; `changed` gives a tensor another shape (same number of values), or None to leave it out."""
    rng = np.random.default_rng(5)
    packed, tensors = {}, []
    for key, (kind, dtype, shape) in DT.items():
        w = (rng.standard_normal((shape[0] * shape[1], shape[2])) * 0.02).astype(np.float32)
        packed[key] = kq.quantize(kind, w).reshape(shape[0], shape[1], -1)
        if changed.get(key, shape) is not None:
            tensors.append((f"blk.4.{key}.weight", int(dtype), changed.get(key, shape), packed[key].reshape(-1)))
    buf = io.BytesIO()
    write(buf, [("general.architecture", Value.string("llama"))], tensors)
    buf.seek(0)
    return buf, Content.read(buf), packed


def test_files_without_a_whole_layer_are_refused():
    buf, content, _ = expert_file()
    with pytest.raises(GgufError, match="cannot find"):
        lg.load_experts(buf, content, 3)
    buf, content, _ = expert_file(ffn_up_exps=None)
    with pytest.raises(GgufError, match="ffn_up_exps"):
        lg.load_experts(buf, content, 4)
    buf, content, _ = expert_file(ffn_gate_exps=(EXPERTS * FFN, HIDDEN))
    with pytest.raises(GgufError, match="one matrix per expert"):
        lg.load_experts(buf, content, 4)
    buf, content, _ = expert_file(ffn_down_exps=(HIDDEN, EXPERTS, FFN))
    with pytest.raises(GgufError, match="do not make a layer"):
        lg.load_experts(buf, content, 4)


@pytest.mark.gpu
def test_a_layer_from_a_file_is_the_layer_of_its_bytes():
    buf, content, packed = expert_file()
    layer = lg.load_experts(buf, content, 4)
    tensors = [pkg.Int8Tensor.from_qtensor(*(pkg.QTensor.from_packed(packed[key][e], dtype, shape[1:]) for e in range(EXPERTS)))
               for key, (_, dtype, shape) in DT.items()]
    want = pkg.Int8Experts(*tensors)
    assert torch.equal(layer.gate_up, want.gate_up) and torch.equal(layer.gate_up_scales, want.gate_up_scales)
    assert torch.equal(layer.down.data, want.down.data) and torch.equal(layer.down.scales, want.down.scales)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(7, HIDDEN, device="cuda", generator=g).to(torch.bfloat16)
    top, ids = torch.randn(7, EXPERTS, device="cuda", generator=g).topk(2)
    y = layer(x, ids, top.softmax(1))
    assert torch.equal(y, want(x, ids, top.softmax(1)))
    # two quantizations to 8 bits away from the file's weights: 1/254 of the largest value of a row each, against rows whose values are
    # a fourth of it and more: a few percent of the output
    dense = [w.dequantize().double() for w in tensors]
    for t in range(7):
        h = sum(float(wt) * dense[2][e] @ (torch.nn.functional.silu(dense[0][e] @ x[t].double()) * (dense[1][e] @ x[t].double()))
                for e, wt in zip(ids[t].tolist(), top[t].softmax(0).tolist()))
        assert float((y[t].double() - h).norm() / h.norm()) < 0.05
