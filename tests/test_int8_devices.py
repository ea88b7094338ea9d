"""Weights on another GPU than the current one, shown with stand-ins for the devices: no GPU needed."""
from contextlib import contextmanager
from types import SimpleNamespace

import pytest
import torch

import inference_rs_b200 as pkg
from inference_rs_b200 import ops


def weight(device, calls, current):
    """A QTensor that notes which device is current when it is expanded."""
    data = SimpleNamespace(is_cuda=device.type == "cuda", device=device)
    return SimpleNamespace(shape=(4, 32), data=data, device=device, dequantize=lambda dtype: calls.append(current[-1]) or torch.zeros(4, 32))


def test_gguf_weights_are_expanded_on_their_own_device(monkeypatch):
    calls, current = [], [torch.device("cuda", 0)]

    @contextmanager
    def device(d):
        current.append(d)
        yield
        current.pop()

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ops, "int8_quantize", lambda x: (torch.zeros(4, 32, dtype=torch.int8), torch.ones(4)))
    there = torch.device("cuda", 1)
    for count in (1, 3):
        calls.clear()
        t = pkg.Int8Tensor.from_qtensor(*(weight(there, calls, current) for _ in range(count)))
        assert calls == [there] * count and len(current) == 1
        assert t.shape == ((4, 32) if count == 1 else (3, 4, 32))
    with pytest.raises(ValueError, match="tensors on"):
        pkg.Int8Tensor.from_qtensor(weight(there, calls, current), weight(torch.device("cuda", 0), calls, current))
    with pytest.raises(ValueError, match="CUDA"):
        pkg.Int8Tensor.from_qtensor(weight(torch.device("cpu"), calls, current))
