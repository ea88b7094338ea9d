"""Weights as 8-bit integers with a scale per output channel, and what multiplies them: `Int8MatMul`, the counterpart of `QMatMul`, and
`Int8Experts`, a layer of gated experts.

Activations become int8 too, with a scale per token, on the way into a product; the product itself is the exact integer sum, scaled in
f32. Checkpoints in this form are used as they are (`Int8Tensor(data, scales)`); GGUF weights are converted on the device
(`Int8Tensor.from_qtensor`): Q8_0 keeps about its size, and prompts then run at the tensor cores' 8-bit rate with nothing to expand.
"""
from __future__ import annotations

import torch

from . import kernel_library as kl
from . import ops
from .dtypes import pad
from .qmatmul import QTensor


def _no_grad_through(*tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError("int8 products have no gradient: call them under torch.no_grad(), or on detached tensors")
    if ops.has_tangent(*tensors):
        raise ValueError("int8 products have no gradient in forward mode either: call them on primals")


class Int8Tensor:
    """int8 rows with a scale each: a matrix [n, k], or one for each expert [experts, n, k]. `data` holds the rows padded to 16 bytes
    with zeros, `scales` [n] or [experts, n] their scales, constants to autograd; row i stands for data[i] * scales[i]."""

    def __init__(self, data: torch.Tensor, scales: torch.Tensor):
        if data.dtype != torch.int8 or scales.dtype != torch.float32:
            raise TypeError(f"expected int8 values and f32 scales, got {data.dtype} and {scales.dtype}")
        if data.dim() not in (2, 3) or tuple(scales.shape) != tuple(data.shape[:-1]):
            raise ValueError(f"values {tuple(data.shape)} and scales {tuple(scales.shape)}: expected [n, k] and [n], or with experts in front")
        if data.device != scales.device:
            raise ValueError(f"values on {data.device}, scales on {scales.device}")
        self.shape = tuple(data.shape)
        k, kp = data.shape[-1], pad(data.shape[-1], ops.INT8_ROW_ALIGN)
        if kp != k or not data.is_contiguous() or data.data_ptr() % 16:
            padded = data.new_zeros(*data.shape[:-1], kp)
            padded[..., :k] = data
            data = padded
        self.data, self.scales = data, scales.detach().contiguous()

    @classmethod
    def _of_rows(cls, q: torch.Tensor, scales: torch.Tensor, shape: tuple[int, ...]) -> "Int8Tensor":
        self = cls.__new__(cls)
        self.shape, self.data, self.scales = shape, q, scales
        if len(shape) == 3:
            self.data, self.scales = q.view(*shape[:-1], q.shape[-1]), scales.view(shape[:-1])
        return self

    @classmethod
    def quantize(cls, src: torch.Tensor) -> "Int8Tensor":
        """A weight [n, k] or [experts, n, k] of f32, f16 or bf16, each row with the scale max|row| / 127; brought to the GPU where it is
        not there."""
        if src.dim() not in (2, 3):
            raise ValueError(f"quantize takes a matrix, or one per expert, got {tuple(src.shape)}")
        if not src.is_cuda:
            src = src.cuda()
        return cls._of_rows(*ops.int8_quantize(src if src.dim() == 2 else src.detach().reshape(-1, src.shape[-1])), tuple(src.shape))

    @classmethod
    def from_qtensor(cls, *weights: QTensor) -> "Int8Tensor":
        """GGUF weights, quantized again with one scale per row: [n, k] of one matrix, [experts, n, k] of several."""
        if not weights or any(w.shape != weights[0].shape for w in weights):
            raise ValueError(f"expected matrices of one shape, got {[w.shape for w in weights]}")
        with torch.cuda.device(ops._one_device(*(w.data for w in weights))):  # QTensor launches on the current device
            parts = [ops.int8_quantize(w.dequantize(torch.float32)) for w in weights]
        if len(parts) == 1:
            return cls._of_rows(*parts[0], weights[0].shape)
        return cls._of_rows(torch.cat([q for q, _ in parts]), torch.cat([s for _, s in parts]), (len(parts), *weights[0].shape))

    def dequantize(self, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values as a dense tensor of this shape."""
        out = kl.host().int8_dequantize(self.data, self.scales, self.shape[-1], ops.elem_of(out_dtype))
        if out is not None:
            return out
        return ops.int8_dequantize(self.data.view(-1, self.data.shape[-1]), self.scales.view(-1), self.shape[-1], out_dtype).view(self.shape)

    @property
    def device(self) -> torch.device:
        return self.data.device


class Int8MatMul:
    """`y = x @ W^T` for an int8 `W` [n, k]; x `[..., k]` contiguous -> y `[..., n]` in x's type, plus a bias where there is one."""

    def __init__(self, w: Int8Tensor, b: torch.Tensor | None = None):
        if len(w.shape) != 2:
            raise ValueError(f"expected a matrix, got {w.shape}")
        self.w, self.b = w, b

    @classmethod
    def from_qtensor(cls, q: QTensor, bias: torch.Tensor | None = None) -> "Int8MatMul":
        return cls(Int8Tensor.from_qtensor(q), bias)

    def forward(self, xs: torch.Tensor) -> torch.Tensor:
        n, k = self.w.shape
        y = kl.host().int8_forward(self.w.data, self.w.scales, n, k, xs)
        if y is None:
            y = self._forward(xs, n, k)
        return y if self.b is None else y + self.b.to(y.dtype)

    __call__ = forward

    def _forward(self, xs: torch.Tensor, n: int, k: int) -> torch.Tensor:
        """What the native path declines as it stands: errors among them."""
        if xs.dim() < 2:
            raise ValueError(f"input tensor has only one dimension {tuple(xs.shape)}")
        if not xs.is_contiguous():
            raise ValueError(f"input tensor is not contiguous {tuple(xs.shape)}")
        if xs.shape[-1] != k:
            raise ValueError(f"input tensor {tuple(xs.shape)} incompatible with {(n, k)}")
        if xs.device != self.w.device:
            raise ValueError(f"input on {xs.device}, weights on {self.w.device}")
        _no_grad_through(xs)
        return ops.int8_matmul(xs.view(-1, k), self.w.data, self.w.scales).view(*xs.shape[:-1], n)


class Int8Experts:
    """A layer of gated experts, `down_e(act(gate_e(x)) * up_e(x))`, on int8 weights: gate and up [experts, ffn, hidden], down [experts,
    hidden, ffn]. Holds gate and up as one matrix per expert, 8 rows of the one and 8 of the other in turn, so that one product forms
    both and multiplies them out."""

    def __init__(self, gate: Int8Tensor, up: Int8Tensor, down: Int8Tensor, activation: str = "silu"):
        if len(gate.shape) != 3 or gate.shape != up.shape or down.shape != (gate.shape[0], gate.shape[2], gate.shape[1]):
            raise ValueError(f"gate {gate.shape}, up {up.shape}, down {down.shape}: expected [experts, ffn, hidden] twice and [experts, hidden, ffn]")
        if activation not in ops.GLU_ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}; one of {sorted(ops.GLU_ACTIVATIONS)}")
        if not gate.device == up.device == down.device:
            raise ValueError(f"gate on {gate.device}, up on {up.device}, down on {down.device}")
        self.experts, self.ffn, self.hidden = gate.shape
        self.activation, self.down = activation, down
        p = pad(self.ffn, 8)
        data = gate.data.new_zeros(self.experts, p // 8, 2, 8, gate.data.shape[-1])
        scales = gate.scales.new_zeros(self.experts, p // 8, 2, 8)
        for i, part in enumerate((gate, up)):
            rows = part.data if p == self.ffn else torch.nn.functional.pad(part.data, (0, 0, 0, p - self.ffn))
            data[:, :, i] = rows.view(self.experts, p // 8, 8, -1)
            scales[:, :, i] = torch.nn.functional.pad(part.scales, (0, p - self.ffn)).view(self.experts, p // 8, 8)
        self.gate_up, self.gate_up_scales = data.view(self.experts, 2 * p, -1), scales.view(self.experts, 2 * p)

    def forward(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """x [..., hidden]; ids [..., slots] (int32 or int64) names each token's experts, weights [..., slots] their weights. A slot
        whose id is not one of 0..experts - 1 counts for nothing. -> [..., hidden] in x's type."""
        out = kl.host().int8_experts(x, ids, weights, self.gate_up, self.gate_up_scales, self.down.data, self.down.scales, self.ffn,
                                     ops.GLU_ACTIVATIONS[self.activation])
        if out is not None:
            return out
        if x.dim() < 2 or x.shape[-1] != self.hidden or ids.shape != weights.shape or tuple(ids.shape[:-1]) != tuple(x.shape[:-1]):
            raise ValueError(f"tokens {tuple(x.shape)}, ids {tuple(ids.shape)}, weights {tuple(weights.shape)} for a layer of width {self.hidden}")
        _no_grad_through(x, weights)
        topk = ids.shape[-1]
        if x.numel() == 0 or topk == 0:
            return torch.zeros_like(x, memory_format=torch.contiguous_format)
        out = ops.int8_experts(x.reshape(-1, self.hidden), ids.reshape(-1, topk).contiguous(),
                               weights.to(torch.float32).reshape(-1, topk).contiguous(), self.gate_up, self.gate_up_scales, self.down.data,
                               self.down.scales, self.ffn, self.activation)
        return out.view(x.shape)

    __call__ = forward
