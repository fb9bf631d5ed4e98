"""8-bit rows with a scale each, and the linear layer over them (no reference counterpart: the
serving path of a decoder whose projections run on 8-bit integer tensor cores).

    rows, h = add_rms_norm_int8(x, h, norm.weight)   # norm in front of a projection
    y = int8_linear(rows, weight_rows)               # weight_rows = quant_int8(linear.weight)
    down = int8_linear(swiglu_int8(gate_up), down_rows)

A row is q[k] = round(v[k] / scale), scale = max|v| times fp32's 1/127, the same numbers as a
division in fp32 gives: symmetric, one scale per token for activations and one per output channel
for weights.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import ops


class Int8Rows:
    """int8 rows q [..., K] and their float32 scales [...]; row r stands for q[r] * scale[r].

    The quantisers start each row at a multiple of 16 bytes (q is then not contiguous where K is
    no multiple of 16), which lets int8_linear read them in place."""

    __slots__ = ("q", "scale")

    def __init__(self, q, scale):
        self.q, self.scale = q, scale

    @property
    def shape(self):
        return self.q.shape

    def dequant(self, dtype=torch.bfloat16):
        """The values the rows stand for."""
        return ops.dequant_int8(self.q, self.scale, dtype)


def quant_int8(x) -> Int8Rows:
    """x [..., K] (fp32 or bf16) as 8-bit rows."""
    return Int8Rows(*ops.quant_int8(x))


def add_rms_norm_int8(x, residual=None, weight=None, eps=1e-5):
    """(rows, h): add_rms_norm's y as 8-bit rows, quantised from fp32, and h (not differentiable)."""
    q, scale, h = ops.rms_norm_int8(x, residual, weight, eps)
    return Int8Rows(q, scale), h


def swiglu_int8(gate_up) -> Int8Rows:
    """silu(gate) * up of gate_up [..., 2 F] = [gate | up] as 8-bit rows [..., F]."""
    return Int8Rows(*ops.swiglu_int8(gate_up))


def int8_linear(x: Int8Rows, w: Int8Rows, bias=None, dtype=torch.bfloat16):
    """x [..., K] times w [N, K] transposed, scaled, plus bias [N] float32 -> [..., N] of dtype.

    The integer sums are exact; the scales and the bias are applied in fp32."""
    return ops.int8_linear(x.q, x.scale, w.q, w.scale, bias, dtype)


class Int8Linear(nn.Module):
    """A linear layer over 8-bit rows: weight rows and scales are buffers (inference only).

    forward takes Int8Rows, or a float tensor which it quantises first.  The weight rows are held
    padded to a multiple of 16 bytes, and the scales stay float32 when the module's type changes."""

    def __init__(self, weight, bias=None, dtype=torch.bfloat16):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        self.dtype = dtype
        rows = quant_int8(weight.detach())
        q = rows.q
        if self.in_features % 16:
            q = nn.functional.pad(q, (0, -self.in_features % 16))
        self.register_buffer("q", q)
        self.register_buffer("scale", rows.scale)
        self.register_buffer("bias", None if bias is None else bias.detach().float().contiguous())

    @classmethod
    def from_linear(cls, linear: nn.Linear):
        return cls(linear.weight, linear.bias, linear.weight.dtype)

    def _apply(self, fn, *args, **kwargs):
        held = {"scale": self.scale, "bias": self.bias}
        super()._apply(fn, *args, **kwargs)
        for name, t in held.items():
            moved = getattr(self, name)
            if t is not None and moved.dtype != t.dtype:
                setattr(self, name, t.to(moved.device))
        return self

    def forward(self, x):
        rows = x if isinstance(x, Int8Rows) else quant_int8(x)
        q = self.q if self.q.shape[1] == self.in_features else self.q[:, :self.in_features]
        return int8_linear(rows, Int8Rows(q, self.scale), self.bias, self.dtype)
