"""Linear layers in 8-bit integers: the projections of a language model that
answers over retrieved vectors.

``Int8Linear`` keeps a layer's weights as codes of -127 to 127 with a scale for
each output channel.  A call quantises each token by its largest magnitude,
multiplies the codes on the int8 matrix cores into exact 32-bit sums and scales
them back.  As in ``kvcache``, tensors are torch tensors on the context's GPU,
calls are queued on torch's current stream, do not wait, and record no
gradients.  The reference's counterparts are its matrixMultiply
(Acceleration/MetalAccelerationEngine.swift:209-229) and scalar quantizer.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib
from ._lib import VSKError
from .engine import Context
from .kvcache import _TYPES, _stream, _tensor

# (vsk_int8_rows as bytes, as kvcache's structures)
_ROWS = struct.Struct("@QQqqqQqii")
assert _ROWS.size == ctypes.sizeof(_lib.vsk_int8_rows)
_MOST = 131072


def _dense(x):
    """x with a dense last dimension, or a copy."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


class Int8Linear:
    """y = x W^T + b with W (outputs x inputs) in 8 bits.

    ``weight`` (f32, f16 or bf16) is quantised, each channel by its largest
    magnitude / 127; a channel that holds an infinity or NaN gives NaN.
    ``bias``: a value a channel.  At most 131,072 inputs, whose sums fit 32
    bits."""

    def __init__(self, ctx: Context, weight, bias=None):
        _tensor(ctx.device, weight, "weight", None, 2)
        if weight.dtype not in _TYPES:
            raise VSKError(-8, f"{weight.dtype} is not supported")
        self._hold(ctx, weight, torch.empty(weight.shape[0], dtype=torch.float32,
                                            device=weight.device), bias, _TYPES[weight.dtype])

    @classmethod
    def over(cls, ctx: Context, codes, scales, bias=None) -> "Int8Linear":
        """A layer of codes (int8, outputs x inputs) and scales (f32, a value a
        channel), which are copied."""
        _tensor(ctx.device, codes, "codes", torch.int8, 2)
        _tensor(ctx.device, scales, "scales", torch.float32, 1)
        if scales.shape[0] != codes.shape[0]:
            raise VSKError(-4, f"{scales.shape[0]} scales for {codes.shape[0]} channels")
        self = cls.__new__(cls)
        self._hold(ctx, codes, scales.clone(memory_format=torch.contiguous_format), bias, 3)
        return self

    def _hold(self, ctx, rows, scales, bias, dtype):
        self.ctx, (self.outputs, self.inputs) = ctx, rows.shape
        if not self.outputs or not self.inputs:
            raise VSKError(-3, "an empty layer")
        if self.inputs > _MOST or self.outputs >= 1 << 31:
            raise VSKError(-9, f"{self.outputs} x {self.inputs}: at most {_MOST:,} inputs and "
                           "2^31 - 1 outputs")
        if bias is not None:
            _tensor(ctx.device, bias, "bias", None, 1)
            if bias.shape[0] != self.outputs:
                raise VSKError(-4, f"{bias.shape[0]} bias values for {self.outputs} channels")
            if bias.dtype not in _TYPES:
                raise VSKError(-8, f"{bias.dtype} is not supported")
            bias = bias.detach().to(torch.float32, copy=True).contiguous()
        need = ctx.lib.vsk_int8_packed_bytes(self.outputs, self.inputs)
        self.scales, self.bias, self.device = scales, bias, rows.device
        self.packed = torch.empty(need, dtype=torch.uint8, device=rows.device)
        w = _lib.vsk_int8_weight(self.packed.data_ptr(), scales.data_ptr(),
                                 bias.data_ptr() if bias is not None else None, self.outputs,
                                 self.inputs)
        self._weight, self._ref = w, ctypes.byref(w)
        rows = _dense(rows.detach())
        ctx.check(ctx.lib.vsk_int8_pack(ctx.handle, _stream(ctx.device), dtype, rows.data_ptr(),
                                        rows.stride(0), self._ref))

    def codes(self):
        """The codes, outputs x inputs (a copy, in their own order)."""
        x = self.packed.view(torch.int8).view(-(-self.outputs // 32), -1, 2, 32, 16)
        return x.permute(0, 3, 1, 2, 4).flatten(2, 4).flatten(0, 1)[:self.outputs, :self.inputs]

    def __call__(self, x, dtype=None):
        """x (... x inputs; f32, f16 or bf16) to ... x outputs of ``dtype``
        (default: x's).  Each token's codes are x * (127 / largest), rounded to
        even in 32 bits, with the scale largest / 127; a token that holds an
        infinity or NaN gets NaN."""
        ctx = self.ctx
        _tensor(ctx.device, x, "x")
        if x.dtype not in _TYPES:
            raise VSKError(-8, f"{x.dtype} is not supported")
        if x.dim() < 1 or x.shape[-1] != self.inputs:
            raise VSKError(-4, f"x is {tuple(x.shape)}: the layer has {self.inputs} inputs")
        dtype = x.dtype if dtype is None else dtype
        if dtype not in _TYPES:
            raise VSKError(-8, f"{dtype} is not supported")
        rows = _dense(x if x.dim() == 2 else x.reshape(-1, self.inputs))
        tokens, lib = rows.shape[0], ctx.lib
        out = rows.new_empty((tokens, self.outputs), dtype=dtype)
        shaped = out if x.dim() == 2 else out.view(x.shape[:-1] + (self.outputs,))
        if not tokens:
            return shaped
        if tokens >= 1 << 31:
            raise VSKError(-9, f"{tokens} tokens: at most 2^31 - 1")
        need = lib.vsk_int8_linear_workspace(self._ref, tokens)
        work = rows.new_empty(need, dtype=torch.uint8) if need else None
        status = lib.vsk_int8_linear(
            ctx.handle, _stream(ctx.device), self._ref,
            _ROWS.pack(rows.data_ptr(), out.data_ptr(), rows.stride(0), self.outputs, tokens,
                       work.data_ptr() if need else 0, need, _TYPES[x.dtype], _TYPES[dtype]))
        if status:
            ctx.check(status)
        return shaped
