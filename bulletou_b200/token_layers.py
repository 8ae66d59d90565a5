"""Operators of a token model over feature rows: a learned LayerStack router.

The reference chooses the LayerStack of a position by a fixed rule
(ShogiSfnnLayerStackBucketKind::bucket_from_board, game/outputs.rs:1227-1231);
these operators are what a router that learns the choice is made of (see
``StackRouter``): lookup with scaling and its gradient, dropout, routing with a
balance loss, and the 8-bit product that evaluates a dense layer.

Every operand is a matrix in device memory: a ``DeviceMatrix`` over the
library's buffers, a buffer itself (one row), or a CUDA tensor of torch with
one or two dimensions whose last one is contiguous.  Calls go to the context's
stream and return at once: a torch tensor that was written on another stream
has to be ordered by an event, as with any stream (``bo.Context(device,
stream=torch.cuda.current_stream().cuda_stream)`` shares torch's).
"""
from __future__ import annotations

import struct

from ._lib import CudaCppError
from .cuda_cpp import Context, F32Buffer, I32Buffer

F32, BF16, I8, I32 = "f32", "bf16", "i8", "i32"
_TYPE_IDS = {F32: 0, BF16: 1, I8: 2, I32: 3}
_TYPE_BYTES = {F32: 4, BF16: 2, I8: 1, I32: 4}
_TORCH_TYPES: dict = {}  # torch dtype -> type id, filled when the first tensor comes


# BulletOuB200Matrix as bytes (the type is followed by padding): a call reads
# it before it returns, and building it costs a quarter of a ctypes structure.
_pack = struct.Struct("=QiiQQQ").pack


class DeviceMatrix:
    """rows x cols elements of a library buffer from element `offset` on, rows
    `row_stride` elements apart (default: without a gap).  bf16 and i8 elements
    live packed in an I32Buffer, as the quantised tensors do."""

    def __init__(self, buffer, rows: int, cols: int, type: str | None = None, row_stride: int | None = None,
                 offset: int = 0):
        own = F32 if isinstance(buffer, F32Buffer) else I32
        type = own if type is None else type
        if type not in _TYPE_IDS or (own == F32) != (type == F32):
            raise CudaCppError(f"a {buffer.__class__.__name__} does not hold {type!r} elements")
        stride = cols if row_stride is None else int(row_stride)
        if min(rows, cols, offset) < 0 or (rows > 1 and stride < cols):
            raise CudaCppError(f"invalid matrix: {rows} x {cols}, row stride {stride}, offset {offset}")
        held = len(buffer) * 4 // _TYPE_BYTES[type]
        used = offset + ((rows - 1) * stride + cols if rows and cols else 0)
        if used > held:
            raise CudaCppError(f"matrix of {rows} x {cols} {type} (row stride {stride}, offset {offset}) needs {used} "
                               f"elements, the buffer holds {held}")
        self.buffer, self.type, self.rows, self.cols, self.row_stride = buffer, type, rows, cols, stride
        self.data = (buffer.device_ptr() or 0) + offset * _TYPE_BYTES[type]
        self.device = buffer.ctx.device
        self.packed = _pack(self.data, _TYPE_IDS[type], 0, rows, cols, stride)


def _matrix(x, ctx: Context):
    """The C view of an operand (None stays None)."""
    kind = _TORCH_TYPES.get(getattr(x, "dtype", None))
    if kind is None:
        return _other_matrix(x, ctx)
    if x.get_device() != ctx.device:
        raise CudaCppError(f"tensor is on {x.device}, the context on cuda:{ctx.device}")
    shape, stride = x.shape, x.stride()
    if len(shape) == 2:
        rows, cols = shape
        if stride[1] != 1 and cols > 1 and rows:
            raise CudaCppError(f"tensor of strides {stride}: its last dimension must be contiguous")
        return _pack(x.data_ptr(), kind, 0, rows, cols, stride[0])
    if len(shape) != 1 or (stride[0] != 1 and shape[0] > 1):
        raise CudaCppError(f"tensor of shape {tuple(shape)} and strides {stride}: one or two dimensions, the last one "
                           "contiguous, are supported")
    return _pack(x.data_ptr(), kind, 0, 1, shape[0], shape[0])


def _other_matrix(x, ctx: Context):
    if x is None:
        return None
    if isinstance(x, DeviceMatrix):
        if x.device != ctx.device:
            raise CudaCppError(f"matrix is on device {x.device}, the context on {ctx.device}")
        return x.packed
    if isinstance(x, (F32Buffer, I32Buffer)):
        return _other_matrix(DeviceMatrix(x, 1, len(x)), ctx)
    if not hasattr(x, "data_ptr"):
        raise CudaCppError(f"a matrix is expected, got {type(x).__name__}")
    if _TORCH_TYPES:
        raise CudaCppError(f"tensor type {x.dtype} is not supported")
    import torch

    _TORCH_TYPES.update({torch.float32: 0, torch.bfloat16: 1, torch.int8: 2, torch.int32: 3})
    return _matrix(x, ctx)


def embedding_forward(ctx: Context, table, tokens, out, *, scale: float = 1.0) -> None:
    """out[n] = scale * table[tokens[n]]; zeros where a token is outside the table (-1: padding)."""
    ctx.lib.call("bulletou_b200_embedding_forward_device", ctx.as_ptr(), _matrix(table, ctx), _matrix(tokens, ctx),
                 scale, _matrix(out, ctx))


def embedding_backward(ctx: Context, tokens, out_gradients, table_gradients, *, scale: float = 1.0) -> None:
    """table_gradients[v] = scale * sum of out_gradients[n] over the tokens n that name v; all rows are written."""
    ctx.lib.call("bulletou_b200_embedding_backward_device", ctx.as_ptr(), _matrix(tokens, ctx),
                 _matrix(out_gradients, ctx), scale, _matrix(table_gradients, ctx))


def dropout(ctx: Context, x, out, *, probability: float, seed: int, offset: int = 0, residual=None) -> None:
    """out = x * [kept] / (1 - p) (+ residual); the mask is a function of (seed, offset, element index)."""
    ctx.lib.call("bulletou_b200_dropout_device", ctx.as_ptr(), _matrix(x, ctx), _matrix(residual, ctx), probability,
                 seed & 0xFFFFFFFFFFFFFFFF, offset & 0xFFFFFFFFFFFFFFFF, _matrix(out, ctx))


def dropout_backward(ctx: Context, out_gradients, x_gradients, *, probability: float, seed: int,
                     offset: int = 0) -> None:
    """The gradient of dropout's x (that of its residual is out_gradients)."""
    dropout(ctx, out_gradients, x_gradients, probability=probability, seed=seed, offset=offset)


def router_forward(ctx: Context, logits, experts, gates, counts, mean_probabilities, loss, *, balance: float,
                   normalize_gates: bool = False) -> None:
    """Top-k choice (k = the columns of experts), gates, counts of each expert (and, last, the rows alive), mean
    probabilities and the balance loss of softmax(logits)."""
    ctx.lib.call("bulletou_b200_router_forward_device", ctx.as_ptr(), _matrix(logits, ctx), balance,
                 int(normalize_gates), _matrix(experts, ctx), _matrix(gates, ctx), _matrix(counts, ctx),
                 _matrix(mean_probabilities, ctx), _matrix(loss, ctx))


def router_backward(ctx: Context, logits, experts, counts, gate_gradients, loss_gradient, logit_gradients, *,
                    balance: float, normalize_gates: bool = False) -> None:
    """logit_gradients from the gradients of gates and of the loss (either may be None)."""
    ctx.lib.call("bulletou_b200_router_backward_device", ctx.as_ptr(), _matrix(logits, ctx), _matrix(experts, ctx),
                 _matrix(counts, ctx), _matrix(gate_gradients, ctx), _matrix(loss_gradient, ctx), balance,
                 int(normalize_gates), _matrix(logit_gradients, ctx))


def int8_quantize_rows(ctx: Context, x, q, scales) -> None:
    """q = round(x * 127 / max |x|) and scales = max |x| / 127, row by row."""
    ctx.lib.call("bulletou_b200_int8_quantize_rows_device", ctx.as_ptr(), _matrix(x, ctx), _matrix(q, ctx),
                 _matrix(scales, ctx))


def int8_matmul(ctx: Context, q, scales, weights, weight_scales, out, *, bias=None) -> None:
    """out = (q @ weights.T) * scales[:, None] * weight_scales (+ bias), the product exact in integers."""
    ctx.lib.call("bulletou_b200_int8_matmul_device", ctx.as_ptr(), _matrix(q, ctx), _matrix(scales, ctx),
                 _matrix(weights, ctx), _matrix(weight_scales, ctx), _matrix(bias, ctx), _matrix(out, ctx))


def int8_linear(ctx: Context, x, weights, weight_scales, out, *, bias=None) -> None:
    """int8_matmul of x's rows, quantised on the way."""
    ctx.lib.call("bulletou_b200_int8_linear_device", ctx.as_ptr(), _matrix(x, ctx), _matrix(weights, ctx),
                 _matrix(weight_scales, ctx), _matrix(bias, ctx), _matrix(out, ctx))
