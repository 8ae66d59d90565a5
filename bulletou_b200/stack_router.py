"""A learned choice of the LayerStack.

The reference picks a position's dense stack by a fixed rule on the kings'
ranks (ShogiSfnnLayerStackBucketKind::bucket_from_board, game/outputs.rs:1227-1231).
``StackRouter`` learns it from what each stack costs on each position: the
feature rows of the sparse batch are looked up token by token, dropped out,
multiplied with one weight row for each stack, and the logits choose.  Training
minimises the expected cost under the chosen gates plus a balance loss that
keeps all stacks in use; evaluation multiplies in 8-bit integers, as the engine
does, and writes the choices as the ``buckets`` that an SFNN runner steps on.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import numpy as np

from ._lib import CudaCppError
from .cuda_cpp import Context, F32Buffer, I32Buffer, RangerDeviceState, RangerParamState, RangerUpdateParams, ranger_update_device
from .token_layers import (DeviceMatrix, dropout, dropout_backward, embedding_backward, embedding_forward, int8_linear,
                           int8_quantize_rows, router_backward, router_forward)


class StackRouter:
    """Tokens [batch][max_active] (feature rows, -1 padded) to one of `stacks`.

    table [vocab][width] and weights [stacks][max_active * width] are f32 and
    trained by Ranger; `top_k` stacks share a position's gates in training."""

    def __init__(self, ctx: Context, vocab: int, max_active: int, width: int, stacks: int, batch_size: int, *,
                 top_k: int = 2, balance: float = 0.01, drop_probability: float = 0.1, seed: int = 0,
                 table: Optional[np.ndarray] = None, weights: Optional[np.ndarray] = None):
        if min(vocab, max_active, width, stacks, batch_size) <= 0 or not 1 <= top_k <= stacks:
            raise CudaCppError(f"invalid stack router: vocab {vocab}, {max_active} tokens of width {width}, {stacks} "
                               f"stacks, top {top_k}, batch {batch_size}")
        rng = np.random.default_rng(seed)
        inner = max_active * width
        if table is None:
            table = rng.standard_normal((vocab, width)).astype(np.float32) * 0.1
        if weights is None:
            weights = rng.standard_normal((stacks, inner)).astype(np.float32) / math.sqrt(inner)
        self.ctx, self.seed, self.step = ctx, seed, 0
        self.vocab, self.max_active, self.width, self.stacks = vocab, max_active, width, stacks
        self.batch_size, self.top_k = batch_size, top_k
        self.balance, self.drop_probability = balance, drop_probability
        self.scale = 1.0 / math.sqrt(max_active)  # so many tokens add up to a logit

        def parameter(values, shape, name):
            values = np.ascontiguousarray(values, np.float32)
            if values.shape != shape:
                raise CudaCppError(f"stack router {name} has shape {values.shape}, expected {shape}")
            return F32Buffer.from_host(ctx, values), RangerParamState(ctx, values.reshape(-1)), F32Buffer(ctx, values.size)

        self.table, self.table_state, self.table_gradients = parameter(table, (vocab, width), "table")
        self.weights, self.weight_state, self.weight_gradients = parameter(weights, (stacks, inner), "weights")
        rows, b = batch_size * max_active, batch_size
        self.hidden, self.hidden_gradients = F32Buffer(ctx, b * inner), F32Buffer(ctx, b * inner)
        self.logits, self.logit_gradients = F32Buffer(ctx, b * stacks), F32Buffer(ctx, b * stacks)
        self.experts, self.gates = I32Buffer(ctx, b * top_k), F32Buffer(ctx, b * top_k)
        self.gate_gradients = F32Buffer(ctx, b * top_k)
        self.counts, self.mean_probabilities = I32Buffer(ctx, stacks + 1), F32Buffer(ctx, stacks)
        self.loss, self.expected_cost, self.one = F32Buffer(ctx, 1), F32Buffer(ctx, 1), F32Buffer.from_host(ctx, [1.0])
        self.choice_loss = F32Buffer(ctx, 1)  # the balance loss of a choice
        self.weights8, self.weight_scales = I32Buffer(ctx, (stacks * inner + 3) // 4), F32Buffer(ctx, stacks)
        self.choice_gates = F32Buffer(ctx, b)
        self._m = {
            "table": DeviceMatrix(self.table, vocab, width), "d_table": DeviceMatrix(self.table_gradients, vocab, width),
            "tokens_hidden": DeviceMatrix(self.hidden, rows, width),
            "d_tokens_hidden": DeviceMatrix(self.hidden_gradients, rows, width),
            "hidden": DeviceMatrix(self.hidden, b, inner), "weights": DeviceMatrix(self.weights, stacks, inner),
            "weights8": DeviceMatrix(self.weights8, stacks, inner, "i8"),
            "logits": DeviceMatrix(self.logits, b, stacks), "d_logits": DeviceMatrix(self.logit_gradients, b, stacks),
            "experts": DeviceMatrix(self.experts, b, top_k), "gates": DeviceMatrix(self.gates, b, top_k),
            "d_gates": DeviceMatrix(self.gate_gradients, b, top_k), "choice_gates": DeviceMatrix(self.choice_gates, b, 1),
        }
        self.quantized = False

    def _torch(self):
        """torch, with its work ordered on the context's stream."""
        import torch

        p = ctypes.c_void_p()
        self.ctx.lib.call("bulletou_b200_context_stream", self.ctx.as_ptr(), ctypes.byref(p))
        return torch, torch.cuda.stream(torch.cuda.ExternalStream(p.value or 0, device=self.ctx.device))

    def _view(self, torch, buffer, *shape):
        return torch.as_tensor(buffer, device=f"cuda:{self.ctx.device}").view(*shape)

    def _lookup(self, tokens: I32Buffer) -> None:
        embedding_forward(self.ctx, self._m["table"], DeviceMatrix(tokens, self.batch_size, self.max_active),
                          self._m["tokens_hidden"], scale=self.scale)

    def train_step(self, params: RangerUpdateParams, tokens: I32Buffer, costs: F32Buffer) -> None:
        """``gradients`` and ``update``."""
        self.gradients(tokens, costs)
        self.update(params)

    def gradients(self, tokens: I32Buffer, costs: F32Buffer) -> None:
        """table_gradients and weight_gradients of mean(sum_j gate_j cost[choice_j]) + the
        balance loss, on tokens [batch][max_active] and costs [batch][stacks]: what each
        stack loses on each position."""
        ctx, m, b = self.ctx, self._m, self.batch_size
        if len(costs) != b * self.stacks:
            raise CudaCppError(f"costs have {len(costs)} values, expected {b * self.stacks}")
        self._lookup(tokens)
        drop = {"probability": self.drop_probability, "seed": self.seed, "offset": self.step}
        dropout(ctx, m["tokens_hidden"], m["tokens_hidden"], **drop)
        torch, on_stream = self._torch()
        with on_stream:
            hidden = self._view(torch, self.hidden, b, -1)
            weights = self._view(torch, self.weights, self.stacks, -1)
            torch.mm(hidden, weights.T, out=self._view(torch, self.logits, b, -1))
        router_forward(ctx, m["logits"], m["experts"], m["gates"], self.counts, self.mean_probabilities, self.loss,
                       balance=self.balance, normalize_gates=True)
        with on_stream:
            experts = self._view(torch, self.experts, b, -1).long()
            picked = self._view(torch, costs, b, -1).gather(1, experts.clamp(min=0)).masked_fill(experts < 0, 0.0)
            torch.sum(self._view(torch, self.gates, b, -1) * picked / b, dim=(0, 1), out=self._view(torch, self.expected_cost, 1)[0])
            self._view(torch, self.gate_gradients, b, -1).copy_(picked / b)
        router_backward(ctx, m["logits"], m["experts"], self.counts, m["d_gates"], self.one, m["d_logits"],
                        balance=self.balance, normalize_gates=True)
        with on_stream:
            d_logits = self._view(torch, self.logit_gradients, b, -1)
            torch.mm(d_logits.T, hidden, out=self._view(torch, self.weight_gradients, self.stacks, -1))
            torch.mm(d_logits, weights, out=self._view(torch, self.hidden_gradients, b, -1))
        dropout_backward(ctx, m["d_tokens_hidden"], m["d_tokens_hidden"], **drop)
        embedding_backward(ctx, DeviceMatrix(tokens, b, self.max_active), m["d_tokens_hidden"], m["d_table"],
                           scale=self.scale)
        self.step += 1

    def update(self, params: RangerUpdateParams) -> None:
        """Ranger on both parameters; it clears their gradients."""
        for values, state, gradients in ((self.table, self.table_state, self.table_gradients),
                                         (self.weights, self.weight_state, self.weight_gradients)):
            ranger_update_device(self.ctx, params, RangerDeviceState(gradients, values, state.momentum, state.velocity,
                                                                     state.slow_params))
        self.quantized = False

    def quantize(self) -> None:
        """The weights as 8-bit rows with a scale for each stack."""
        int8_quantize_rows(self.ctx, self._m["weights"], self._m["weights8"], self.weight_scales)
        self.quantized = True

    def choose(self, tokens: I32Buffer, buckets: I32Buffer, *, keep_weights: bool = False) -> None:
        """buckets [batch] = the best stack of each position (a position without tokens: the first among equals).  A
        position whose logits are not finite (its rows hold NaN or infinities) gets -1, a bucket that an SFNN step gives
        to no stack; ``read_counts`` then adds up to fewer than the batch.

        The weights are quantised as the buffer holds them now.  A program that serves fixed weights sets
        `keep_weights`: those of the last ``quantize`` or choice are then taken, unless ``update`` has run since."""
        if len(buckets) != self.batch_size:
            raise CudaCppError(f"buckets have {len(buckets)} values, expected {self.batch_size}")
        if not (keep_weights and self.quantized):
            self.quantize()
        m = self._m
        self._lookup(tokens)
        int8_linear(self.ctx, m["hidden"], m["weights8"], self.weight_scales, m["logits"])
        router_forward(self.ctx, m["logits"], DeviceMatrix(buckets, self.batch_size, 1), m["choice_gates"], self.counts,
                       self.mean_probabilities, self.choice_loss, balance=self.balance)

    def read_counts(self) -> np.ndarray:
        """Choices of each stack in the last step or choice (a device-to-host read)."""
        return self.counts.download()[:-1]

    def read_losses(self) -> tuple:
        """(expected cost, balance loss) of the last step; a choice leaves them."""
        return float(self.expected_cost.download()[0]), float(self.loss.download()[0])
