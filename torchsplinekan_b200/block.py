"""
Operators around a KAN layer: the norm in front of it, the gated residual connection behind it, and 8-bit checkpoints of
what a training step keeps for its backward.  The reference has no counterpart (its networks are plain chains of
layers); deep chains need the inputs of every layer inside that layer's knots, a residual path around it, and less memory
per layer.

Rows are the leading dimensions, columns the last one.  The *stream* (``x``, the result of :func:`gated_residual`) may
be float32, float64, bfloat16 or float16; the *branch* (``y``, gates, parameters, the norm's result) is what
:class:`KANLinear` computes in: float64 next to a float64 stream, float32 otherwise.

CUDA tensors run on the native kernels (one kernel forward; backward one kernel plus the fixed-order sum of the
parameter gradients), CPU tensors on dense PyTorch formulas.  Any strides and alignments are taken; widths that are a
multiple of four with rows and parameters on 16-byte boundaries run fastest.  ``create_graph=True`` is exact without a
checkpoint and raises with one.  Fake tensors and ``torch.func`` transforms are refused on CUDA.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn as nn

from . import _C

NORMS = {None: 0, "rms": 1, "layer": 2}
GATE_ACTIVATIONS = {None: 0, "sigmoid": 1, "silu": 2}
CHECKPOINTS = {None: 0, "int8": 1, "e4m3": 2}
PACK_GROUP = int(_C.PACK_GROUP)


def _code(table: dict, name: str, value) -> int:
    if value is None:
        return 0
    try:
        return table[value]
    except (KeyError, TypeError):
        raise ValueError(f"{name} must be one of {list(table)}, got {value!r}") from None


def block_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               kind: str = "rms", eps: float = 1e-6, checkpoint: Optional[str] = None) -> torch.Tensor:
    """``(x - m) r * weight + bias`` over the last dimension, in the branch's type: the norm in front of a layer.

    ``kind``: "rms" (``m = 0``, ``r = (mean(x^2) + eps)^-1/2``) or "layer" (``m = mean(x)``,
    ``r = (mean((x - m)^2) + eps)^-1/2``).  Rows whose sum of squares overflows the branch's type have ``r = 0``;
    rows whose sum overflows as well come back as NaN from "layer".

    ``checkpoint``: None keeps ``x`` for the backward; "int8" / "e4m3" keep 8-bit codes of it instead (see
    :func:`pack_activation`), written by the same kernel.  The result is the same; the gradients are those of the
    formulas with the restored ``x`` next to the exact ``m`` and ``r``."""
    if kind is None:
        raise ValueError("kind must be 'rms' or 'layer', got None")
    return _C.block_norm(x, weight, bias, _code(NORMS, "kind", kind), eps, _code(CHECKPOINTS, "checkpoint", checkpoint))


def gated_residual(x: torch.Tensor, y: torch.Tensor, *, gate: Union[torch.Tensor, str, None] = None,
                   gate_activation: Optional[str] = None, scale: Optional[torch.Tensor] = None,
                   post_norm: Optional[str] = None, post_weight: Optional[torch.Tensor] = None,
                   post_bias: Optional[torch.Tensor] = None, next_norm: Optional[str] = None,
                   next_weight: Optional[torch.Tensor] = None, next_bias: Optional[torch.Tensor] = None,
                   eps: float = 1e-6, checkpoint: Optional[str] = None
                   ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The connection behind a layer, ``out = x + scale * act(gate) * post(y)``, in one pass.

    ``gate``: None; a tensor of ``x``'s shape; one of size 1 in trailing row dimensions (``[B, 1, D]`` next to an ``x`` of
    ``[B, T, D]``: one gate per sequence; ``[D]``: one for all rows); or "packed": ``y`` is ``[..., 2 D]`` and holds value
    and gate side by side.  ``gate_activation``: None, "sigmoid" or "silu".  ``scale``: ``[D]``.
    ``post_norm`` / ``next_norm``: None, "rms" or "layer", as in :func:`block_norm`.

    With ``next_norm`` the result is ``(out, h)`` where ``h`` is the norm of ``out`` (as stored, in ``x``'s type) for the
    next block.  ``checkpoint``: what the backward reads of ``y``, of a gate per row and of ``out`` is kept as 8-bit codes;
    a shared gate is kept as it is."""
    packed = isinstance(gate, str)
    if packed:
        if gate != "packed":
            raise ValueError(f"gate must be a tensor, None or 'packed', got {gate!r}")
        gate = None
    return _C.gated_residual(x, y, gate, packed, _code(GATE_ACTIVATIONS, "gate_activation", gate_activation), scale,
                             _code(NORMS, "post_norm", post_norm), post_weight, post_bias,
                             _code(NORMS, "next_norm", next_norm), next_weight, next_bias, eps,
                             _code(CHECKPOINTS, "checkpoint", checkpoint))


def pack_activation(x: torch.Tensor, format: str = "int8") -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)``: ``x`` in 8 bits with one scale per 128 columns of a row.

    Per group, with ``A = max|x|``: ``scale = max(A / 127, smallest normal)`` ("e4m3": ``A / 448``) and
    ``codes = round(x / scale)``, int8 or float8_e4m3fn.  "int8" has the smaller error on inputs of about one size
    (at most ``A / 254``), "e4m3" keeps relative precision (``2^-4``) over a wide range.  A group that holds a NaN or an
    infinity comes back as NaN, so an overflow stays visible.  CUDA tensors only; no gradient flows through it."""
    if format is None:
        raise ValueError("format must be 'int8' or 'e4m3', got None")
    return _C.pack_activation(x, _code(CHECKPOINTS, "format", format))


def unpack_activation(codes: torch.Tensor, scales: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``codes * scales`` in ``dtype`` (default: the type of the scales)."""
    return _C.unpack_activation(codes, scales, scales.dtype if dtype is None else dtype)


class BlockNorm(nn.Module):
    """:func:`block_norm` with its parameters: weight (ones) and, for "layer", bias (zeros)."""

    def __init__(self, width: int, kind: str = "rms", eps: float = 1e-6, checkpoint: Optional[str] = None) -> None:
        super().__init__()
        if kind is None:
            raise ValueError("kind must be 'rms' or 'layer', got None")
        _code(NORMS, "kind", kind)
        _code(CHECKPOINTS, "checkpoint", checkpoint)
        self.kind, self.eps, self.checkpoint = kind, eps, checkpoint
        self.weight = nn.Parameter(torch.ones(width))
        self.bias = nn.Parameter(torch.zeros(width)) if kind == "layer" else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return block_norm(x, self.weight, self.bias, kind=self.kind, eps=self.eps,
                          checkpoint=self.checkpoint if x.is_cuda else None)


class GatedResidual(nn.Module):
    """:func:`gated_residual` with its parameters: scale (``scale_init``) and those of the post norm.

    ``gate``: None, "sigmoid" or "silu": the activation of the second half of ``y``, which then holds value and gate side
    by side.  ``next_norm``: the :class:`BlockNorm` of the next block, fused into the same pass."""

    def __init__(self, width: int, gate: Optional[str] = None, post_norm: Optional[str] = "rms", scale_init: float = 1.0,
                 eps: float = 1e-6, checkpoint: Optional[str] = None) -> None:
        super().__init__()
        _code(GATE_ACTIVATIONS, "gate", gate)
        _code(NORMS, "post_norm", post_norm)
        _code(CHECKPOINTS, "checkpoint", checkpoint)
        self.gate, self.post_norm, self.eps, self.checkpoint = gate, post_norm, eps, checkpoint
        self.scale = nn.Parameter(torch.full((width,), float(scale_init)))
        self.post_weight = nn.Parameter(torch.ones(width)) if post_norm is not None else None
        self.post_bias = nn.Parameter(torch.zeros(width)) if post_norm == "layer" else None

    def forward(self, x: torch.Tensor, y: torch.Tensor, next_norm: Optional[BlockNorm] = None):
        if next_norm is not None and next_norm.eps != self.eps:
            raise ValueError(f"the norms of one connection share eps, got {self.eps} and {next_norm.eps}")
        return gated_residual(x, y, gate="packed" if self.gate else None, gate_activation=self.gate, scale=self.scale,
                              post_norm=self.post_norm, post_weight=self.post_weight, post_bias=self.post_bias,
                              next_norm=next_norm.kind if next_norm is not None else None,
                              next_weight=next_norm.weight if next_norm is not None else None,
                              next_bias=next_norm.bias if next_norm is not None else None, eps=self.eps,
                              checkpoint=self.checkpoint if x.is_cuda else None)
