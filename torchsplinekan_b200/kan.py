"""KAN: a stack of :class:`KANLinear` layers (API of spline_kan/kan.py), optionally of residual blocks."""
from __future__ import annotations

import copy
from typing import Callable, List, Optional, Tuple

import torch
import torch.nn as nn

from .block import GATE_ACTIVATIONS, NORMS, BlockNorm, GatedResidual
from .kan_linear import KANLinear


class KAN(nn.Module):
    """Kolmogorov-Arnold network ``layers_hidden[0] -> ... -> layers_hidden[-1]``; every keyword up to
    ``backend`` is forwarded to each :class:`KANLinear` (kan.py:40-81).

    The others turn the chain into blocks (no counterpart in the reference; the defaults are its chain):

    ``norm``: "rms" or "layer": every layer reads the norm of its input (:class:`BlockNorm`), which
    keeps deep stacks inside the knots.  ``residual``: a layer of equal widths becomes
    ``x + scale * post(layer(norm(x)))`` (:class:`GatedResidual`; its post norm is of kind ``norm``), and
    the norm of the next layer is fused into that connection.  ``gate``: "sigmoid" or "silu": such a
    layer has twice the outputs, value and gate, and the connection multiplies by ``act(gate)``.
    ``scale_init``: the residual scales' first value.  ``activation_checkpoint``: "int8" or "e4m3": layers,
    norms and connections keep what their backward reads as 8-bit codes (CUDA inputs).

    A float16 or bfloat16 input is a stream of that type through the connections and needs ``norm``: the layers
    compute in the type of their parameters, which is what a norm returns, and refuse another one."""

    def __init__(self, layers_hidden: List[int], grid_size: int = 5, spline_order: int = 3,
                 scale_noise: float = 0.1, scale_base: float = 1.0, scale_spline: float = 1.0,
                 enable_standalone_scale_spline: bool = True, base_activation=nn.SiLU, grid_eps: float = 0.02,
                 grid_range: tuple = (-1.0, 1.0), backend: str = "auto", norm: Optional[str] = None,
                 residual: bool = False, gate: Optional[str] = None, scale_init: float = 1.0,
                 activation_checkpoint: Optional[str] = None) -> None:
        super().__init__()
        if len(layers_hidden) < 2:
            raise ValueError("layers_hidden must have at least two entries (in_features and out_features "
                             f"of the first layer), got {layers_hidden}")
        if norm not in NORMS:
            raise ValueError(f"norm must be one of {list(NORMS)}, got {norm!r}")
        if gate not in GATE_ACTIVATIONS:
            raise ValueError(f"gate must be one of {list(GATE_ACTIVATIONS)}, got {gate!r}")
        if gate is not None and not residual:
            raise ValueError("gate needs residual=True")
        pairs = list(zip(layers_hidden[:-1], layers_hidden[1:]))
        if residual and all(a != b for a, b in pairs):
            raise ValueError(f"residual=True needs a layer of equal widths, got {layers_hidden}")
        self.layers = nn.ModuleList(
            KANLinear(a, 2 * b if residual and a == b and gate is not None else b, grid_size=grid_size,
                      spline_order=spline_order, scale_noise=scale_noise, scale_base=scale_base, scale_spline=scale_spline,
                      enable_standalone_scale_spline=enable_standalone_scale_spline,
                      base_activation=base_activation, grid_eps=grid_eps, grid_range=grid_range, backend=backend,
                      activation_checkpoint=activation_checkpoint)
            for a, b in pairs)
        self.norms = nn.ModuleList(BlockNorm(a, norm, checkpoint=activation_checkpoint) for a, _ in pairs) \
            if norm is not None else None
        self.connections = nn.ModuleDict({
            str(i): GatedResidual(a, gate, norm, scale_init, checkpoint=activation_checkpoint)
            for i, (a, b) in enumerate(pairs) if a == b}) if residual else None

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        for part in ("norms", "connections"):                # of networks pickled before the blocks existed
            if part not in self.__dict__ and part not in self._modules:
                setattr(self, part, None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self._walk(x, lambda layer, h: layer(h))

    def _walk(self, x: torch.Tensor, call: Callable[[KANLinear, torch.Tensor], torch.Tensor]) -> torch.Tensor:
        """The network with ``call(layer, layer's input)`` in the place of every layer's evaluation."""
        if self.norms is None and self.connections is None:
            for layer in self.layers:
                x = call(layer, x)
            return x
        h = None                                             # norm of x, where a connection already formed it
        for i, layer in enumerate(self.layers):
            if h is None:
                h = self.norms[i](x) if self.norms is not None else x
            y = call(layer, h)
            h = None
            if self.connections is None or str(i) not in self.connections:
                x = y
            elif self.norms is not None and i + 1 < len(self.layers):
                x, h = self.connections[str(i)](x, y, self.norms[i + 1])
            else:
                x = self.connections[str(i)](x, y)
        return x

    def update_grid(self, x: torch.Tensor, margin: float = 0.01) -> None:
        """Updates each layer's knots with the activations that layer actually sees (kan.py:88-99)."""
        def call(layer, h):
            layer.update_grid(h, margin=margin)
            return layer(h)
        with torch.no_grad():
            self._walk(x, call)

    def regularization_loss(self, reg_act: float = 1.0, reg_entropy: float = 1.0, *, x: torch.Tensor,
                            mode: str = "activation", reg_impl: str = "auto", chunk_size: int = 1024,
                            reg_group=None) -> torch.Tensor:
        """Sum of the layers' penalties, each evaluated on that layer's real input; hidden
        activations are not detached (kan.py:101-148)."""
        if mode == "coefficient":
            total = x.new_zeros(())
            for layer in self.layers:
                total = total + layer.regularization_loss(reg_act, reg_entropy, mode="coefficient")
            return total
        return self.forward_with_regularization(x, reg_act, reg_entropy, mode=mode, reg_impl=reg_impl,
                                                chunk_size=chunk_size, reg_group=reg_group)[1]

    def forward_with_regularization(self, x: torch.Tensor, reg_act: float = 1.0, reg_entropy: float = 1.0, *,
                                    mode: str = "activation", reg_impl: str = "auto", chunk_size: int = 1024,
                                    reg_group=None) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(self(x), regularization_loss)`` from a single pass (kan.py:150-175).  ``reg_group``: a
        process group (True = the default one) makes every layer penalise the statistic of the global
        batch instead of this process's rows (see :meth:`KANLinear.forward_with_regularization`)."""
        if mode == "coefficient":
            return self(x), self.regularization_loss(reg_act, reg_entropy, x=x, mode="coefficient")
        total = x.new_zeros((), dtype=self.layers[0].grid.dtype)

        def call(layer, h):
            nonlocal total
            h, r = layer.forward_with_regularization(h, reg_act, reg_entropy, mode=mode, reg_impl=reg_impl,
                                                     chunk_size=chunk_size, reg_group=reg_group)
            total = total + r
            return h
        return self._walk(x, call), total

    def export_inference(self, requires_grad: bool = False) -> "KAN":
        """Independent network built from the layers' :meth:`KANLinear.export_inference` (kan.py:177-187)."""
        twin = self._with_layers([layer.export_inference(requires_grad) for layer in self.layers])
        for part in (twin.norms, twin.connections):
            if part is not None:
                part.requires_grad_(requires_grad)
        return twin.train(self.training and requires_grad)

    def _with_layers(self, layers: List[KANLinear]) -> "KAN":
        """Network of other layers of the same widths, with copies of the norms and connections."""
        net = KAN.__new__(KAN)
        nn.Module.__init__(net)
        net.layers = nn.ModuleList(layers)
        net.norms, net.connections = copy.deepcopy(self.norms), copy.deepcopy(self.connections)
        return net

    @classmethod
    def from_layers(cls, layers: List[KANLinear]) -> "KAN":
        """Wraps existing layers; widths must chain (kan.py:189-199)."""
        for a, b in zip(layers[:-1], layers[1:]):
            if a.out_features != b.in_features:
                raise ValueError(f"layer widths do not chain: {a.out_features} -> {b.in_features}")
        net = cls.__new__(cls)
        nn.Module.__init__(net)
        net.layers = nn.ModuleList(layers)
        net.norms = net.connections = None
        return net

    def parameter_modules(self) -> List[nn.Module]:
        """The modules that own the parameters, in forward order: every layer with its norm in front of it and its
        connection behind it (what :class:`GradientBucket` reduces for this network)."""
        modules: List[nn.Module] = []
        for i, layer in enumerate(self.layers):
            if self.norms is not None:
                modules.append(self.norms[i])
            modules.append(layer)
            if self.connections is not None and str(i) in self.connections:
                modules.append(self.connections[str(i)])
        return modules

    @property
    def widths(self) -> List[int]:
        """Widths of the stream (a gated connection halves its layer's outputs)."""
        connected = self.connections if self.connections is not None else {}
        return [self.layers[0].in_features] + [layer.in_features if str(i) in connected else layer.out_features
                                               for i, layer in enumerate(self.layers)]

    def prune(self, x_calib: torch.Tensor, threshold: float = 1e-2, **kw):
        """:func:`~torchsplinekan_b200.pruning.prune_nodes` on this network (kan.py:204-207)."""
        from .pruning import prune_nodes
        return prune_nodes(self, x_calib, threshold, **kw)

    @torch.no_grad()
    def extend_grid(self, new_grid_size: int, x: torch.Tensor, **kw) -> "KAN":
        """NEW network with every layer refined to ``new_grid_size``, each fitted on the original
        network's activations (kan.py:208-223)."""
        refined = []

        def call(layer, h):
            refined.append(layer.extend_grid(new_grid_size, h, **kw))
            return layer(h)
        self._walk(x, call)
        return self._with_layers(refined).train(self.training)
