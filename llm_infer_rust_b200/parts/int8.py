"""Parts whose projections are held in 8-bit integers (see kernels/int8.py): one scale an output channel, found when a
weight is bound, and the activations' scales, one a token, on the way into every product.

``int8_projections(spec)`` names them in the place of the parts of a model that have such a form; embedding, head, norms and what
attention does between its projections stay as they are.
"""
from __future__ import annotations

from dataclasses import replace
from typing import Dict

import torch

from ..config.spec import ConfigError, ModelSpec, PartSpec
from ..kernels import int8
from .attention import GQAttention
from .feed_forward import GatedActFF, SwiGLU
from .registry import register_part


class _Int8Projections:
    """A part whose matrices named by ``INT8`` are taken to 8 bits as they are bound: of a checkpoint's matrix only the 8-bit
    values and the scales stay (``params`` holds the values, as the parameter's memory).  What its products read may be a norm
    that has not run: it runs on the way to 8 bits, whatever the number of tokens."""
    INT8 = ()
    chainable = True

    def bind(self, name: str, tensor: torch.Tensor) -> None:
        super().bind(name, tensor)
        if name in self.INT8:
            weight = int8.int8_weight(tensor.contiguous())
            self.params[name] = weight.values
            self.int8: Dict[str, int8.Int8Weight] = dict(getattr(self, "int8", {}), **{name: weight})

    def takes_pending(self, tokens: int) -> bool:
        return True


class Int8SwiGLU(_Int8Projections, SwiGLU):
    """``SwiGLU`` in 8-bit integers: (norm,) gate and up with silu(gate) * up behind the product, then down."""
    INT8 = ("gate_up_proj", "down_proj")

    def forward(self, x):
        return int8.int8_linear(int8.int8_glu(x, self.int8["gate_up_proj"]), self.int8["down_proj"])


class Int8GatedActFF(_Int8Projections, GatedActFF):
    """``GatedActFF`` in 8-bit integers."""
    INT8 = ("gate_up_proj", "down_proj")

    def forward(self, x):
        h = int8.int8_glu(x, self.int8["gate_up_proj"], self._GLU[self.activation], self.limit, self.alpha)
        return int8.int8_linear(h, self.int8["down_proj"])


class Int8GQAttention(_Int8Projections, GQAttention):
    """``GQAttention`` with its packed q, k, v projection and its output projection in 8-bit integers."""
    INT8 = ("qkv_proj", "o_proj")

    def _fuses_heads(self, tokens: int) -> bool:
        return False

    def _project_heads(self, x):
        return int8.int8_linear(x, self.int8["qkv_proj"])

    def _project_out(self, out):
        return int8.int8_linear(out, self.int8["o_proj"])


_KINDS = {"swiglu": "swiglu_int8", "gated_act": "gated_act_int8", "gqa_attention": "gqa_attention_int8"}


def int8_projections(spec: ModelSpec) -> ModelSpec:
    """``spec`` with the parts that have a form in 8-bit integers named in it; refused where none has."""
    def of(part: PartSpec) -> PartSpec:
        return PartSpec(_KINDS.get(part.kind, part.kind), part.params)

    layers = tuple(replace(layer, parts={name: of(part) for name, part in layer.parts.items()}) for layer in spec.layers)
    if layers == spec.layers:
        raise ConfigError(f"no layer of {spec.architecture} has projections with a form in 8-bit integers "
                          f"(kinds that have one: {', '.join(sorted(_KINDS))})")
    return replace(spec, layers=layers)


register_part("feed_forward", "swiglu_int8", Int8SwiGLU)
register_part("feed_forward", "gated_act_int8", Int8GatedActFF)
register_part("mixer", "gqa_attention_int8", Int8GQAttention)
