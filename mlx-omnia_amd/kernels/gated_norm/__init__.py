"""The norm and the gate of a mixer's output, in groups: one facade, two bindings.

    y = norm(x) * weight * act(gate)          as models/qwen3_5 norms its mixer's heads
    y = norm(x * act(gate)) * weight          gate_first, as core/kernels/mamba_step's groups

norm(v) = v / sqrt(mean(v^2) + eps) over each `group` consecutive values of a row (a head), act
silu or sigmoid; in fp32, rounded once. The declaration is the norm leaf (`.weight` [group] or
[row width], `.eps`); a call takes x and the gate [..., width] or, with a weight [group],
[..., heads, group], alike in shape, row-strided views of wider rows among them.
`HipGatedRmsNorm` (`omnia_gated_rms_norm`, csrc/block_norms.hip) serves bf16 on a gfx950 device,
`DefaultGatedRmsNorm` everything else and calls that autograd follows.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Protocol, runtime_checkable

import torch

from ...runtime import ops
from .._device import hip_device, in_place
from ..attention.prefill import unfollowed
from ..resolve import record_fallback, resolve

__all__ = ["DefaultGatedRmsNorm", "GatedRmsNorm", "GatedRmsNormStrategy", "HipGatedRmsNorm", "applies"]

MAX_GROUP = 8192
ACTIVATIONS = ("silu", "sigmoid")


@runtime_checkable
class GatedRmsNormStrategy(Protocol):
    def __call__(self, x: torch.Tensor, gate: torch.Tensor) -> torch.Tensor: ...


def applies(group: int) -> bool:
    """The group tiles as 16-byte vectors, at most 16 per lane of one wave64."""
    return 0 < group <= MAX_GROUP and group % 8 == 0


@dataclass(frozen=True)
class DefaultGatedRmsNorm(GatedRmsNormStrategy):
    weight: torch.Tensor
    eps: float
    group: int
    activation: str
    gate_first: bool

    @classmethod
    def build(cls, leaf, *, group, activation, gate_first) -> "DefaultGatedRmsNorm":
        return cls(leaf.weight, float(leaf.eps), group, activation, gate_first)

    def __call__(self, x, gate):
        kind = torch.promote_types(x.dtype, torch.float32)
        wide, z = (t.to(kind).unflatten(-1, (t.shape[-1] // self.group, self.group)) for t in (x, gate))
        weight = self.weight.to(kind).unflatten(0, (-1, self.group))   # of each group, or of all
        z = torch.sigmoid(z) * (z if self.activation == "silu" else 1)
        y = wide * z if self.gate_first else wide
        y = y * (1.0 / torch.sqrt((y * y).mean(dim=-1, keepdim=True) + self.eps)) * weight
        return (y if self.gate_first else y * z).reshape(x.shape).to(x.dtype)


@dataclass(frozen=True, eq=False)
class HipGatedRmsNorm(GatedRmsNormStrategy):
    core: DefaultGatedRmsNorm
    weight: torch.Tensor

    @classmethod
    def build(cls, leaf, *, group, activation, gate_first) -> "HipGatedRmsNorm | None":
        weight = leaf.weight
        if weight.dtype != torch.bfloat16 or not applies(group) or not hip_device(weight):
            return None
        if not in_place(weight):
            return None
        return cls(DefaultGatedRmsNorm.build(leaf, group=group, activation=activation, gate_first=gate_first), weight)

    def __call__(self, x, gate):
        core = self.core
        if x.dtype is not torch.bfloat16 or gate.dtype is not torch.bfloat16 or not unfollowed(x, gate, self.weight):
            record_fallback(self, core)
            return core(x, gate)
        return ops.gated_rms_norm(x, gate, self.weight, group=core.group, eps=core.eps, silu=core.activation == "silu",
                                  gate_first=core.gate_first)


_STRATEGIES = (HipGatedRmsNorm, DefaultGatedRmsNorm)


class GatedRmsNorm(GatedRmsNormStrategy):
    """Picks its binding once, then forwards every call. `group` is the leaf's width unless the
    weight covers a row of several groups."""

    def __init__(self, leaf, *, group: int | None = None, activation: str = "silu", gate_first: bool = False,
                 reference: bool = False) -> None:
        self.width = leaf.weight.numel()
        self.group = self.width if group is None else group
        if leaf.weight.dim() != 1 or self.group < 1 or self.width % self.group:
            raise ValueError(f"GatedRmsNorm: a weight {tuple(leaf.weight.shape)} in groups of {self.group}")
        if activation not in ACTIVATIONS:
            raise ValueError(f"GatedRmsNorm: activation {activation!r}, not one of {ACTIVATIONS}")
        self.strategy: GatedRmsNormStrategy = resolve(
            (DefaultGatedRmsNorm,) if reference else _STRATEGIES, leaf, group=self.group, activation=activation,
            gate_first=gate_first)

    def __call__(self, x: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
        if x.shape != gate.shape:
            raise ValueError(f"GatedRmsNorm: x {tuple(x.shape)} and gate {tuple(gate.shape)} differ")
        width = x.shape[-1]
        if width % self.group or not width or self.width not in (self.group, width):
            raise ValueError(f"GatedRmsNorm: rows of {width} with a weight of {self.width} in groups of {self.group}")
        return self.strategy(x, gate)
