"""The join of two blocks that are normed on both sides: one facade, two bindings.

    s = residual_scale * x + block_scale * act(gate) * norm(block; post)
    joined(x, block) -> (s, norm(s; pre))

The counterpart of `AddRmsNorm` (core/kernels/add_norm) for blocks whose output is normed,
gated or scaled before the residual takes it. `pre` is the norm leaf of the block ahead, `post`
that of the block behind (or None); the gate is a tensor like x, or one row [hidden], taken as
it is or through a sigmoid. In fp32, each output rounded once: the norm reads s before its
rounding (`AddRmsNorm`, as its reference does, after). `HipBlockNorm` (`omnia_block_norm`,
csrc/block_norms.hip) serves bf16 rows on a gfx950 device, `DefaultBlockNorm` everything else
and calls that autograd follows.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Protocol, runtime_checkable

import torch

from ...runtime import ops
from .._device import hip_device, in_place
from ..attention.prefill import unfollowed
from ..resolve import record_fallback, resolve

__all__ = ["BlockNorm", "BlockNormStrategy", "DefaultBlockNorm", "HipBlockNorm", "applies"]

MAX_HIDDEN = 16384
BF16 = torch.bfloat16
ACTIVATIONS = (None, "sigmoid")


@runtime_checkable
class BlockNormStrategy(Protocol):
    def __call__(self, x: torch.Tensor, block: torch.Tensor,
                 gate: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]: ...


def applies(hidden: int) -> bool:
    """The row tiles as 16-byte vectors, four at most per lane of a workgroup of eight waves."""
    return 0 < hidden <= MAX_HIDDEN and hidden % 8 == 0


def _norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    return x * (1.0 / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + eps)) * weight.to(x.dtype)


@dataclass(frozen=True)
class DefaultBlockNorm(BlockNormStrategy):
    pre: torch.Tensor
    pre_eps: float
    post: torch.Tensor | None
    post_eps: float
    residual_scale: float
    block_scale: float
    activation: str | None

    @classmethod
    def build(cls, pre, post, *, residual_scale, block_scale, activation) -> "DefaultBlockNorm":
        return cls(pre.weight, float(pre.eps), None if post is None else post.weight,
                   0.0 if post is None else float(post.eps), residual_scale, block_scale, activation)

    def __call__(self, x, block, gate=None):
        hidden = self.pre.numel()
        if x.shape != block.shape or x.shape[-1] != hidden:
            raise ValueError(f"block norm: x {tuple(x.shape)} and block {tuple(block.shape)} are not rows of {hidden}")
        if gate is not None and gate.shape != x.shape and gate.shape != (hidden,):
            raise ValueError(f"block norm: a gate {tuple(gate.shape)} for rows {tuple(x.shape)}")
        kind = torch.promote_types(x.dtype, torch.float32)
        y = block.to(kind)
        if self.post is not None:
            y = _norm(y, self.post, self.post_eps)
        if gate is not None:
            y = y * (gate.to(kind) if self.activation is None else torch.sigmoid(gate.to(kind)))
        s = self.residual_scale * x.to(kind) + self.block_scale * y
        return s.to(x.dtype), _norm(s, self.pre, self.pre_eps).to(x.dtype)


@dataclass(frozen=True, eq=False)
class HipBlockNorm(BlockNormStrategy):
    core: DefaultBlockNorm

    @classmethod
    def build(cls, pre, post, *, residual_scale, block_scale, activation) -> "HipBlockNorm | None":
        weights = [leaf.weight for leaf in (pre, post) if leaf is not None]
        if any(w.dtype != torch.bfloat16 or not applies(w.numel()) for w in weights) or not hip_device(*weights):
            return None
        if not all(in_place(w) for w in weights):
            return None
        return cls(DefaultBlockNorm.build(pre, post, residual_scale=residual_scale, block_scale=block_scale,
                                          activation=activation))

    def __call__(self, x, block, gate=None):
        core, post = self.core, self.core.post
        fine = x.dtype is BF16 and block.dtype is BF16
        if gate is None:
            fine = fine and (unfollowed(x, block, core.pre) if post is None else unfollowed(x, block, core.pre, post))
        else:
            fine = fine and gate.dtype is BF16 and unfollowed(x, block, gate, core.pre, *(() if post is None else (post,)))
        if not fine:
            record_fallback(self, core)
            return core(x, block, gate)
        return ops.block_norm(x, block, core.pre, post, gate, pre_eps=core.pre_eps, post_eps=core.post_eps,
                              residual_scale=core.residual_scale, block_scale=core.block_scale,
                              sigmoid=core.activation is not None)


_STRATEGIES = (HipBlockNorm, DefaultBlockNorm)


class BlockNorm(BlockNormStrategy):
    """The join that two blocks declare: picks its binding once, then forwards every call."""

    def __init__(self, pre, post=None, *, residual_scale: float = 1.0, block_scale: float = 1.0,
                 activation: str | None = None, reference: bool = False) -> None:
        if pre.weight.dim() != 1 or (post is not None and post.weight.shape != pre.weight.shape):
            raise ValueError("BlockNorm: both norms must have one weight for each value of a row")
        if activation not in ACTIVATIONS:
            raise ValueError(f"BlockNorm: gate activation {activation!r}, not one of {ACTIVATIONS}")
        self.strategy: BlockNormStrategy = resolve(
            (DefaultBlockNorm,) if reference else _STRATEGIES, pre, post, residual_scale=float(residual_scale),
            block_scale=float(block_scale), activation=activation)

    def __call__(self, x: torch.Tensor, block: torch.Tensor,
                 gate: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        return self.strategy(x, block, gate)
