"""`[trainer] linear_precision = "fp8"`: the projections of every transformer block on 8-bit products.

Marks the `nn.Linear` layers of attention and MLP in every block of the algorithm (encoder, decoder, teacher);
`apply_linear` then runs them through `ops.fp8.fp8_linear`. Patch embedding, heads and everything outside the
blocks stay in bf16, and the optimizer keeps its fp32 master weights.
"""

from __future__ import annotations

import logging

import torch.nn as nn

from ..layers.common.blocks import TransformerBlock
from ..layers.common.lora import LoRAMixin, use_fp8
from ..layers.dinov3.block import SelfAttentionBlock

logger = logging.getLogger(__name__)


def fp8_targets(root: nn.Module) -> dict[str, nn.Linear]:
    out: dict[str, nn.Linear] = {}
    for name, block in root.named_modules():
        if isinstance(block, (TransformerBlock, SelfAttentionBlock)):
            for part in ("attn", "mlp"):
                for sub, m in getattr(block, part).named_modules():
                    if isinstance(m, nn.Linear):
                        out[f"{name}.{part}.{sub}"] = m
    return out


def apply_fp8_linears(algorithm: nn.Module, tp: int = 1) -> int:
    """Mark every block projection of `algorithm`; returns how many."""
    targets = fp8_targets(algorithm)
    if not targets:
        raise ValueError(f"linear_precision = 'fp8', but nothing under {type(algorithm).__name__} is a transformer block")
    adapted = [name for name, m in targets.items() if isinstance(m, LoRAMixin)]
    if adapted:
        raise ValueError(
            f"linear_precision = 'fp8' cannot be combined with [lora] ({adapted[0]}, ... {len(adapted)} adapted layers): "
            "the adapters' base products stay in bf16"
        )
    if tp > 1:
        raise ValueError(f"linear_precision = 'fp8' cannot be combined with tensor parallelism (tp = {tp})")
    for m in targets.values():
        use_fp8(m)
    logger.info("fp8: %d projections", len(targets))
    return len(targets)
