"""Dropout from a counter-based generator, fused with a residual add; the mask is never stored.

`dropout(x, p, residual=, rng=)` returns `residual + keep * x / (1 - p')` with
`p' = round(65536 p) / 65536`: element i is kept where a 16-bit random value h(i) is at least
`65536 p'`. h(i) is a half of a word of Philox4x32-10 for the counter (i // 8, offset) under the key
`seed` (`csrc/dropout.cu` states the layout), so the backward pass recomputes the mask from
(seed, offset) and keeps nothing of the size of x. i counts x's elements in row-major order, whatever
its strides.

`rng` is an int64 tensor (seed, offset) on x's device, which makes the mask a function of the
inputs; without it the pair is drawn from PyTorch's generator of that device, so `torch.manual_seed`
reproduces it, activation checkpointing's saved generator state replays it, and every replay of a
captured graph draws a new one. `set_rank(r)` takes the drawn seeds of data-parallel ranks, which seed
their generators alike, apart; the Trainer calls it. Calls that share an `rng` share their mask. CPU tensors run the
same generator in PyTorch and give the same masks.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._native import native, use_native

STEPS = 65536  # resolution of the drop probability
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_WORD = 0xFFFFFFFF


def _mul_hi_lo(a: torch.Tensor, m: int) -> tuple[torch.Tensor, torch.Tensor]:
    low = (a & 0xFFFF) * m
    high = (a >> 16) * m + (low >> 16)
    return high >> 16, ((high & 0xFFFF) << 16) | (low & 0xFFFF)


def random_halves_reference(count: int, rng: torch.Tensor) -> torch.Tensor:
    """h(0) .. h(count - 1) as int64, from `rng` = (seed, offset)."""
    group = torch.arange(-(-count // 8), device=rng.device)
    seed, offset = rng[0], rng[1]
    c0, c1 = group & _WORD, group >> 32
    c2, c3 = (offset & _WORD).expand_as(group), ((offset >> 32 & _WORD) | 0x80000000).expand_as(group)
    k0, k1 = seed & _WORD, seed >> 32 & _WORD
    for _ in range(10):
        h0, l0 = _mul_hi_lo(c0, 0xD2511F53)
        h1, l1 = _mul_hi_lo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & _WORD, (k1 + 0xBB67AE85) & _WORD
    words = torch.stack([c0, c1, c2, c3], 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:count]


def dropout_reference(
    x: torch.Tensor, dropped: int, rng: torch.Tensor, residual: torch.Tensor | None = None
) -> torch.Tensor:
    """`dropped` = round(65536 p) of every 65536 elements go; fp32 math (fp64 for fp64), rounded once."""
    acc = torch.promote_types(x.dtype, torch.float32)
    scale = 0.0 if dropped >= STEPS else STEPS / (STEPS - dropped)
    keep = (random_halves_reference(x.numel(), rng) >= dropped).view(x.shape)
    y = torch.where(keep, x.to(acc) * scale, torch.zeros((), dtype=acc, device=x.device))
    return (y if residual is None else residual.to(acc) + y).to(x.dtype)


_rank_key = 0


def set_rank(rank: int) -> None:
    """Masks that this process draws from here on are those of data-parallel rank `rank`; 0 is what one process draws.
    An `rng` that a caller passes is taken as it is."""
    global _rank_key
    if rank < 0:
        raise ValueError(f"rank must not be negative, got {rank}")
    key = rank * 0x9E3779B97F4A7C15 % (1 << 64)  # odd: distinct for distinct ranks
    _rank_key = key - (1 << 64) if key >> 63 else key


def _draw(device: torch.device) -> torch.Tensor:
    seed = torch.randint(-(1 << 63), (1 << 63) - 1, (1,), device=device) ^ _rank_key
    return torch.cat([seed, torch.zeros_like(seed)])


class _Dropout(torch.autograd.Function):
    """The PyTorch path; on CUDA `csrc/block_ops.cpp` holds the same node."""

    @staticmethod
    def forward(ctx, x, residual, dropped, rng):  # type: ignore[override]
        # the pair is copied, as the kernel does: the caller may advance its own before the backward pass
        used = _draw(x.device) if rng is None else rng.clone()
        ctx.dropped = dropped
        ctx.save_for_backward(used)
        return dropout_reference(x, dropped, used, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):  # type: ignore[override]
        (used,) = ctx.saved_tensors
        dx = dropout_reference(dy, ctx.dropped, used) if ctx.needs_input_grad[0] else None
        return dx, (dy if ctx.needs_input_grad[1] else None), None, None


def dropout(
    x: torch.Tensor,
    p: float,
    *,
    residual: torch.Tensor | None = None,
    training: bool = True,
    rng: torch.Tensor | None = None,
) -> torch.Tensor:
    """`residual + dropout(x, p)`; see the module docstring. `training=False` is `residual + x`."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be within [0, 1], got {p}")
    if not x.is_floating_point():
        raise ValueError(f"dropout needs a floating-point tensor, got {x.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(
            f"residual must match x in shape, dtype and device: got {tuple(residual.shape)} {residual.dtype} "
            f"{residual.device} for {tuple(x.shape)} {x.dtype} {x.device}"
        )
    if rng is not None and (rng.dtype != torch.int64 or rng.shape != (2,) or rng.device != x.device):
        raise ValueError(
            f"rng must be an int64 (seed, offset) tensor of shape (2,) on {x.device}, got {rng.dtype} "
            f"{tuple(rng.shape)} on {rng.device}"
        )
    dropped = round(p * STEPS) if training else 0
    if dropped == 0:
        return x if residual is None else residual + x
    if x.dtype in _DTYPES and use_native(x):
        return native().dropout(x, residual, dropped, rng, _rank_key)
    return _Dropout.apply(x, residual, dropped, rng)
