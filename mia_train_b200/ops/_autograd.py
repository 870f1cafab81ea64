"""Refusal of second derivatives, shared by the Python autograd nodes."""

from __future__ import annotations

import functools
from collections.abc import Callable
from typing import Any

import torch


def differentiable_once(what: str) -> Callable:
    """For a node's `backward`: runs it without recording, and refuses to run it under `create_graph` where its result
    depends on anything that wants a gradient: the incoming gradient, or (`ctx.open`) an operand. PyTorch's
    `once_differentiable` looks at the incoming gradient alone, so that behind a constant one the second
    derivative would be missing without a word."""

    def wrap(backward: Callable) -> Callable:
        @functools.wraps(backward)
        def run(ctx: Any, *grads: torch.Tensor | None) -> Any:
            if torch.is_grad_enabled() and (ctx.open or any(g is not None and g.requires_grad for g in grads)):
                raise RuntimeError(f"{what}: the backward pass is differentiable once only")
            with torch.no_grad():
                return backward(ctx, *grads)

        return run

    return wrap
